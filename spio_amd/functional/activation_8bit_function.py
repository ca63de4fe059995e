"""The 8-bit form of activations between the forward and the backward pass: `pack_8bit`, `unpack_8bit`, and
`activation_8bit`, which keeps its input that way.

A tensor is cut into blocks of 32 values that are neighbours in memory; a block is a signed byte a value and a byte
for its power-of-two step, the smallest of which the largest magnitude is less than 127.5 (csrc/spio_pointwise.h).
Values come back off by half a step at most, 1/127.5 of the block's largest at the most.  A block that holds an infinity or
a NaN comes back as NaN.

The reference has no such operators.
"""

from typing import List, NamedTuple, Tuple

import torch

from .. import native
from ..kernels.activation_8bit_kernel import (
    BLOCK,
    Activation8bitParams,
    activation_8bit_bwd_kernel_factory,
    activation_8bit_kernel_factory,
    pack_8bit_kernel_factory,
    unpack_8bit_kernel_factory,
)
from ..kernels.group_norm_2d_kernel import ACTIVATIONS, DTYPES
from ..util.math import divup
from .group_norm_2d_function import aligned, refuse_forward_derivatives, refuse_second_derivatives

POINTWISE = tuple(name for name in ACTIVATIONS if name != "none")


class Packed8bit(NamedTuple):
    """A tensor in the 8-bit form: codes and exponents in the order of the memory that `shape` and `strides` describe,
    and the type it had."""

    codes: torch.Tensor
    exponents: torch.Tensor
    shape: Tuple[int, ...]
    strides: Tuple[int, ...]
    dtype: torch.dtype


def _is_dense(shape, strides) -> bool:
    """Whether strides of that shape leave no gap and no overlap."""
    expected = 1
    for stride, size in sorted((st, sz) for sz, st in zip(shape, strides) if sz != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def dense(t: torch.Tensor) -> torch.Tensor:
    """The tensor, or a copy without gaps where it has some."""
    return t if t.numel() == 0 or _is_dense(t.shape, t.stride()) else t.contiguous()


def _require_gpu(t, what):
    if t.device.type != "cuda":
        raise ValueError(f"spio::{what} runs on the GPU only")


def _kept_sizes(n, activation=None):
    """Bytes of codes and of exponents: one a value and one a block, or, for relu, a bit a value and none."""
    return (divup(n, 8), 0) if activation == "relu" else (n, divup(n, BLOCK))


def _empty_kept(t, kept=True, activation=None):
    sizes = _kept_sizes(t.numel() if kept else 0, activation)
    return t.new_empty((sizes[0],), dtype=torch.int8), t.new_empty((sizes[1],), dtype=torch.uint8)


def _check_kept(codes, exponents, n, device, activation=None):
    sizes = _kept_sizes(n, activation)
    assert codes.dtype == torch.int8 and tuple(codes.shape) == (sizes[0],), "codes of another tensor"
    assert exponents.dtype == torch.uint8 and tuple(exponents.shape) == (sizes[1],), "exponents of another tensor"
    assert codes.device == exponents.device == device, "codes and exponents must be on one device"


@torch.library.custom_op("spio::pack_8bit", mutates_args=())
def pack_8bit_op(inputs: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes, exponents) of a tensor without gaps, in the order of its memory."""
    assert inputs.dtype in DTYPES, "pack_8bit takes float16, bfloat16 or float32 tensors"
    assert inputs.numel() == 0 or _is_dense(inputs.shape, inputs.stride()), "pack_8bit takes a tensor without gaps"
    _require_gpu(inputs, "pack_8bit")
    x = aligned(inputs)
    codes, exponents = _empty_kept(x)
    n = x.numel()
    if n:
        kernel = pack_8bit_kernel_factory.get_kernel(Activation8bitParams(DTYPES[x.dtype]), x.device)
        kernel(codes, exponents, x, n)
    return codes, exponents


@pack_8bit_op.register_fake
def _pack_fake(inputs):
    return _empty_kept(inputs)


@torch.library.custom_op("spio::unpack_8bit", mutates_args=())
def unpack_8bit_op(codes: torch.Tensor, exponents: torch.Tensor, shape: List[int], strides: List[int],
                   dtype: torch.dtype) -> torch.Tensor:  # fmt: skip
    """The values of codes and exponents in a new tensor of that shape, strides and type."""
    assert dtype in DTYPES, "unpack_8bit makes float16, bfloat16 or float32 tensors"
    assert len(shape) == len(strides)
    n = 1
    for size in shape:
        assert size >= 0
        n *= size
    assert n == 0 or _is_dense(shape, strides), "unpack_8bit makes tensors without gaps"
    _check_kept(codes, exponents, n, codes.device)
    _require_gpu(codes, "unpack_8bit")
    out = torch.empty_strided(tuple(shape), tuple(strides), dtype=dtype, device=codes.device)
    if n:
        kernel = unpack_8bit_kernel_factory.get_kernel(Activation8bitParams(DTYPES[dtype]), codes.device)
        kernel(out, aligned(codes.contiguous()), exponents.contiguous(), n)
    return out


@unpack_8bit_op.register_fake
def _unpack_fake(codes, exponents, shape, strides, dtype):
    return torch.empty_strided(tuple(shape), tuple(strides), dtype=dtype, device=codes.device)


def pack_8bit(inputs: torch.Tensor) -> Packed8bit:
    """A float16, bfloat16 or float32 GPU tensor of any shape in the 8-bit form, 33/64 of its size in 16 bits.  A
    tensor with gaps is packed as its contiguous copy.  No gradient passes through."""
    x = dense(inputs.detach())
    kept = native.call("pack_8bit", x)
    return Packed8bit(*(pack_8bit_op(x) if kept is NotImplemented else kept), tuple(x.shape), tuple(x.stride()), x.dtype)


def unpack_8bit(packed: Packed8bit, dtype: torch.dtype = None) -> torch.Tensor:
    """The tensor that `packed` stands for, in its own type or another one (float16: the largest finite value in
    place of larger ones)."""
    dtype = packed.dtype if dtype is None else dtype
    out = native.call("unpack_8bit", packed.codes, packed.exponents, packed.shape, packed.strides, dtype)
    if out is not NotImplemented:
        return out
    return unpack_8bit_op(packed.codes, packed.exponents, list(packed.shape), list(packed.strides), dtype)


# ---- an activation that keeps its input in 8 bits ----


def _check_activation(inputs, activation):
    assert inputs.dtype in DTYPES, "activation_8bit takes float16, bfloat16 or float32 tensors"
    assert activation in POINTWISE, f"activation must be one of {POINTWISE}, not {activation!r}"


@torch.library.custom_op("spio::activation_8bit_forward", mutates_args=())
def activation_8bit_forward(inputs: torch.Tensor, activation: str,
                            keep: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:  # fmt: skip
    """(act(inputs), codes, exponents) of a tensor without gaps; the last two are empty unless `keep`.  relu's codes are
    a bit a value, whether its gradient passes there (bit e of byte u is value 8u + e's), and it has no exponents."""
    _check_activation(inputs, activation)
    assert inputs.numel() == 0 or _is_dense(inputs.shape, inputs.stride()), "activation_8bit takes a tensor without gaps"
    _require_gpu(inputs, "activation_8bit")
    x = aligned(inputs)
    out = torch.empty_like(x)
    codes, exponents = _empty_kept(x, keep, activation)
    n = x.numel()
    if n:
        params = Activation8bitParams(DTYPES[x.dtype], ACTIVATIONS[activation], keep)
        kernel = activation_8bit_kernel_factory.get_kernel(params, x.device)
        kernel(out, *((codes, exponents) if keep else (None, None)), x, n)
    return out, codes, exponents


@activation_8bit_forward.register_fake
def _activation_fake(inputs, activation, keep):
    _check_activation(inputs, activation)
    return (torch.empty_like(inputs), *_empty_kept(inputs, keep, activation))


@torch.library.custom_op("spio::activation_8bit_backward", mutates_args=())
def activation_8bit_backward(grad_output: torch.Tensor, codes: torch.Tensor, exponents: torch.Tensor,
                             activation: str) -> torch.Tensor:  # fmt: skip
    """grad_output * act'(the kept input), for relu act'(the input); grad_output lies in memory as the input did."""
    _check_activation(grad_output, activation)
    n = grad_output.numel()
    assert n == 0 or _is_dense(grad_output.shape, grad_output.stride())
    _check_kept(codes, exponents, n, grad_output.device, activation)
    _require_gpu(grad_output, "activation_8bit")
    dy = aligned(grad_output)
    grad_input = torch.empty_like(dy)
    if n:
        params = Activation8bitParams(DTYPES[dy.dtype], ACTIVATIONS[activation])
        kernel = activation_8bit_bwd_kernel_factory.get_kernel(params, dy.device)
        kernel(grad_input, aligned(codes.contiguous()), exponents.contiguous(), dy, n)
    return grad_input


@activation_8bit_backward.register_fake
def _activation_backward_fake(grad_output, codes, exponents, activation):
    return torch.empty_like(grad_output)


def laid_out(t: torch.Tensor, strides) -> torch.Tensor:
    """The tensor with these strides, itself if it has them."""
    if t.stride() == tuple(strides) or t.numel() == 0:
        return t
    return torch.empty_strided(t.shape, tuple(strides), dtype=t.dtype, device=t.device).copy_(t)


def activation_8bit_gradient(grad_output, codes, exponents, activation, strides):
    """grad_input of activation_8bit whose input lay in memory by these strides."""
    refuse_second_derivatives()
    return activation_8bit_backward(laid_out(grad_output, strides), codes, exponents, activation)


def _setup_context(ctx, inputs, output):
    out, codes, exponents = output
    ctx.mark_non_differentiable(codes, exponents)
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(codes, exponents)
    ctx.activation = inputs[1]
    ctx.strides = out.stride()


def _backward(ctx, grad_output, *_unused):
    if grad_output is None:
        return None, None, None
    codes, exponents = ctx.saved_tensors
    return activation_8bit_gradient(grad_output, codes, exponents, ctx.activation, ctx.strides), None, None


activation_8bit_forward.register_autograd(_backward, setup_context=_setup_context)


def activation_8bit(inputs: torch.Tensor, activation: str = "gelu") -> torch.Tensor:
    """relu, silu or gelu (of the normal distribution) of a GPU tensor of any shape, in its type; what the backward
    pass needs of the input is kept in 8 bits.  relu needs its sign only and keeps that, in one bit: its gradient is the
    input's own."""
    y = native.call("activation_8bit", inputs, activation)
    if y is not NotImplemented:
        return y
    refuse_forward_derivatives(inputs)
    keep = torch.is_grad_enabled() and inputs.requires_grad
    return activation_8bit_forward(dense(inputs), activation, keep)[0]
