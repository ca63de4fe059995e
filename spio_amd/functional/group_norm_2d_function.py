"""`spio::group_norm_2d_forward` and its backward: group norm with an activation over channels_last tensors.

    mean, var over the pixels and the C/G channels of a group;  z = (x - mean) * rsqrt(var + eps) * weight + bias
    y = act(z),  act one of none, relu, silu, gelu (of the normal distribution)

With `checkpoint_8bit` the forward pass writes its input in the 8-bit form of csrc/spio_pointwise.h (blocks of up to
32 channels of a pixel, a power-of-two step each) and the backward pass reads that in the input's place: half of what
a float16 input keeps, a quarter of a float32 one's.  Mean and rstd are those of the input itself.  The gradients are
then those of the formula at the values the checkpoint stands for, each off by half a step at most; but where relu's passes,
which half a step would decide, is that of the input itself and kept in a bit a value more.

All sums are float32: those of a group's values and of the squares of their differences to the mean have to stay below
its largest number (3.4e38), which bfloat16 and float32 values beyond 10^16 may pass.

The reference has no such operator; its sibling here is `layernorm_2d`.
"""

from typing import Optional, Tuple

import torch
from torch.autograd.forward_ad import unpack_dual

from .. import native
from ..kernels.group_norm_2d_kernel import (
    ACTIVATIONS,
    DTYPES,
    GroupNorm2dParams,
    group_norm_2d_bwd_kernel_factory,
    group_norm_2d_kernel_factory,
    kept_shapes,
)

CL = torch.channels_last


def aligned(t: torch.Tensor) -> torch.Tensor:
    """The tensor, or a copy where it does not start on 16 bytes (the kernels load that much at once)."""
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.preserve_format)


def _vector(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.detach().float().contiguous()


def _params(shape, num_groups, dtype, activation, eps, weight, bias, kept) -> GroupNorm2dParams:
    n, c, h, w = (int(v) for v in shape)
    return GroupNorm2dParams(n=n, c=c, h=h, w=w, groups=int(num_groups), dtype=DTYPES[dtype],
                             activation=ACTIVATIONS[activation], eps=float(eps), has_weight=weight is not None,
                             has_bias=bias is not None, kept=bool(kept))  # fmt: skip


def _check(inputs, num_groups, weight, bias, eps, activation):
    assert inputs.dim() == 4, "group_norm_2d takes an NCHW tensor"
    assert inputs.dtype in DTYPES, "group_norm_2d takes float16, bfloat16 or float32 tensors"
    assert activation in ACTIVATIONS, f"activation must be one of {tuple(ACTIVATIONS)}, not {activation!r}"
    c = inputs.shape[1]
    assert num_groups > 0 and c % num_groups == 0, "channels must be a multiple of num_groups"
    assert c > 0 and c % 8 == 0, "channels must be a multiple of 8 (16-byte units)"
    assert 0 < eps < float("inf"), "eps must be positive and finite"
    for t in (weight, bias):
        assert t is None or (t.dim() == 1 and t.shape[0] == c and t.is_floating_point()), "weight and bias are [C]"
        assert t is None or t.device == inputs.device, "weight and bias must be on the inputs' device"


def _empty_like_kept(inputs, kept, activation):
    """Codes and exponents of an input, empty where it is not kept."""
    shapes = kept_shapes(*inputs.shape, ACTIVATIONS[activation]) if kept else ((0,), (0,))
    return inputs.new_empty(shapes[0], dtype=torch.int8), inputs.new_empty(shapes[1], dtype=torch.uint8)


@torch.library.custom_op("spio::group_norm_2d_forward", mutates_args=())
def group_norm_2d_forward(
    inputs: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float,
    activation: str, checkpoint_8bit: bool,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:  # fmt: skip
    """(output, statistics [n, groups, 2] = mean and rstd in float32, codes, exponents); the last two are empty
    without `checkpoint_8bit`.  Codes are [n, h, w, c], exponents [n, h, w, ceil(c / 32)], with relu followed by c / 8
    bytes of bits, whether the gradient of an output passes."""
    _check(inputs, num_groups, weight, bias, eps, activation)
    if inputs.device.type != "cuda":
        raise ValueError("spio::group_norm_2d runs on the GPU only")
    params = _params(inputs.shape, num_groups, inputs.dtype, activation, eps, weight, bias, checkpoint_8bit)
    x = aligned(inputs.contiguous(memory_format=CL))
    out = torch.empty_like(x, memory_format=CL)
    stats = torch.empty((params.n, params.groups, 2), dtype=torch.float32, device=x.device)
    codes, exponents = _empty_like_kept(x, params.kept, activation)
    if x.numel() == 0:
        return out, stats.zero_(), codes, exponents
    kernel = group_norm_2d_kernel_factory.get_kernel(params, x.device)
    kept = (codes, exponents) if params.kept else (None, None)
    kernel(out, *kept, stats, x, _vector(weight), _vector(bias), params.pixels, params.n)
    return out, stats, codes, exponents


@group_norm_2d_forward.register_fake
def _forward_fake(inputs, num_groups, weight, bias, eps, activation, checkpoint_8bit):
    _check(inputs, num_groups, weight, bias, eps, activation)
    return (torch.empty_like(inputs, memory_format=CL),
            inputs.new_empty((inputs.shape[0], num_groups, 2), dtype=torch.float32),
            *_empty_like_kept(inputs, checkpoint_8bit, activation))  # fmt: skip


@torch.library.custom_op("spio::group_norm_2d_backward", mutates_args=())
def group_norm_2d_backward(
    grad_output: torch.Tensor, inputs: torch.Tensor, exponents: Optional[torch.Tensor], stats: torch.Tensor,
    num_groups: int, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float, activation: str,
) -> Tuple[torch.Tensor, torch.Tensor]:  # fmt: skip
    """(grad_input in grad_output's type, [grad_weight; grad_bias] float32 as one [2, C] tensor).  With `exponents`,
    `inputs` are codes [n, h, w, c] of the 8-bit form."""
    assert grad_output.dim() == 4 and grad_output.dtype in DTYPES
    n, c, h, w = (int(v) for v in grad_output.shape)
    kept = exponents is not None
    _check(grad_output, num_groups, weight, bias, eps, activation)
    if grad_output.device.type != "cuda":
        raise ValueError("spio::group_norm_2d runs on the GPU only")
    assert inputs.device == stats.device == grad_output.device
    assert stats.dtype == torch.float32 and tuple(stats.shape) == (n, num_groups, 2), "statistics of another norm"
    if kept:
        shapes = kept_shapes(n, c, h, w, ACTIVATIONS[activation])
        assert inputs.dtype == torch.int8 and tuple(inputs.shape) == shapes[0], "codes of another input"
        assert exponents.dtype == torch.uint8 and tuple(exponents.shape) == shapes[1], "exponents of another input"
        assert exponents.device == grad_output.device
        x, exponents = aligned(inputs.contiguous()), exponents.contiguous()
    else:
        assert inputs.shape == grad_output.shape and inputs.dtype == grad_output.dtype, "inputs of another norm"
        x = aligned(inputs.contiguous(memory_format=CL))
    dy = aligned(grad_output.contiguous(memory_format=CL))
    grad_input = torch.empty_like(dy, memory_format=CL)
    sums = torch.empty((2, c), dtype=torch.float32, device=dy.device)
    if dy.numel() == 0:
        return grad_input, sums.zero_()
    params = _params(dy.shape, num_groups, dy.dtype, activation, eps, weight, bias, kept)
    kernel = group_norm_2d_bwd_kernel_factory.get_kernel(params, dy.device)
    affine = weight is not None or bias is not None
    kernel(sums if affine else None, grad_input, x, exponents, dy, stats.contiguous(), _vector(weight), _vector(bias),
           params.pixels, params.n)  # fmt: skip
    return grad_input, sums if affine else sums.zero_()


@group_norm_2d_backward.register_fake
def _backward_fake(grad_output, inputs, exponents, stats, num_groups, weight, bias, eps, activation):
    c = grad_output.shape[1]
    return (torch.empty_like(grad_output, memory_format=CL),
            grad_output.new_empty((2, c), dtype=torch.float32))  # fmt: skip


def refuse_second_derivatives():
    """What is kept in 8 bits has no history: a gradient of a gradient would take it for a constant."""
    if torch.is_grad_enabled() and not torch.compiler.is_compiling():
        raise RuntimeError("an input that was kept in 8 bits has no second derivatives (create_graph=True)")


def refuse_forward_derivatives(*tensors):
    """The operators have no formula for forward mode; a tangent would vanish on the way, as if it were zero."""
    if not torch.compiler.is_compiling() and any(t is not None and unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("no forward-mode derivatives of this operator")


def group_norm_2d_gradients(grad_output, inputs, exponents, stats, num_groups, weight, bias, eps, activation, needs_input,
                            needs_weight, needs_bias):  # fmt: skip
    """Gradients of group_norm_2d in the types of the tensors they belong to, None where not needed."""
    if exponents is not None:
        refuse_second_derivatives()
    grad_input, sums = group_norm_2d_backward(grad_output, inputs, exponents, stats, num_groups, weight, bias, eps,
                                              activation)  # fmt: skip
    return (
        grad_input if needs_input else None,
        sums[0].to(weight.dtype) if needs_weight else None,
        sums[1].to(bias.dtype) if needs_bias else None,
    )


def _setup_context(ctx, inputs, output):
    x, num_groups, weight, bias, eps, activation, kept = inputs
    _, stats, codes, exponents = output
    ctx.mark_non_differentiable(stats, codes, exponents)
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(codes if kept else x, exponents if kept else None, stats, weight, bias)
    ctx.numbers = (num_groups, eps, activation)


def _backward(ctx, grad_output, *_unused):
    if grad_output is None:
        return (None,) * 7
    x, exponents, stats, weight, bias = ctx.saved_tensors
    num_groups, eps, activation = ctx.numbers
    needs = ctx.needs_input_grad
    dx, dw, db = group_norm_2d_gradients(grad_output, x, exponents, stats, num_groups, weight, bias, eps, activation,
                                         needs[0], weight is not None and needs[2], bias is not None and needs[3])  # fmt: skip
    return dx, None, dw, db, None, None, None


group_norm_2d_forward.register_autograd(_backward, setup_context=_setup_context)


def group_norm_2d(
    inputs: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
    eps: float = 1e-5, activation: str = "none", checkpoint_8bit: bool = False,
) -> torch.Tensor:  # fmt: skip
    """act(group_norm(inputs) * weight + bias) for an NCHW tensor with channels_last strides.

    Args:
        inputs: (N, C, H, W) float16, bfloat16 or float32; C a multiple of 8 (up to 4096) and of num_groups.
        weight, bias: optional (C,), any float type.
        eps: positive and finite; below 2^-126 it counts as that.
        activation: "none", "relu", "silu" or "gelu".
        checkpoint_8bit: keep the input for the backward pass in 8 bits (and a bit more for relu).

    Returns:
        (N, C, H, W) in the inputs' type, channels_last.
    """
    y = native.call("group_norm_2d", inputs, num_groups, weight, bias, eps, activation, checkpoint_8bit)
    if y is not NotImplemented:
        return y
    refuse_forward_derivatives(inputs, weight, bias)
    kept = bool(checkpoint_8bit) and torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (inputs, weight, bias))  # fmt: skip
    return group_norm_2d_forward(inputs, num_groups, weight, bias, eps, activation, kept)[0]
