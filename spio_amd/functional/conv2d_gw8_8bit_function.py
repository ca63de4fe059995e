"""`conv2d_gw8_8bit`: spio::conv2d_gw8 with its input kept in 8 bits between the forward and the backward pass.

The output is conv2d_gw8's, and so is grad_input, which needs the weights only; grad_weight is that of the input as the
8-bit form (functional/activation_8bit_function.py) stands for it.  The reference has no such operator.
"""

from typing import Optional, Tuple

import torch

from .. import native
from .activation_8bit_function import pack_8bit_op, unpack_8bit_op
from .conv2d_gw8_function import conv2d_gw8, conv2d_gw8_backward_op
from .group_norm_2d_function import refuse_forward_derivatives, refuse_second_derivatives

CL = torch.channels_last


def _half(t):
    return t.to(torch.float16).contiguous(memory_format=CL)


@torch.library.custom_op("spio::conv2d_gw8_8bit_forward", mutates_args=())
def conv2d_gw8_8bit_forward(
    inputs: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], padding_y: int, padding_x: int,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:  # fmt: skip
    """(conv2d_gw8's output in the inputs' type, codes, exponents of the input with channels_last strides).  Tensors
    of other types than conv2d_gw8's are rounded to those first."""
    x = _half(inputs)
    out = conv2d_gw8(x, _half(weight), None if bias is None else bias.float(), 1, padding_y, padding_x, 1,
                     inputs.shape[1] // 8)  # fmt: skip
    return (out.to(inputs.dtype), *pack_8bit_op(x))


@conv2d_gw8_8bit_forward.register_fake
def _forward_fake(inputs, weight, bias, padding_y, padding_x):
    n, c, h, w = inputs.shape
    out = (n, c, h + 2 * padding_y - weight.shape[2] + 1, w + 2 * padding_x - weight.shape[3] + 1)
    return (inputs.new_empty(out).to(memory_format=CL), *pack_8bit_op(_half(inputs)))


def _setup_context(ctx, inputs, output):
    x, weight, bias, *ctx.padding = inputs
    _, codes, exponents = output
    ctx.mark_non_differentiable(codes, exponents)
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(codes, exponents, weight, bias)
    ctx.shape, ctx.dtype = x.shape, x.dtype


def conv2d_gw8_8bit_gradients(grad_output, codes, exponents, weight, bias, shape, padding_y, padding_x, needs_input,
                              needs_weight, needs_bias):  # fmt: skip
    """Gradients of conv2d_gw8_8bit in conv2d_gw8's types, None where not needed."""
    refuse_second_derivatives()
    n, c, h, w = shape
    if needs_weight:
        x = unpack_8bit_op(codes, exponents, [n, c, h, w], [h * w * c, 1, w * c, c], torch.float16)
    else:  # the operator asks for its sizes only
        x = torch.empty((n, c, h, w), dtype=torch.float16, device=grad_output.device, memory_format=CL)
    return conv2d_gw8_backward_op(x, _half(weight), None if bias is None else bias.float(), _half(grad_output),
                                  padding_y, padding_x, needs_input, needs_weight, needs_bias)  # fmt: skip


def _backward(ctx, grad_output, *_unused):
    if grad_output is None:
        return (None,) * 5
    codes, exponents, weight, bias = ctx.saved_tensors
    needs = ctx.needs_input_grad
    dx, dw, db = conv2d_gw8_8bit_gradients(grad_output, codes, exponents, weight, bias, tuple(ctx.shape), *ctx.padding,
                                           needs[0], needs[1], bias is not None and needs[2])  # fmt: skip
    return (None if dx is None else dx.to(ctx.dtype), None if dw is None else dw.to(weight.dtype),
            None if db is None else db.to(bias.dtype), None, None)  # fmt: skip


conv2d_gw8_8bit_forward.register_autograd(_backward, setup_context=_setup_context)


def conv2d_gw8_8bit(
    inputs: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, stride: int = 1,
    padding_y: int = 0, padding_x: int = 0, dilation: int = 1, groups: int = 1,
) -> torch.Tensor:  # fmt: skip
    """conv2d_gw8 (the same arguments, checks and autocast rules) that keeps its input for grad_weight in 8 bits.
    Where no grad_weight is wanted it is conv2d_gw8."""
    if not (torch.is_grad_enabled() and weight.requires_grad):
        refuse_forward_derivatives(inputs, weight, bias)
        return conv2d_gw8(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)
    y = native.call("conv2d_gw8_8bit", inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)
    if y is not NotImplemented:
        return y
    refuse_forward_derivatives(inputs, weight, bias)
    if not torch.is_autocast_enabled("cuda"):
        assert inputs.dtype == torch.float16 and weight.dtype == torch.float16
        assert bias is None or bias.dtype == torch.float32
    assert stride in (1, (1, 1)) and dilation in (1, (1, 1)) and groups == inputs.shape[1] // 8
    with torch.autocast("cuda", enabled=False):
        return conv2d_gw8_8bit_forward(inputs, weight, bias, padding_y, padding_x)[0]
