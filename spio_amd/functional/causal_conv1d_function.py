"""`spio::causal_conv1d_forward`, its backward and `spio::causal_conv1d_step`: a short convolution along the tokens of
[sequences, tokens, channels] tensors, each channel with its own filter, and an activation.

    z[t] = bias + sum_i weight[:, i] inputs[t - W + 1 + i],   y = act(z),   act none or silu

A token sees itself and the W - 1 before it: zeros before the first one, or the `initial_state` that a call before this
one returned.  Sums are float32; the activation's derivative is taken at z as it is computed again from the inputs.

The reference has no such operator; its sibling here is `conv2d_gw8`.
"""

from typing import Optional, Tuple, Union

import torch

from .. import native
from ..kernels.causal_conv1d_kernel import (
    ACTIVATIONS,
    MAX_WIDTH,
    MIN_WIDTH,
    CausalConv1dParams,
    causal_conv1d_bwd_kernel_factory,
    causal_conv1d_kernel_factory,
    causal_conv1d_step_kernel_factory,
    causal_conv1d_sums_kernel_factory,
    slice_tokens,
)
from ..kernels.group_norm_2d_kernel import DTYPES
from ..kernels.token_args import Arguments
from ..util.math import divup
from .group_norm_2d_function import aligned, refuse_forward_derivatives
from .token_rows import (
    check_out_state,
    check_parameters,
    check_tokens,
    refuse_inference_state,
    refuse_state_gradients,
    require_gpu,
    rows_of,
)

STRUCT = "SpioConv1dArgs"
SUM_COLUMNS = 32  # of a workgroup that adds up partial sums


def _check(what, inputs, dims, weight, bias, activation, state):
    assert inputs.dim() == dims, f"{what} takes {'[sequences, tokens, channels]' if dims == 3 else '[sequences, channels]'}"
    c = inputs.shape[-1]
    assert weight.dim() == 2 and MIN_WIDTH <= weight.shape[1] <= MAX_WIDTH, f"weight is [channels, {MIN_WIDTH}..{MAX_WIDTH}]"
    assert c > 0 and c % 8 == 0, "channels must be a multiple of 8 (16-byte units)"
    assert activation in ACTIVATIONS, f"activation must be one of {tuple(ACTIVATIONS)}, not {activation!r}"
    check_tokens(what, inputs=inputs, state=state)
    check_parameters(what, inputs, weight=(weight, (c, weight.shape[1])), bias=(bias, (c,)))
    if state is not None:
        assert tuple(state.shape) == (inputs.shape[0], weight.shape[1] - 1, c), "a state is [sequences, width - 1, channels]"


def _filters(weight, bias):
    """Weight and bias as the kernels read them: one type, no gaps, on 16 bytes."""
    weight, bias = weight.detach(), None if bias is None else bias.detach()
    if weight.dtype not in DTYPES or (bias is not None and bias.dtype != weight.dtype):
        weight, bias = weight.float(), None if bias is None else bias.float()
    return aligned(weight.contiguous()), None if bias is None else aligned(bias.contiguous())


def _params(inputs, weight, activation):
    return CausalConv1dParams(weight.shape[1], DTYPES[inputs.dtype], DTYPES[weight.dtype], ACTIVATIONS[activation])


@torch.library.custom_op("spio::causal_conv1d_forward", mutates_args=())
def causal_conv1d_forward(
    inputs: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], activation: str,
    initial_state: Optional[torch.Tensor], keep_state: bool,
) -> Tuple[torch.Tensor, torch.Tensor]:  # fmt: skip
    """(outputs, the last W - 1 inputs; empty unless `keep_state`)."""
    _check("causal_conv1d", inputs, 3, weight, bias, activation, initial_state)
    require_gpu("causal_conv1d", inputs)
    n, l, c = inputs.shape
    x, row = rows_of(inputs, 8)
    out = torch.empty((n, l, c), dtype=x.dtype, device=x.device)
    after = x.new_empty((n, weight.shape[1] - 1, c) if keep_state else (0,))
    if out.numel() == 0:
        if after.numel():
            after.copy_(initial_state) if initial_state is not None else after.zero_()
        return out, after
    weight, bias = _filters(weight, bias)
    kernel = causal_conv1d_kernel_factory.get_kernel(_params(x, weight, activation), x.device)
    size = slice_tokens(l, c, n, False)
    before = None if initial_state is None else aligned(initial_state.contiguous())
    arguments = Arguments(STRUCT, x=x, weight=weight, bias=bias, before=before, out=out, after=after if keep_state else None,
                          tokens=l, channels=c, sequences=n, slice=size, x_row=row)  # fmt: skip
    kernel.launch_structure(divup(n * divup(l, size) * (c // 8), 256), arguments)
    return out, after


@causal_conv1d_forward.register_fake
def _forward_fake(inputs, weight, bias, activation, initial_state, keep_state):
    _check("causal_conv1d", inputs, 3, weight, bias, activation, initial_state)
    n, l, c = inputs.shape
    return inputs.new_empty((n, l, c)), inputs.new_empty((n, weight.shape[1] - 1, c) if keep_state else (0,))


@torch.library.custom_op("spio::causal_conv1d_backward", mutates_args=())
def causal_conv1d_backward(
    grad_output: torch.Tensor, inputs: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], activation: str,
    initial_state: Optional[torch.Tensor],
) -> Tuple[torch.Tensor, torch.Tensor]:  # fmt: skip
    """(grad_inputs, float32 [C * W + C]: grad_weight, then grad_bias)."""
    _check("causal_conv1d", inputs, 3, weight, bias, activation, initial_state)
    assert grad_output.shape == inputs.shape and grad_output.dtype == inputs.dtype and grad_output.device == inputs.device
    require_gpu("causal_conv1d", inputs)
    n, l, c = inputs.shape
    x, row = rows_of(inputs, 8)
    dy = aligned(grad_output.contiguous())
    weight, bias = _filters(weight, bias)
    width = weight.shape[1]
    dx = torch.empty((n, l, c), dtype=x.dtype, device=x.device)
    sums = torch.empty((c * (width + 1),), dtype=torch.float32, device=x.device)
    if dx.numel() == 0:
        return dx, sums.zero_()
    size = slice_tokens(l, c, n, True)
    slices = divup(l, size)
    partials = torch.empty((n * slices * (width + 1) * c,), dtype=torch.float32, device=x.device)
    params = _params(x, weight, activation)
    before = None if initial_state is None else aligned(initial_state.contiguous())
    arguments = Arguments(STRUCT, x=x, weight=weight, bias=bias, dy=dy, before=before, dx=dx, partials=partials, dweight=sums,
                          dbias=sums[width * c :],
                          tokens=l, channels=c, sequences=n, slice=size, x_row=row)  # fmt: skip
    main = causal_conv1d_bwd_kernel_factory.get_kernel(params, x.device)
    main.launch_structure(divup(n * slices * (c // 8), 256), arguments)
    second = causal_conv1d_sums_kernel_factory.get_kernel(params, x.device)
    second.launch_structure(divup((width + 1) * c, SUM_COLUMNS), arguments)
    return dx, sums


@causal_conv1d_backward.register_fake
def _backward_fake(grad_output, inputs, weight, bias, activation, initial_state):
    c, width = weight.shape
    return inputs.new_empty(tuple(inputs.shape)), inputs.new_empty((c * (width + 1),), dtype=torch.float32)


def causal_conv1d_gradients(grad_output, inputs, weight, bias, activation, initial_state, needs_input, needs_weight, needs_bias):
    """Gradients of causal_conv1d in the types of the tensors they belong to, None where not needed."""
    refuse_forward_derivatives(grad_output, inputs, weight, bias)
    dx, sums = causal_conv1d_backward(grad_output, inputs, weight, bias, activation, initial_state)
    return (
        dx if needs_input else None,
        sums[: weight.numel()].view(weight.shape).to(weight.dtype) if needs_weight else None,
        sums[weight.numel() :].to(bias.dtype) if needs_bias else None,
    )


def _setup_context(ctx, inputs, output):
    x, weight, bias, activation, initial_state, _ = inputs
    ctx.mark_non_differentiable(output[1])
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(x, weight, bias, initial_state)
    ctx.activation = activation


def _backward(ctx, grad_output, *_unused):
    if grad_output is None:
        return (None,) * 6
    x, weight, bias, initial_state = ctx.saved_tensors
    needs = ctx.needs_input_grad
    return (*causal_conv1d_gradients(grad_output, x, weight, bias, ctx.activation, initial_state, needs[0], needs[1],
                                     bias is not None and needs[2]), None, None, None)  # fmt: skip


causal_conv1d_forward.register_autograd(_backward, setup_context=_setup_context)


def causal_conv1d(
    inputs: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
    initial_state: Optional[torch.Tensor] = None, return_state: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:  # fmt: skip
    """act(convolution along the tokens), each channel by itself.  The state is that of the last tokens as they are: of
    sequences padded behind it holds the padding.

    Args:
        inputs: (N, L, C) float16, bfloat16 or float32, C a multiple of 8; rows may be part of wider ones.
        weight, bias: (C, W) with W from 2 to 8, the last tap the token's own; optional (C,); any float type.
        activation: "none" or "silu".
        initial_state: (N, W - 1, C) in the inputs' type, the inputs before the first token (default: zeros).
        return_state: also return the last W - 1 inputs, for `causal_conv1d_step` or the next piece of the sequences.

    Returns:
        (N, L, C) in the inputs' type, or that and the state, which has no history.  No gradients pass through states.
    """
    result = native.call("causal_conv1d", inputs, weight, bias, activation, initial_state, return_state)
    if result is not NotImplemented:
        return result
    refuse_forward_derivatives(inputs, weight, bias, initial_state)
    refuse_state_gradients(initial_state)
    y, state = causal_conv1d_forward(inputs, weight, bias, activation, initial_state, bool(return_state))
    return (y, state) if return_state else y


@torch.library.custom_op("spio::causal_conv1d_step", mutates_args=("out_state",))
def causal_conv1d_step_op(
    inputs: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], activation: str,
    out_state: torch.Tensor,
) -> torch.Tensor:  # fmt: skip
    """The outputs of one token a sequence; the last W - 1 inputs go to `out_state`, which may be `state`."""
    _check("causal_conv1d_step", inputs, 2, weight, bias, activation, state)
    check_out_state("causal_conv1d_step", state, out_state, inputs)
    require_gpu("causal_conv1d_step", inputs)
    assert state.data_ptr() % 16 == 0 and out_state.data_ptr() % 16 == 0, "states must start on 16 bytes"
    n, c = inputs.shape
    x, row = rows_of(inputs, 8)
    out = torch.empty((n, c), dtype=x.dtype, device=x.device)
    if n == 0:
        return out
    weight, bias = _filters(weight, bias)
    kernel = causal_conv1d_step_kernel_factory.get_kernel(_params(x, weight, activation), x.device)
    arguments = Arguments(STRUCT, x=x, weight=weight, bias=bias, before=state, out=out, after=out_state, tokens=1, channels=c,
                          sequences=n, slice=1, x_row=row)  # fmt: skip
    kernel.launch_structure(divup(n * (c // 8), 64), arguments)
    return out


@causal_conv1d_step_op.register_fake
def _step_fake(inputs, state, weight, bias, activation, out_state):
    _check("causal_conv1d_step", inputs, 2, weight, bias, activation, state)
    return inputs.new_empty(tuple(inputs.shape))


def causal_conv1d_step(
    inputs: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
    activation: str = "none", out_state: Optional[torch.Tensor] = None,
) -> torch.Tensor:  # fmt: skip
    """`causal_conv1d` of the next token of every sequence, without gradients.

    Args:
        inputs: (N, C).
        state: (N, W - 1, C) in the inputs' type, without gaps: the inputs before.
        weight, bias, activation: as in `causal_conv1d`.
        out_state: where the state behind the token goes; default: in place of `state`.

    Returns:
        (N, C) in the inputs' type.
    """
    out_state = state if out_state is None else out_state
    refuse_state_gradients(out_state)
    y = native.call("causal_conv1d_step", inputs, state, weight, bias, activation, out_state)
    if y is not NotImplemented:
        return y
    refuse_forward_derivatives(inputs, state, weight, bias, out_state)
    refuse_inference_state(out_state)
    with torch.no_grad():
        return causal_conv1d_step_op(inputs, state, weight, bias, activation, out_state)
