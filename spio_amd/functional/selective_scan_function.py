"""`spio::selective_scan_forward`, its backward and `spio::selective_scan_step`: the recurrence of a state-space layer whose
rates follow its input, over [sequences, tokens, channels] tensors.

    dl   = softplus(delta[t] + delta_bias)                     (without delta_softplus: the sum itself)
    h    = exp(dl A) h + dl inputs[t] B[t]                     h [channels, states] of a sequence, in float32
    y    = sum over states of C[t] h + D inputs[t];            out[t] = y silu(gate[t]), or y without a gate

The gradients are those of these formulas; the backward pass goes through the tokens from the last to the first and computes
the states between those that the forward pass kept (every few tokens) again.  All arithmetic is float32.

The reference has no such operator; its sibling here is `causal_conv1d`, which precedes it in a layer.
"""

from typing import Optional, Tuple, Union

import torch

from .. import native
from ..kernels.group_norm_2d_kernel import DTYPES
from ..kernels.selective_scan_kernel import (
    LANES,
    MAX_STATES,
    SelectiveScanParams,
    chunk_tokens,
    selective_scan_bwd_kernel_factory,
    selective_scan_ends_bwd_kernel_factory,
    selective_scan_ends_kernel_factory,
    selective_scan_join_bwd_kernel_factory,
    selective_scan_join_kernel_factory,
    selective_scan_kernel_factory,
    selective_scan_step_kernel_factory,
    selective_scan_sums_kernel_factory,
    tile_tokens,
)
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
    vector,
)

STRUCT = "SpioScanArgs"
SUM_COLUMNS = 32  # of a workgroup that adds up partial sums


def _check(what, inputs, dims, delta, A, B, C, D, gate, delta_bias, state):
    assert inputs.dim() == dims, f"{what} takes {'[sequences, tokens, channels]' if dims == 3 else '[sequences, channels]'}"
    c = inputs.shape[-1]
    assert 0 < c < 1 << 24, f"{what} takes from one to 2^24 - 1 channels"
    assert inputs.shape[-2] < 1 << 30, f"{what} takes fewer than 2^30 tokens of a sequence"
    assert A.dim() == 2 and 1 <= A.shape[1] <= MAX_STATES, f"A is [channels, 1..{MAX_STATES}]"
    s = A.shape[1]
    check_tokens(what, inputs=inputs, delta=delta, B=B, C=C, gate=gate)
    for name, t in (("delta", delta), ("gate", gate)):
        assert t is None or t.shape == inputs.shape, f"{what}: {name} must have the inputs' shape"
    for name, t in (("B", B), ("C", C)):
        assert tuple(t.shape) == (*inputs.shape[:-1], s), f"{what}: {name} must be {[*inputs.shape[:-1], s]}"
    check_parameters(what, inputs, A=(A, (c, s)), D=(D, (c,)), delta_bias=(delta_bias, (c,)))
    if state is not None:
        assert tuple(state.shape) == (inputs.shape[0], c, s) and state.dtype == torch.float32, (
            "a state is [sequences, channels, states] in float32")  # fmt: skip
        assert state.device == inputs.device, f"{what}: the state must be on the inputs' device"


def _rows(inputs, delta, B, C, gate):
    """Fields of the structure for the tensors that may be rows of wider ones."""
    fields = {}
    for name, row, t in (("u", "u_row", inputs), ("delta", "delta_row", delta), ("B", "b_row", B), ("C", "c_row", C),
                         ("gate", "gate_row", gate)):  # fmt: skip
        fields[name], fields[row] = rows_of(None if t is None else t.detach())
    return fields


@torch.library.custom_op("spio::selective_scan_forward", mutates_args=())
def selective_scan_forward(
    inputs: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: Optional[torch.Tensor],
    gate: Optional[torch.Tensor], delta_bias: Optional[torch.Tensor], delta_softplus: bool,
    initial_state: Optional[torch.Tensor], keep_state: bool, keep_tiles: bool,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:  # fmt: skip
    """(outputs, state behind the last token, states before every tile of tokens); the last two are empty unless kept."""
    _check("selective_scan", inputs, 3, delta, A, B, C, D, gate, delta_bias, initial_state)
    require_gpu("selective_scan", inputs)
    n, l, c = inputs.shape
    s = A.shape[1]
    f32 = dict(dtype=torch.float32, device=inputs.device)
    out = torch.empty((n, l, c), dtype=inputs.dtype, device=inputs.device)
    after = torch.empty((n, c, s) if keep_state else (0,), **f32)
    kept = torch.empty((n, divup(l, tile_tokens(s)), s, c) if keep_tiles else (0,), **f32)
    if out.numel() == 0:
        if after.numel():
            after.copy_(initial_state) if initial_state is not None else after.zero_()
        return out, after, kept
    dtype, gated, softplus = DTYPES[inputs.dtype], gate is not None, bool(delta_softplus)
    chunk = chunk_tokens(l, c, n, False)
    chunks, blocks = divup(l, chunk), divup(c, LANES)
    ends = torch.empty((n, chunks, s + 1, c), **f32) if chunks > 1 else None
    arguments = Arguments(
        STRUCT, **_rows(inputs, delta, B, C, gate), A=vector(A), D=vector(D), bias=vector(delta_bias),
        before=None if initial_state is None else initial_state.contiguous(), out=out, after=after if keep_state else None,
        kept=kept if keep_tiles else None, ends=ends, tokens=l, channels=c, chunk=chunk, sequences=n)  # fmt: skip
    grid = n * chunks * blocks
    if chunks > 1:
        ends_kernel = selective_scan_ends_kernel_factory.get_kernel(SelectiveScanParams(s, dtype, False, softplus), inputs.device)
        ends_kernel.launch_structure(grid, arguments)
        join = selective_scan_join_kernel_factory.get_kernel(SelectiveScanParams(s, dtype), inputs.device)
        join.launch_structure(n * s * blocks, arguments)
    kernel = selective_scan_kernel_factory.get_kernel(SelectiveScanParams(s, dtype, gated, softplus, bool(keep_tiles)), inputs.device)
    kernel.launch_structure(grid, arguments)
    return out, after, kept


@selective_scan_forward.register_fake
def _forward_fake(inputs, delta, A, B, C, D, gate, delta_bias, delta_softplus, initial_state, keep_state, keep_tiles):
    _check("selective_scan", inputs, 3, delta, A, B, C, D, gate, delta_bias, initial_state)
    n, l, c = inputs.shape
    s = A.shape[1]
    return (inputs.new_empty((n, l, c)), inputs.new_empty((n, c, s) if keep_state else (0,), dtype=torch.float32),
            inputs.new_empty((n, divup(l, tile_tokens(s)), s, c) if keep_tiles else (0,), dtype=torch.float32))  # fmt: skip


@torch.library.custom_op("spio::selective_scan_backward", mutates_args=())
def selective_scan_backward(
    grad_output: torch.Tensor, inputs: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
    D: Optional[torch.Tensor], gate: Optional[torch.Tensor], delta_bias: Optional[torch.Tensor], delta_softplus: bool,
    kept: torch.Tensor,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:  # fmt: skip
    """(grad_inputs, grad_delta, grad_B, grad_C, grad_gate (empty without a gate), float32 [C * S + 2 C]: grad_A, grad_D,
    grad_delta_bias)."""
    _check("selective_scan", inputs, 3, delta, A, B, C, D, gate, delta_bias, None)
    assert grad_output.shape == inputs.shape and grad_output.dtype == inputs.dtype and grad_output.device == inputs.device
    require_gpu("selective_scan", inputs)
    n, l, c = inputs.shape
    s = A.shape[1]
    assert tuple(kept.shape) == (n, divup(l, tile_tokens(s)), s, c) and kept.dtype == torch.float32, "states of another scan"
    assert kept.device == inputs.device
    f32 = dict(dtype=torch.float32, device=inputs.device)
    du, ddelta = (torch.empty((n, l, c), dtype=inputs.dtype, device=inputs.device) for _ in range(2))
    dgate = torch.empty((n, l, c) if gate is not None else (0,), dtype=inputs.dtype, device=inputs.device)
    dB, dC = (torch.empty((n, l, s), dtype=inputs.dtype, device=inputs.device) for _ in range(2))
    sums = torch.empty((c * (s + 2),), **f32)
    if du.numel() == 0:
        return du, ddelta, dB, dC, dgate, sums.zero_()
    dtype, gated, softplus = DTYPES[inputs.dtype], gate is not None, bool(delta_softplus)
    chunk = chunk_tokens(l, c, n, True)
    chunks, blocks = divup(l, chunk), divup(c, LANES)
    arguments = Arguments(
        STRUCT, **_rows(inputs, delta, B, C, gate), dout=grad_output.contiguous(), A=vector(A), D=vector(D),
        bias=vector(delta_bias), kept=kept.contiguous(), ends=torch.empty((n, chunks, s + 1, c), **f32) if chunks > 1 else None,
        du=du, ddelta=ddelta, dgate=dgate if gate is not None else None,
        token_sums=torch.empty((n, l, blocks, 2 * s), **f32), channel_sums=torch.empty((n, chunks, s + 2, c), **f32),
        dB=dB, dC=dC, dA=sums, dD=sums[c * s :], dbias=sums[c * (s + 1) :], tokens=l, channels=c, chunk=chunk, sequences=n)  # fmt: skip
    params = SelectiveScanParams(s, dtype, gated, softplus)
    if chunks > 1:
        selective_scan_ends_bwd_kernel_factory.get_kernel(params, inputs.device).launch_structure(n * chunks * blocks, arguments)
        join = selective_scan_join_bwd_kernel_factory.get_kernel(SelectiveScanParams(s, dtype), inputs.device)
        join.launch_structure(n * s * blocks, arguments)
    selective_scan_bwd_kernel_factory.get_kernel(params, inputs.device).launch_structure(n * chunks * blocks, arguments)
    grid = divup(n * l * 2 * s, 256) + divup((s + 2) * c, SUM_COLUMNS)
    selective_scan_sums_kernel_factory.get_kernel(SelectiveScanParams(s, dtype), inputs.device).launch_structure(grid, arguments)
    return du, ddelta, dB, dC, dgate, sums


@selective_scan_backward.register_fake
def _backward_fake(grad_output, inputs, delta, A, B, C, D, gate, delta_bias, delta_softplus, kept):
    shape = tuple(inputs.shape)
    rows = (*shape[:-1], A.shape[1])
    return (inputs.new_empty(shape), inputs.new_empty(shape), inputs.new_empty(rows), inputs.new_empty(rows),
            inputs.new_empty(shape if gate is not None else (0,)),
            inputs.new_empty((A.shape[0] * (A.shape[1] + 2),), dtype=torch.float32))  # fmt: skip


def selective_scan_gradients(grad_output, inputs, delta, A, B, C, D, gate, delta_bias, delta_softplus, kept, needs):
    """Gradients of selective_scan for inputs, delta, A, B, C, D, gate and delta_bias in the types of these, None where
    not needed."""
    refuse_forward_derivatives(grad_output, inputs, delta, A, B, C, D, gate, delta_bias)
    du, ddelta, dB, dC, dgate, sums = selective_scan_backward(grad_output, inputs, delta, A, B, C, D, gate, delta_bias,
                                                              delta_softplus, kept)  # fmt: skip
    c, s = A.shape
    return (
        du if needs[0] else None,
        ddelta if needs[1] else None,
        sums[: c * s].view(c, s).to(A.dtype) if needs[2] else None,
        dB if needs[3] else None,
        dC if needs[4] else None,
        sums[c * s : c * (s + 1)].to(D.dtype) if D is not None and needs[5] else None,
        dgate if gate is not None and needs[6] else None,
        sums[c * (s + 1) :].to(delta_bias.dtype) if delta_bias is not None and needs[7] else None,
    )


def _setup_context(ctx, inputs, output):
    *tensors, delta_softplus, _, _, _ = inputs
    _, after, kept = output
    ctx.mark_non_differentiable(after, kept)
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(*tensors, kept)
    ctx.delta_softplus = delta_softplus


def _backward(ctx, grad_output, *_unused):
    if grad_output is None:
        return (None,) * 12
    *tensors, kept = ctx.saved_tensors
    return (*selective_scan_gradients(grad_output, *tensors, ctx.delta_softplus, kept, ctx.needs_input_grad), *(None,) * 4)


selective_scan_forward.register_autograd(_backward, setup_context=_setup_context)


def selective_scan(
    inputs: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
    D: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, delta_bias: Optional[torch.Tensor] = None,
    delta_softplus: bool = False, initial_state: Optional[torch.Tensor] = None, return_state: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:  # fmt: skip
    """The selective scan of (N, L, C) inputs with S states a channel.

    A token whose time step is zero (delta of minus infinity with softplus) leaves the states as they are: so sequences of
    different lengths are padded, in front or behind.  Its inputs and B, with gradients also C, gate and grad_output, have to be
    finite: zero times what is not is NaN.  With gradients the states before every fourth token (eighth with up to eight states)
    are kept, in float32.

    Args:
        inputs, delta, gate: (N, L, C) float16, bfloat16 or float32, all of one type; rows may be part of wider ones.
            `gate` is optional.  C below 2^24.
        A: (C, S), S up to 32; negative where the states are to decay.  D, delta_bias: optional (C,).  Any float type.
        B, C: (N, L, S) in the inputs' type, the same for all channels.
        delta_softplus: softplus of delta (with its bias) instead of that itself.
        initial_state: (N, C, S) float32, the states before the first token (default: zeros).
        return_state: also return the states behind the last token, for `selective_scan_step` or the next piece.

    Returns:
        (N, L, C) in the inputs' type, or that and the state, which has no history.  No gradients pass through states.
    """
    result = native.call("selective_scan", inputs, delta, A, B, C, D, gate, delta_bias, delta_softplus, initial_state,
                         return_state)  # fmt: skip
    if result is not NotImplemented:
        return result
    tensors = (inputs, delta, A, B, C, D, gate, delta_bias)
    refuse_forward_derivatives(*tensors, initial_state)
    refuse_state_gradients(initial_state)
    record = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
    y, state, _ = selective_scan_forward(*tensors, bool(delta_softplus), initial_state, bool(return_state), record)
    return (y, state) if return_state else y


@torch.library.custom_op("spio::selective_scan_step", mutates_args=("out_state",))
def selective_scan_step_op(
    inputs: torch.Tensor, state: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
    D: Optional[torch.Tensor], gate: Optional[torch.Tensor], delta_bias: Optional[torch.Tensor], delta_softplus: bool,
    out_state: torch.Tensor,
) -> torch.Tensor:  # fmt: skip
    """The outputs of one token a sequence; the states behind it go to `out_state`, which may be `state`."""
    _check("selective_scan_step", inputs, 2, delta, A, B, C, D, gate, delta_bias, state)
    check_out_state("selective_scan_step", state, out_state, inputs, delta, B, C, gate)
    require_gpu("selective_scan_step", inputs)
    assert state.data_ptr() % 16 == 0 and out_state.data_ptr() % 16 == 0, "states must start on 16 bytes"
    n, c = inputs.shape
    s = A.shape[1]
    out = torch.empty((n, c), dtype=inputs.dtype, device=inputs.device)
    if n == 0:
        return out
    params = SelectiveScanParams(s, DTYPES[inputs.dtype], gate is not None, bool(delta_softplus))
    kernel = selective_scan_step_kernel_factory.get_kernel(params, inputs.device)
    arguments = Arguments(STRUCT, **_rows(inputs, delta, B, C, gate), A=aligned(vector(A)), D=vector(D), bias=vector(delta_bias),
                          before=state, out=out, after=out_state, tokens=1, channels=c, chunk=1, sequences=n)  # fmt: skip
    lanes = 1 if s <= 4 else 2 if s <= 8 else 4 if s <= 16 else 8
    kernel.launch_structure(divup(n * c * lanes, 256), arguments)
    return out


@selective_scan_step_op.register_fake
def _step_fake(inputs, state, delta, A, B, C, D, gate, delta_bias, delta_softplus, out_state):
    _check("selective_scan_step", inputs, 2, delta, A, B, C, D, gate, delta_bias, state)
    return inputs.new_empty(tuple(inputs.shape))


def selective_scan_step(
    inputs: torch.Tensor, state: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
    D: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, delta_bias: Optional[torch.Tensor] = None,
    delta_softplus: bool = False, out_state: Optional[torch.Tensor] = None,
) -> torch.Tensor:  # fmt: skip
    """`selective_scan` of the next token of every sequence, without gradients.

    Args:
        inputs, delta, gate: (N, C).  B, C: (N, S).  A, D, delta_bias, delta_softplus: as in `selective_scan`.
        state: (N, C, S) float32 without gaps, the states before the token.
        out_state: where the states behind it go; default: in place of `state`.

    Returns:
        (N, C) in the inputs' type.
    """
    out_state = state if out_state is None else out_state
    refuse_state_gradients(out_state)
    y = native.call("selective_scan_step", inputs, state, delta, A, B, C, D, gate, delta_bias, delta_softplus, out_state)
    if y is not NotImplemented:
        return y
    refuse_forward_derivatives(inputs, state, delta, A, B, C, D, gate, delta_bias, out_state)
    refuse_inference_state(out_state)
    with torch.no_grad():
        return selective_scan_step_op(inputs, state, delta, A, B, C, D, gate, delta_bias, bool(delta_softplus), out_state)
