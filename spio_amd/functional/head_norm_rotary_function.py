"""`spio::head_norm_rotary_forward` and its backward: rotation of the heads of queries and keys by their positions, with or
without a norm of every head before it, in one pass over both tensors.

    xhat = x rsqrt(mean over the head of x^2 + eps),  n = xhat weight          (`rotary`: n = x)
    angle = position frequencies[i]
    the i-th pair (n1, n2) of a head becomes scale (n1 cos - n2 sin, n2 cos + n1 sin)

Pair i is the channels (2i, 2i + 1) of a head with `interleaved`, else (i, pairs + i); channels behind the pairs stay as they
are.  Angles are taken in float64 and there is no table of them: one is off by position * frequency * 2^-52 radians, and by 2^-24
turns, so that positions have no bound in practice.  Everything else is float32; the sum of a head's squares has to stay below
its largest number (3.4e38).

The reference has no such operators; their siblings here are the norms.
"""

import math
from typing import Optional, Tuple

import torch

from .. import native
from ..kernels.group_norm_2d_kernel import DTYPES
from ..kernels.head_norm_rotary_kernel import (
    MAX_HEAD,
    HeadNormRotaryParams,
    grid_of,
    head_norm_rotary_bwd_kernel_factory,
    head_norm_rotary_kernel_factory,
    head_norm_rotary_sums_kernel_factory,
    parts_of,
)
from ..kernels.token_args import Arguments
from ..util.math import divup
from .group_norm_2d_function import aligned, refuse_forward_derivatives
from .token_rows import check_parameters, check_tokens, require_gpu, vector

STRUCT = "SpioRotaryArgs"
SUM_COLUMNS = 32  # of a workgroup that adds up partial sums


def _check(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, scale):
    what = "head_norm_rotary"
    assert q.dim() == 4 and k.dim() == 4, "queries and keys are [sequences, tokens, heads, channels]"
    assert q.shape[:2] == k.shape[:2] and q.shape[3] == k.shape[3], "queries and keys must have the same tokens and channels"
    d = q.shape[3]
    assert d % 8 == 0 and 8 <= d <= MAX_HEAD, f"a head has a multiple of 8 channels, up to {MAX_HEAD}"
    check_tokens(what, q=q, k=k)
    check_parameters(what, q, q_weight=(q_weight, (d,)), k_weight=(k_weight, (d,)))
    assert (q_weight is None) == (k_weight is None), "weights of both norms or of none"
    assert q_weight is None or 0 < eps < float("inf"), "eps must be positive and finite"
    assert abs(scale) <= torch.finfo(torch.float32).max, "scale must be a finite float32 number"
    assert frequencies.dim() == 1 and frequencies.dtype == torch.float64, "frequencies are float64 [pairs]"
    pairs = frequencies.shape[0]
    assert 0 < pairs and 2 * pairs <= d, "a head has two channels for every frequency"
    assert interleaved or pairs % 8 == 0, "pairs of both halves come in multiples of 8"
    assert positions.dtype in (torch.int32, torch.int64), "positions are int32 or int64"
    n, l = q.shape[:2]
    assert tuple(positions.shape) in ((l,), (n, l)), f"positions must be {[l]} or {[n, l]}"
    assert n * l * max(q.shape[2], k.shape[2]) < 1 << 31, "fewer than 2^31 heads"
    assert positions.device == q.device == frequencies.device, "positions and frequencies must be on the queries' device"


def _heads_of(t):
    """[sequences, tokens, heads, channels] as equally distant rows of equally distant heads that start on 16 bytes: the tensor
    or a copy without gaps; the distances in values."""
    n, l, h, d = t.shape
    s = t.stride()
    row = s[1] if l != 1 else s[0] if n != 1 else h * d
    head = s[2] if h != 1 else d
    even = n == 1 or l == 1 or s[0] == l * s[1]
    size = t.element_size()
    if even and s[3] == 1 and t.data_ptr() % 16 == row * size % 16 == head * size % 16 == 0:
        return t, row, head
    return t.clone(memory_format=torch.contiguous_format), h * d, d


def _fields(q, k, positions, frequencies, eps, scale):
    n, l, h, d = q.shape
    return dict(positions=positions.contiguous(), frequencies=frequencies.contiguous(), tokens=n * l, q_heads=h,
                k_heads=k.shape[2], pairs=frequencies.shape[0], wide_positions=positions.dtype == torch.int64,
                position_tokens=positions.numel(), eps=eps, scale=scale)  # fmt: skip


def _weight(t):
    return None if t is None else aligned(vector(t))


def _params(q, norm, interleaved):
    return HeadNormRotaryParams(q.shape[3], DTYPES[q.dtype], norm, bool(interleaved))


@torch.library.custom_op("spio::head_norm_rotary_forward", mutates_args=())
def head_norm_rotary_forward(
    q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
    positions: torch.Tensor, frequencies: torch.Tensor, eps: float, interleaved: bool, scale: float,
) -> Tuple[torch.Tensor, torch.Tensor]:  # fmt: skip
    """(queries, keys); without weights there is no norm."""
    _check(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, scale)
    require_gpu("head_norm_rotary", q)
    outputs = [torch.empty(tuple(t.shape), dtype=t.dtype, device=t.device) for t in (q, k)]
    tokens, heads, d = q.shape[0] * q.shape[1], max(q.shape[2], k.shape[2]), q.shape[3]
    if tokens * heads == 0:
        return tuple(outputs)
    (qx, q_row, q_head), (kx, k_row, k_head) = _heads_of(q), _heads_of(k)
    norm = q_weight is not None
    parts = parts_of(tokens, heads, d, norm)
    arguments = Arguments(STRUCT, **_fields(q, k, positions, frequencies, eps, scale), q=qx, k=kx, q_row=q_row, q_head=q_head,
                          k_row=k_row, k_head=k_head, q_weight=_weight(q_weight), k_weight=_weight(k_weight), q_out=outputs[0],
                          k_out=outputs[1], parts=parts)  # fmt: skip
    kernel = head_norm_rotary_kernel_factory.get_kernel(_params(q, norm, interleaved), q.device)
    kernel.launch_structure(grid_of(tokens, parts, d, norm, False), arguments)
    return tuple(outputs)


@head_norm_rotary_forward.register_fake
def _forward_fake(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, scale):
    _check(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, scale)
    return q.new_empty(tuple(q.shape)), k.new_empty(tuple(k.shape))


@torch.library.custom_op("spio::head_norm_rotary_backward", mutates_args=())
def head_norm_rotary_backward(
    grad_q: torch.Tensor, grad_k: torch.Tensor, q: Optional[torch.Tensor], k: Optional[torch.Tensor],
    q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor,
    eps: float, interleaved: bool, scale: float,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:  # fmt: skip
    """(gradients of queries and keys, float32 [2, channels]: those of the weights, empty without).  Without weights the
    inputs are not needed."""
    norm = q_weight is not None
    _check(grad_q, grad_k, q_weight, k_weight, positions, frequencies, eps, interleaved, scale)
    require_gpu("head_norm_rotary", grad_q)
    outputs = [torch.empty(tuple(t.shape), dtype=t.dtype, device=t.device) for t in (grad_q, grad_k)]
    tokens, heads, d = grad_q.shape[0] * grad_q.shape[1], max(grad_q.shape[2], grad_k.shape[2]), grad_q.shape[3]
    sums = torch.empty((2, d) if norm else (0,), dtype=torch.float32, device=grad_q.device)
    if tokens * heads == 0:
        return (*outputs, sums.zero_())
    fields = _fields(grad_q, grad_k, positions, frequencies, eps, scale)
    parts = parts_of(tokens, heads, d, norm)
    grid = grid_of(tokens, parts, d, norm, norm)
    if norm:
        assert q.shape == grad_q.shape and k.shape == grad_k.shape and q.dtype == k.dtype == grad_q.dtype, "inputs of another norm"
        assert q.device == k.device == grad_q.device
        for name, t in (("q", q), ("k", k)):
            fields[name], fields[name + "_row"], fields[name + "_head"] = _heads_of(t)
        fields["partials"] = torch.empty((grid, 2, d), dtype=torch.float32, device=grad_q.device)
        fields["dq_weight"], fields["dk_weight"] = sums
    fields.update(dq=aligned(grad_q.contiguous()), dk=aligned(grad_k.contiguous()), q_weight=_weight(q_weight),
                  k_weight=_weight(k_weight), q_out=outputs[0], k_out=outputs[1])  # fmt: skip
    params = _params(grad_q, norm, interleaved)
    main = head_norm_rotary_bwd_kernel_factory.get_kernel(params, grad_q.device)
    main.launch_structure(grid, Arguments(STRUCT, **fields, parts=parts))
    if norm:
        second = head_norm_rotary_sums_kernel_factory.get_kernel(params, grad_q.device)
        second.launch_structure(divup(2 * d, SUM_COLUMNS), Arguments(STRUCT, **fields, parts=grid))
    return (*outputs, sums)


@head_norm_rotary_backward.register_fake
def _backward_fake(grad_q, grad_k, q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, scale):
    d = grad_q.shape[3]
    return (grad_q.new_empty(tuple(grad_q.shape)), grad_k.new_empty(tuple(grad_k.shape)),
            grad_q.new_empty((2, d) if q_weight is not None else (0,), dtype=torch.float32))  # fmt: skip


def head_norm_rotary_gradients(grad_q, grad_k, q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, scale, needs):
    """Gradients for q, k, q_weight and k_weight in the types of these, None where not needed.  Without a norm q and k are
    not needed."""
    refuse_forward_derivatives(grad_q, grad_k, q, k, q_weight, k_weight)
    norm = q_weight is not None
    dq, dk, sums = head_norm_rotary_backward(grad_q, grad_k, q, k, q_weight, k_weight, positions, frequencies, eps, interleaved,
                                             scale)  # fmt: skip
    return (
        dq if needs[0] else None,
        dk if needs[1] else None,
        sums[0].to(q_weight.dtype) if norm and needs[2] else None,
        sums[1].to(k_weight.dtype) if norm and needs[3] else None,
    )


def _setup_context(ctx, inputs, output):
    q, k, *rest, eps, interleaved, scale = inputs
    ctx.set_materialize_grads(False)
    norm = rest[0] is not None
    ctx.save_for_backward(q if norm else None, k if norm else None, *rest)
    ctx.numbers = (eps, interleaved, scale)
    ctx.shapes = (tuple(q.shape), tuple(k.shape))


def _backward(ctx, grad_q, grad_k):
    if grad_q is None and grad_k is None:
        return (None,) * 9
    grad_q = grad_k.new_zeros(ctx.shapes[0]) if grad_q is None else grad_q
    grad_k = grad_q.new_zeros(ctx.shapes[1]) if grad_k is None else grad_k
    return (*head_norm_rotary_gradients(grad_q, grad_k, *ctx.saved_tensors, *ctx.numbers, ctx.needs_input_grad), *(None,) * 5)


head_norm_rotary_forward.register_autograd(_backward, setup_context=_setup_context)


def _call(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, scale):
    result = native.call("head_norm_rotary", q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, scale)
    if result is not NotImplemented:
        return result
    refuse_forward_derivatives(q, k, q_weight, k_weight)
    if torch.is_grad_enabled() and frequencies.requires_grad:
        raise RuntimeError("no gradients pass to frequencies: detach them")
    return head_norm_rotary_forward(q, k, q_weight, k_weight, positions, frequencies, float(eps), bool(interleaved), float(scale))


def rotary(
    q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, interleaved: bool = False,
    scale: float = 1.0,
) -> Tuple[torch.Tensor, torch.Tensor]:  # fmt: skip
    """Queries and keys turned by their positions.

    Args:
        q, k: (N, L, heads, D) float16, bfloat16 or float32 of one type, each with its own number of heads; D a multiple of 8
            up to 256; rows and heads may be part of wider ones.
        positions: (L,) or (N, L) int32 or int64.
        frequencies: (pairs,) float64, radians a position (`rotary_frequencies`); 2 * pairs channels of a head are turned.
            Without `interleaved` a multiple of 8.
        interleaved: pairs are neighbouring channels instead of one of each half.
        scale: factor of the turned channels, a finite float32 number.

    Returns:
        Queries and keys of the same shapes and type, without gaps.
    """
    return _call(q, k, None, None, positions, frequencies, 1.0, interleaved, scale)


def head_norm_rotary(
    q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, positions: torch.Tensor,
    frequencies: torch.Tensor, eps: float = 1e-6, interleaved: bool = False, scale: float = 1.0,
) -> Tuple[torch.Tensor, torch.Tensor]:  # fmt: skip
    """`rotary` of heads that are divided by the root of their mean square and multiplied by a weight first.

    Args:
        q_weight, k_weight: (D,), any float type.
        eps: positive and finite, added to the mean square; below 2^-126 it counts as that.
        (the others as in `rotary`)
    """
    assert q_weight is not None and k_weight is not None, "head_norm_rotary takes weights of both norms"
    return _call(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, scale)


def rotary_frequencies(
    channels: int, base: float = 10000.0, factor: float = 1.0, method: str = "linear", trained_tokens: int = 4096,
    slow_turns: float = 1.0, fast_turns: float = 32.0, device=None,
) -> torch.Tensor:  # fmt: skip
    """Frequencies of `channels` / 2 pairs, float64: base^(-2i / channels) radians a position, scaled for contexts that are
    `factor` times as long as the trained ones.

    Args:
        channels: even; how many channels of a head are turned.
        method: "linear": all frequencies divided by the factor; "base": a larger base, by which the slowest one is divided
            by the factor and the fastest stays; "ramp": frequencies that make `fast_turns` turns or more in `trained_tokens`
            positions stay, those that make `slow_turns` or fewer are divided by the factor, and in between the share of the
            two goes linearly with the turns.  (What such methods multiply the turned channels with is `scale`.)
    """
    if channels < 2 or channels % 2 or base <= 1 or factor < 1:
        raise ValueError("channels must be even and positive, base above 1, factor at least 1")
    exponents = torch.arange(channels // 2, dtype=torch.float64) * (2.0 / channels)
    if method == "base":
        if channels > 2:
            base *= factor ** (channels / (channels - 2))
        frequencies = base**-exponents
    elif method == "linear":
        frequencies = base**-exponents / factor
    elif method == "ramp":
        if not 0 <= slow_turns < fast_turns or trained_tokens < 1:
            raise ValueError("slow_turns must be below fast_turns, trained_tokens positive")
        frequencies = base**-exponents
        turns = frequencies * (trained_tokens / (2 * math.pi))
        stay = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
        frequencies = frequencies * (stay + (1 - stay) / factor)
    else:
        raise ValueError(f"method must be 'linear', 'base' or 'ramp', not {method!r}")
    return frequencies.to(device)
