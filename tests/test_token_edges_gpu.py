"""The operators over sequences of tokens at their edges on the GPU: derivatives that are refused, inference mode, padded
sequences, rates and values that are not finite, hooks on saved tensors, offsets that pass 31 bits."""

import pytest
import torch
from torch.autograd import forward_ad

from spio_amd import native
from spio_amd.functional import (
    causal_conv1d,
    causal_conv1d_step,
    head_norm_rotary,
    rotary,
    rotary_frequencies,
    selective_scan,
    selective_scan_step,
)
from spio_amd.layers import HeadNormRotary, SelectiveScan
from spio_amd.native import Bypass
from tests import token_reference as ref

pytestmark = pytest.mark.gpu
HALF, BF16, FLOAT = torch.float16, torch.bfloat16, torch.float32


def _normal(*shape, dtype=FLOAT, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _calls():
    """Name: (operator of the tensors that have gradients, these tensors)."""
    frequencies, positions = rotary_frequencies(16, device="cuda"), torch.arange(6, device="cuda")
    x, h = _normal(2, 6, 16), _normal(2, 6, 3, 16, seed=1)
    A = -_normal(16, 4).abs()
    return {
        "conv": (lambda x, w: causal_conv1d(x, w, None, "silu"), [x, _normal(16, 4, seed=2)]),
        "scan": (lambda x, d, A: selective_scan(x, d, A, x[..., :4], x[..., 4:8], None, x, None, True), [x, _normal(2, 6, 16, seed=3), A]),
        "rotary": (lambda q: rotary(q, q[:, :, :1], positions, frequencies)[0], [h]),
        "norm": (lambda q, w: head_norm_rotary(q, q[:, :, :1], w, w, positions, frequencies)[0], [h, _normal(16, seed=4)]),
    }  # fmt: skip


class _Path:
    """The native or the Python call path."""

    def __init__(self, python):
        self.python = python

    def __enter__(self):
        self.held = Bypass() if self.python else None

    def __exit__(self, *_):
        if self.held:
            self.held.release()


NAMES = ("conv", "scan", "rotary", "norm")


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name, python):
    call, tensors = _calls()[name]
    with _Path(python):
        expected = call(*tensors)
        with forward_ad.dual_level():
            for i, t in enumerate(tensors):
                duals = [forward_ad.make_dual(u.clone(), torch.ones_like(u)) if i == k else u for k, u in enumerate(tensors)]
                with pytest.raises(NotImplementedError):
                    call(*duals)
            assert torch.equal(call(*tensors), expected)
            leaves = [t.clone().requires_grad_() for t in tensors]
            y = call(*leaves)
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(y, leaves, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives_are_refused(name, python):
    call, tensors = _calls()[name]
    with _Path(python):
        leaves = [t.clone().requires_grad_() for t in tensors]
        first = torch.autograd.grad(call(*leaves), leaves, torch.ones_like(call(*tensors)), create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(first[0].square().sum(), leaves)


@pytest.mark.parametrize("name", NAMES)
def test_hooks_on_saved_tensors(name):
    """What hooks hand back with other strides, or from the host, is taken as it is; a gradient may be broadcast."""
    call, tensors = _calls()[name]
    leaves = [t.clone().requires_grad_() for t in tensors]
    expected = torch.autograd.grad(call(*leaves).sum(), leaves)

    def strided(t):
        return t.detach().transpose(0, -1).contiguous().transpose(0, -1) if t.dim() > 1 else t.detach().clone()

    with torch.autograd.graph.saved_tensors_hooks(strided, lambda t: t):
        got = torch.autograd.grad(call(*leaves).sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, expected))
    with torch.autograd.graph.save_on_cpu():
        got = torch.autograd.grad(call(*leaves).sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, expected))


@pytest.mark.parametrize("python", [False, True])
def test_what_was_written_to_is_noticed(python):
    with _Path(python):
        state = torch.zeros(2, 16, 4, device="cuda")
        x, d = _normal(2, 6, 16), _normal(2, 6, 16, seed=3)
        A = -torch.ones(16, 4, device="cuda")
        leaf = state.clone().requires_grad_()
        squares = leaf.mul(1.0)
        y = squares.square()  # keeps `squares`
        with torch.no_grad():
            selective_scan_step(x[:, 0], squares.detach(), d[:, 0], A, x[:, 0, :4], x[:, 0, :4])
        with pytest.raises(RuntimeError):
            y.sum().backward()
        weight = _normal(16, 4).requires_grad_()
        before = torch.zeros(2, 3, 16, device="cuda")
        y = causal_conv1d(x, weight, None, "silu", before)
        causal_conv1d_step(x[:, 0], before, weight.detach())
        with pytest.raises(RuntimeError):
            y.sum().backward()


@pytest.mark.parametrize("python", [False, True])
def test_inference_mode(python):
    """Prompt and steps in inference mode, with states made there and outside; a state made there stays there."""
    w, A = _normal(16, 4), -_normal(16, 4).abs()
    x, d = _normal(2, 6, 16), _normal(2, 6, 16, seed=3)
    whole = causal_conv1d(x, w)
    scanned = selective_scan(x, d, A, x[..., :4], x[..., 4:8], delta_softplus=True)
    with _Path(python):
        with torch.inference_mode():
            y, state = causal_conv1d(x[:, :3], w, return_state=True)
            z, hidden = selective_scan(x[:, :3], d[:, :3], A, x[:, :3, :4], x[:, :3, 4:8], delta_softplus=True, return_state=True)
            for t in range(3, 6):
                torch.testing.assert_close(causal_conv1d_step(x[:, t], state, w), whole[:, t])
                got = selective_scan_step(x[:, t], hidden, d[:, t], A, x[:, t, :4], x[:, t, 4:8], delta_softplus=True)
                torch.testing.assert_close(got, scanned[:, t])
        with pytest.raises(RuntimeError):
            causal_conv1d_step(x[:, 0], state, w)
        normal = torch.zeros(2, 3, 16, device="cuda")
        with torch.inference_mode():
            causal_conv1d_step(x[:, 0], normal, w)
        assert torch.equal(normal[:, 2], x[:, 0])


def test_steps_of_inference_mode_take_the_native_path():
    x, w, A = _normal(2, 16), _normal(16, 4), -torch.ones(16, 4, device="cuda")
    with torch.inference_mode():
        state, hidden = torch.zeros(2, 3, 16, device="cuda"), torch.zeros(2, 16, 4, device="cuda")
        assert native.call("causal_conv1d_step", x, state, w, None, "none", state) is not NotImplemented
        rows = x[:, :4]
        assert native.call("selective_scan_step", x, hidden, x, A, rows, rows, None, None, None, True, hidden) is not NotImplemented
    assert native.call("causal_conv1d_step", x, state, w, None, "none", state) is NotImplemented


def test_padded_sequences():
    """Tokens whose time step is softplus of minus infinity leave the states as they are, in front of and behind the others."""
    n, l, c, s = 2, 200, 70, 5
    x, d, B, C = _normal(n, l, c), _normal(n, l, c, seed=1), _normal(n, l, s, seed=2), _normal(n, l, s, seed=3)
    A = -_normal(c, s, seed=4).abs()
    d[0, 150:] = d[1, :30] = -float("inf")
    whole, state = selective_scan(x, d, A, B, C, delta_softplus=True, return_state=True)
    for i, part in ((0, slice(0, 150)), (1, slice(30, l))):
        one = [t[i : i + 1, part] for t in (x, d)] + [A] + [t[i : i + 1, part] for t in (B, C)]
        y, h = selective_scan(*one, delta_softplus=True, return_state=True)
        expected = ref.scan(*one, None, None, None, True, None, None)
        for got in (y, whole[i : i + 1, part]):
            ref.check("y", got, *expected[0], 3 * l + 100)
        for got in (h, state[i : i + 1]):
            ref.check("state", got, *expected[1], 3 * l + 100)
    leaves = [t.clone().requires_grad_() for t in (x, d, A, B, C)]
    grads = torch.autograd.grad(selective_scan(*leaves, delta_softplus=True).sum(), leaves)
    assert all(g.isfinite().all() for g in grads) and not grads[0][0, 150:].any() and not grads[1][1, :30].any()


@pytest.mark.parametrize("l", [5, 300])  # a part of a tile; chunks
def test_rates_at_the_ends(l):
    """A rate of minus infinity forgets at once; a state of nothing stays so at a rate that grows past all numbers."""
    n, c, s = 1, 8, 3
    x, d, B, C = _normal(n, l, c), torch.full((n, l, c), 0.5, device="cuda"), _normal(n, l, s, seed=2), _normal(n, l, s, seed=3)
    A = torch.full((c, s), -float("inf"), device="cuda")
    A[1], A[2] = -3.4e38, 100.0
    x[..., 2] = 0.0
    leaves = [t.clone().requires_grad_() for t in (x, d, A, B, C)]
    y, state = selective_scan(*leaves, return_state=True)
    now = (0.5 * x.double() * (B.double() * C.double()).sum(-1, keepdim=True))
    size = 0.5 * x.double().abs() * (B.double() * C.double()).abs().sum(-1, keepdim=True)
    assert ((y.double() - now).abs() <= (2.0**-24 * 20) * size + 2.0**-126).all() and not y[..., 2].any() and not state[:, 2].any()
    du = torch.autograd.grad(y[..., :2].sum(), leaves)[0][..., :2]
    expected = 0.5 * (B.double() * C.double()).sum(-1, keepdim=True)
    size = 0.5 * (B.double() * C.double()).abs().sum(-1, keepdim=True)
    assert ((du.double() - expected).abs() <= (2.0**-24 * 20) * size + 2.0**-126).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_channels_behind_the_pairs_are_left_alone(interleaved, norm):
    """... also beside ones that are not finite."""
    q = _normal(1, 4, 2, 32)
    frequencies = rotary_frequencies(16, device="cuda")
    q[0, 1, 0, 20], q[0, 2, 1, 17] = float("inf"), float("nan")
    positions = torch.arange(4, device="cuda")
    if not norm:
        leaf = q.clone().requires_grad_()
        y = rotary(leaf, leaf[:, :, :0], positions, frequencies, interleaved)[0]
        assert y.detach()[..., 16:].eq(q[..., 16:]).logical_or(q[..., 16:].isnan()).all() and y[..., :16].isfinite().all()
        grad = torch.autograd.grad(y, leaf, q)[0]
        assert grad[..., 16:].eq(q[..., 16:]).logical_or(q[..., 16:].isnan()).all() and grad[..., :16].isfinite().all()
    else:
        w = torch.ones(32, device="cuda")
        y = head_norm_rotary(q, q[:, :, :0], w, w, positions, frequencies, interleaved=interleaved)[0]
        assert y[0, 0].isfinite().all() and y[0, 3].isfinite().all() and y[0, 1, 1].isfinite().all() and y[0, 2, 0].isfinite().all()


@pytest.mark.parametrize("eps", [1e-300, 1e-42, 2.0**-126, 1e300])
def test_smallest_and_largest_eps(eps):
    q = _normal(1, 3, 2, 16)
    q[0, 0] = 0.0
    w, positions, frequencies = torch.ones(16, device="cuda"), torch.arange(3, device="cuda"), rotary_frequencies(16, device="cuda")
    leaf = q.clone().requires_grad_()
    y = head_norm_rotary(leaf, q, w, w, positions, frequencies, eps)[0]
    grad = torch.autograd.grad(y.sum(), leaf)[0]
    assert not y[0, 0].any() and y.isfinite().all() and grad[0, 1:].isfinite().all()
    if eps < 1:
        expected = ref.rotary(q[:, 1:], w, positions[1:], frequencies, eps, False, 1.0, None)[0]
        ref.check("out", y[:, 1:], *expected, 16 + 60)


def test_layers_cast_and_made_without_memory():
    scan = SelectiveScan(16, states=4, device="cuda").half()
    state = scan.empty_state(2)
    x = _normal(2, 16, dtype=HALF)
    assert state.dtype == FLOAT and scan.step(x, state, x, x[:, :4], x[:, 4:8]).dtype == HALF
    norm = HeadNormRotary(32, rotated=16, factor=4.0, device="meta").to_empty(device="cuda")
    assert torch.equal(norm.frequencies, rotary_frequencies(16, factor=4.0, device="cuda")) and norm.half().frequencies.dtype == torch.float64


def _far(*shape):
    return torch.empty(*shape, dtype=BF16, device="cuda").normal_()


def test_convolution_past_31_bits():
    l, c = (1 << 21) + 3, 1024
    x, dy = _far(1, l, c).requires_grad_(), _far(1, l, c)
    w = _normal(c, 4).requires_grad_()
    y, state = causal_conv1d(x, w, None, "silu", return_state=True)
    dx = torch.autograd.grad(y, x, dy)[0]
    last = slice(l - 20, l)
    expected = ref.conv1d(x[:, last], w, None, "silu", x[:, l - 23 : l - 20], dy[:, last])
    ref.check("y", y[:, last], *expected[0], 40)
    assert torch.equal(state, x[:, -3:])
    ref.check("dx", dx[:, last], *expected[2], 80)
    del x, dy, y, dx
    torch.cuda.empty_cache()


def test_scan_past_31_bits():
    l, c = (1 << 21) + 3, 1024
    u, dy = _far(1, l, c).requires_grad_(), _far(1, l, c)
    delta = torch.full((1, l, c), 0.5, dtype=BF16, device="cuda").requires_grad_()
    B, C = _far(1, l, 1).requires_grad_(), _far(1, l, 1)
    A = -(1 + torch.rand(c, 1, generator=torch.Generator().manual_seed(0))).cuda()
    y, state = selective_scan(u, delta, A, B, C, return_state=True)
    du, ddelta, dB = torch.autograd.grad(y, (u, delta, B), dy)
    # what came before the last 400 tokens is less than e^-50 of itself at the last 300
    part, last = slice(l - 400, l), slice(l - 300, l)
    expected = ref.scan(*(t[:, part] for t in (u, delta)), A, *(t[:, part] for t in (B, C)), None, None, None, False, None, dy[:, part])
    tail = [(value[:, 100:], size[:, 100:]) for value, size in (expected[0], expected[2], expected[3], expected[5])]
    ref.check("y", y[:, last], *tail[0], 3 * 400 + 100)
    ref.check("state", state, *expected[1], 3 * 400 + 100)
    ref.check("du", du[:, last], *tail[1], 2 * (3 * 400 + 100) + 30)
    ref.check("ddelta", ddelta[:, last], *tail[2], 2 * (3 * 400 + 100) + 30)
    ref.check("dB", dB[:, last], *tail[3], 2 * (3 * 400 + 100) + 30 + c)
    del u, dy, delta, y, du, ddelta
    torch.cuda.empty_cache()


@pytest.mark.parametrize("norm", [False, True])
def test_rotation_past_31_bits(norm):
    l, heads, d = (1 << 21) + 5, 16, 64
    q, k, gq = _far(1, l, heads, d).requires_grad_(), _far(1, l, 1, d), _far(1, l, heads, d)
    w = _normal(d) if norm else None
    positions, frequencies = torch.arange(l, device="cuda"), rotary_frequencies(d, device="cuda")
    out = head_norm_rotary(q, k, w, w, positions, frequencies) if norm else rotary(q, k, positions, frequencies)
    dq = torch.autograd.grad(out[0], q, gq)[0]
    last = slice(l - 5, l)
    expected = ref.rotary(q[:, last], w, positions[last], frequencies, 1e-6, False, 1.0, gq[:, last])
    ref.check("out", out[0][:, last], *expected[0], d + 60)
    ref.check("dx", dq[:, last], *expected[1], 3 * d + 120)
    del q, k, gq, out, dq
    torch.cuda.empty_cache()
