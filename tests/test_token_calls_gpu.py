"""Calls of the operators over sequences of tokens as programs make them beside plain ones: limits on the native path, steps that are
compiled, tensors that are broadcast or in several places, graphs and streams in turn."""

import pytest
import torch

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
from spio_amd.layers import CausalConv1d, HeadNormRotary, SelectiveScan
from tests import token_reference as ref

pytestmark = pytest.mark.gpu


def _normal(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def test_scales_on_the_native_path():
    q, positions, frequencies = _normal(1, 3, 2, 16), torch.arange(3, device="cuda"), rotary_frequencies(16, device="cuda")
    for scale, taken in ((1e39, False), (-float("inf"), False), (float("nan"), False), (3.4028236e38, False), (-3.4028234e38, True)):
        out = native.call("head_norm_rotary", q, q, None, None, positions, frequencies, 1.0, False, scale)
        assert (out is not NotImplemented) == taken
        if not taken:
            with pytest.raises(AssertionError, match="scale"):
                rotary(q, q, positions, frequencies, scale=scale)


@pytest.mark.parametrize("other", [False, True])
def test_compiled_steps(other):
    """Steps update their states in place, or another tensor, also where they are compiled."""
    x, w = _normal(2, 16), _normal(16, 4, seed=1)
    A, rows = -_normal(16, 4, seed=2).abs(), _normal(2, 8, seed=3)

    def step(x, window, state, window_out, state_out):
        y = causal_conv1d_step(x, window, w, None, "silu", window_out)
        return selective_scan_step(y, state, x, A, rows[:, :4], rows[:, 4:], None, x, None, True, state_out)

    window, state = _normal(2, 3, 16, seed=4), _normal(2, 16, 4, seed=5)
    results = []
    for f in (step, torch.compile(step, backend="aot_eager")):
        a, b = window.clone(), state.clone()
        outs = (torch.zeros_like(a), torch.zeros_like(b)) if other else (None, None)
        y = f(x, a, b, *outs)
        results.append((y, a, b, *(t for t in outs if t is not None)))
    assert all(torch.equal(p, q) for p, q in zip(*results))
    assert torch.equal(results[0][1], window) == other


def test_compiled_layers():
    torch.manual_seed(0)
    conv, scan, norm = CausalConv1d(16, 4, activation="silu").cuda(), SelectiveScan(16, 4).cuda(), HeadNormRotary(16).cuda()
    x = _normal(2, 6, 16)

    def model(x):
        y, window = conv(x, return_state=True)
        y, state = scan(y, x, x[..., :4], x[..., 4:8], x, return_state=True)
        q, k = norm(y[:, :, None], x[:, :, None])
        return q + k, window, state

    with torch.no_grad():
        expected, got = model(x), torch.compile(model, backend="aot_eager")(x)
    assert all(torch.equal(a, b) for a, b in zip(expected, got))
    loss = lambda f: f(x)[0].square().sum()  # noqa: E731
    parameters = [p for layer in (conv, scan, norm) for p in layer.parameters()]
    grads = [torch.autograd.grad(loss(f), parameters) for f in (model, torch.compile(model, backend="aot_eager"))]
    for a, b in zip(*grads):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)


def _leaves(*tensors):
    return [t.detach().clone().requires_grad_() for t in tensors]


@pytest.mark.parametrize("python", [False, True])
def test_the_same_tensor_in_several_places(python):
    """Inputs, steps and gate of a scan are one tensor, B and C another; queries are keys.  Gradients add up."""
    bypass = native.Bypass() if python else None
    try:
        x, rows, A = _leaves(_normal(2, 21, 16), _normal(2, 21, 3, seed=1), -_normal(16, 3, seed=2).abs())
        dy = _normal(2, 21, 16, seed=3)
        got = torch.autograd.grad(selective_scan(x, x, A, rows, rows, None, x, None, True), (x, rows, A), dy)
        expected = ref.scan(x, x, A, rows, rows, None, x, None, True, None, dy)
        terms = 2 * (3 * 21 + 3 + 80)
        for what, grad, parts, more in (("x", got[0], (2, 3, 8), 0), ("rows", got[1], (5, 6), 16), ("A", got[2], (4,), 21)):
            value, size = (sum(expected[i][k] for i in parts) for k in (0, 1))
            # (parts that autograd adds are rounded before)
            ref.check(what, grad, value, size, terms + more + 2 * len(parts))
        q, w = _leaves(_normal(2, 7, 3, 32), torch.rand(32, device="cuda") + 0.5)
        positions, frequencies, gq = torch.arange(7, device="cuda"), rotary_frequencies(32, device="cuda"), _normal(2, 7, 3, 32, seed=4)
        out = head_norm_rotary(q, q, w, w, positions, frequencies)
        assert torch.equal(*out)
        dq, dw = torch.autograd.grad(out, (q, w), (gq, gq))
        expected = ref.rotary(q, w, positions, frequencies, 1e-6, False, 1.0, gq)
        ref.check("q", dq, 2 * expected[1][0], 2 * expected[1][1], 3 * 32 + 120)
        ref.check("w", dw, 2 * expected[2][0], 2 * expected[2][1], 2 * 2 * 7 * 3 + 32 + 120)
    finally:
        if bypass:
            bypass.release()


def test_broadcast_and_strided_tensors():
    """Rows, heads, states and parameters that are expanded, transposed, of other types or taken by steps."""
    n, l, c, s = 2, 19, 24, 5
    x, delta = _normal(1, l, c, seed=1).expand(n, l, c), _normal(n, 1, c, seed=2).expand(n, l, c)
    B, C = _normal(n, l, 1, seed=3).expand(n, l, s), _normal(n, s, l, seed=4).transpose(1, 2)
    A, D = -_normal(s, c, seed=5).abs().double().t(), _normal(2 * c, seed=6).half()[::2]
    before = _normal(1, c, s, seed=7).expand(n, c, s)
    y, state = selective_scan(x, delta, A, B, C, D, None, None, True, before, return_state=True)
    expected = ref.scan(x, delta, A, B, C, D, None, None, True, before, None)
    ref.check("scan", y, *expected[0], 3 * l + s + 80)
    ref.check("state", state, *expected[1], 3 * l + s + 80)
    w, bias = _normal(3, c, seed=8).t(), _normal(1, seed=9).expand(c).bfloat16()
    window = _normal(n, 1, c, seed=10).expand(n, 2, c)
    for inputs in (x, delta, _normal(n, c, l, seed=11).transpose(1, 2), _normal(n, l, 2 * c, seed=12)[..., ::2]):
        y, after = causal_conv1d(inputs, w, bias, "silu", window, return_state=True)
        expected = ref.conv1d(inputs, w, bias, "silu", window, None)
        ref.check("conv", y, *expected[0], 3 + 1 + 24)
        assert torch.equal(after.cpu().double(), expected[1][0])
    q, k = _normal(n, l, 1, 32, seed=13).expand(n, l, 4, 32), _normal(n, 2, l, 32, seed=14).transpose(1, 2)
    frequencies = rotary_frequencies(64, device="cuda")[::2]
    for positions in (torch.arange(2 * l, device="cuda")[::2], torch.arange(n, device="cuda").int()[:, None].expand(n, l) - 7,
                      torch.arange(l, device="cuda") - (1 << 40), torch.arange(l, device="cuda") + (1 << 33)):  # fmt: skip
        out = rotary(q, k, positions, frequencies)
        for t, got in zip((q, k), out):
            ref.check("rotary", got, *ref.rotary(t, None, positions, frequencies, 0, False, 1.0, None)[0], 60 + _far(positions))


def _far(positions):
    """Units of 2^-24 that an angle of the largest position is off by, in the kernel and in the definition: 2^-52 of it each."""
    return 2 * int(positions.abs().max()) * 2.0**-28


@pytest.mark.parametrize("python", [False, True])
def test_graphs_and_a_stream_in_turn(python):
    """Two captured training steps and an eager one on another stream, replayed in turn: none works in another's memory."""
    bypass = native.Bypass() if python else None
    try:
        def step(x, A):
            x, A = x.detach().requires_grad_(), A.detach().requires_grad_()
            y = selective_scan(causal_conv1d(x, A[:, :4], None, "silu"), x, -A.abs(), x[..., :5], x[..., 5:10], None, x, None, True)
            return [y.detach(), *torch.autograd.grad(y, (x, A), torch.ones_like(y))]

        data = [(_normal(2, l, 24, seed=l), _normal(24, 5, seed=l + 1)) for l in (40, 90)]
        expected = [[t.clone() for t in step(*d)] for d in data]
        torch.cuda.synchronize()
        graphs = []
        for d in data:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(*d)
            graphs.append((graph, out))
        other = torch.cuda.Stream()
        for turn in range(3):
            for graph, out in graphs:
                for t in out:
                    t.zero_()
            other.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(other):
                aside = step(*data[turn % 2])
            for graph, _ in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for (_, out), e in zip(graphs, expected):
                assert all(torch.equal(a, b) for a, b in zip(out, e))
            assert all(torch.equal(a, b) for a, b in zip(aside, expected[turn % 2]))
    finally:
        if bypass:
            bypass.release()
