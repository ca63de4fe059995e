"""Calls of the operators over sequences of tokens as programs make them beside plain ones: limits on the native path, steps that are
compiled."""

import pytest
import torch

from spio_amd import native
from spio_amd.functional import causal_conv1d_step, rotary, rotary_frequencies, selective_scan_step
from spio_amd.layers import CausalConv1d, HeadNormRotary, SelectiveScan

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
