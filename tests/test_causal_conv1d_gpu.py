"""causal_conv1d, its gradients and its step on the GPU against the definition in 64 bits (token_reference.py)."""

import pytest
import torch

from spio_amd.functional import causal_conv1d, causal_conv1d_step
from spio_amd.functional.causal_conv1d_function import causal_conv1d_forward, causal_conv1d_step_op
from spio_amd.layers import CausalConv1d
from spio_amd.native import Bypass
from tests import token_reference as ref

pytestmark = pytest.mark.gpu
HALF, BF16, FLOAT = torch.float16, torch.bfloat16, torch.float32


def _tensors(n, l, c, width, dtype, wdtype=FLOAT, bias=True, state=False, seed=0, wide=0):
    """Inputs, weight, bias, state, gradient; with `wide` the inputs are part of rows that are so many values longer."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, l, c + wide, generator=g).to(dtype).cuda()[..., wide // 2 : wide // 2 + c]
    weight = (torch.rand(c, width, generator=g) - 0.5).to(wdtype).cuda()
    b = (torch.rand(c, generator=g) - 0.5).to(wdtype).cuda() if bias else None
    before = torch.randn(n, width - 1, c, generator=g).to(dtype).cuda() if state else None
    return x, weight, b, before, torch.randn(n, l, c, generator=g).to(dtype).cuda()


def _train(x, weight, bias, act, before, dy):
    leaves = [t.detach().requires_grad_() for t in (x, weight, bias) if t is not None]
    y = causal_conv1d(*leaves[:2], leaves[2] if bias is not None else None, act, before)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


# one token, fewer than the filter, a slice and one more, several slices (forward 4 to 32, backward 16 to 256 tokens)
@pytest.mark.parametrize("n,l,c,width,dtype,wdtype,act,bias,state,wide", [
    (1, 1, 8, 4, FLOAT, FLOAT, "silu", True, False, 0),
    (2, 2, 24, 4, HALF, FLOAT, "silu", True, True, 0),
    (3, 5, 16, 2, BF16, FLOAT, "none", False, True, 0),
    (1, 17, 200, 4, FLOAT, FLOAT, "silu", True, True, 16),
    (2, 33, 72, 8, FLOAT, FLOAT, "none", True, True, 4),
    (2, 100, 40, 4, BF16, BF16, "silu", True, False, 8),
    (5, 301, 64, 3, HALF, HALF, "silu", True, False, 0),
    (1, 1000, 8, 4, HALF, FLOAT, "silu", False, False, 4),  # rows that do not start on 16 bytes: copied
])  # fmt: skip
def test_outputs_and_gradients(n, l, c, width, dtype, wdtype, act, bias, state, wide):
    x, weight, b, before, dy = _tensors(n, l, c, width, dtype, wdtype, bias, state, wide=wide)
    expected = ref.conv1d(x, weight, b, act, before, dy)
    y, *grads = _train(x, weight, b, act, before, dy)
    assert y.dtype == dtype and grads[0].dtype == dtype and grads[1].dtype == wdtype
    ref.check("y", y, *expected[0], width + 1 + 24)
    ref.check("dx", grads[0], *expected[2], 2 * width + 40)
    # sums over tokens: a lane's in 32 bits, up to 256 and the filter's more, those of the lanes in 64
    ref.check("dweight", grads[1], *expected[3], min(l, 256) + 2 * width + 40)
    if bias:
        ref.check("dbias", grads[2], *expected[4], min(l, 256) + 2 * width + 40)
    with torch.no_grad():
        plain, after = causal_conv1d(x, weight, b, act, before, return_state=True)
    assert torch.equal(plain, y)
    assert torch.equal(after.cpu().double(), expected[1][0])


@pytest.mark.parametrize("dtype,width", [(FLOAT, 4), (BF16, 4), (HALF, 2)])
def test_pieces_and_steps_go_on_from_the_state(dtype, width):
    x, weight, bias, before, _ = _tensors(3, 11, 24, width, dtype, state=True)
    expected = ref.conv1d(x, weight, bias, "silu", before, None)
    first, state = causal_conv1d(x[:, :4], weight, bias, "silu", before, return_state=True)
    second, state = causal_conv1d(x[:, 4:5], weight, bias, "silu", state, return_state=True)
    rows = [first, second]
    for t in range(5, 11):
        kept = state.clone()
        if t % 2:
            other = torch.full_like(state, float("nan"))
            rows.append(causal_conv1d_step(x[:, t], state, weight, bias, "silu", out_state=other)[:, None])
            assert torch.equal(state, kept)  # only out_state is written
            state = other
        else:
            rows.append(causal_conv1d_step(x[:, t], state, weight, bias, "silu")[:, None])
    ref.check("pieces", torch.cat(rows, 1), *expected[0], width + 1 + 24)
    assert torch.equal(state.cpu().double(), expected[1][0])


def test_python_path_is_the_same():
    x, weight, bias, before, dy = _tensors(2, 70, 40, 4, BF16, state=True, wide=8)
    native = _train(x, weight, bias, "silu", before, dy)
    state, other = before.clone(), before.clone()
    stepped = causal_conv1d_step(x[:, 3], state, weight, bias, "silu")
    bypass = Bypass()
    try:
        python = _train(x, weight, bias, "silu", before, dy)
        again = causal_conv1d_step(x[:, 3], other, weight, bias, "silu")
    finally:
        bypass.release()
    assert all(torch.equal(a, b) for a, b in zip(native, python))
    assert torch.equal(stepped, again) and torch.equal(state, other)
    assert all(torch.equal(a, b) for a, b in zip(native, _train(x, weight, bias, "silu", before, dy)))  # no order of atomics


def test_what_is_not_finite_stays_with_its_token_and_channel():
    x, weight, bias, _, dy = _tensors(2, 40, 16, 4, FLOAT)
    clean = _train(x, weight, bias, "silu", None, dy)
    x[0, 39, 3], x[1, 7, 5] = float("nan"), float("inf")
    y, dx, *_ = _train(x, weight, bias, "silu", None, dy)
    touched = torch.zeros_like(y, dtype=torch.bool)
    touched[0, 39, 3], touched[1, 7:11, 5] = True, True
    assert torch.equal(y[~touched], clean[0][~touched]) and y[0, 39, 3].isnan()
    back = torch.zeros_like(y, dtype=torch.bool)
    back[0, 36:, 3], back[1, 4:11, 5] = True, True
    assert torch.equal(dx[~back], clean[1][~back])


def test_empty():
    for n, l in ((0, 4), (2, 0)):
        x, weight, bias, before, dy = _tensors(n, l, 16, 4, HALF, state=True)
        y, dx, dw, db = _train(x, weight, bias, "silu", before, dy)
        assert y.shape == dx.shape == x.shape and not dw.any() and not db.any()
        y, state = causal_conv1d(x, weight, bias, "silu", before, return_state=True)
        assert torch.equal(state, before)
    assert causal_conv1d_step(torch.empty(0, 16, device="cuda"), torch.empty(0, 3, 16, device="cuda"), torch.ones(16, 4, device="cuda")).shape == (0, 16)


def test_refusals():
    x, weight, bias, before, dy = _tensors(2, 5, 16, 4, HALF, state=True)
    for call in (
        lambda: causal_conv1d(x, weight[:, :1], bias),
        lambda: causal_conv1d(x, torch.ones(16, 9, device="cuda"), bias),
        lambda: causal_conv1d(x, weight, bias, "gelu"),
        lambda: causal_conv1d(x, weight, bias.cpu()),
        lambda: causal_conv1d(x, weight, bias, "none", before[:, :2]),
        lambda: causal_conv1d(x, weight, bias, "none", before.float()),
        lambda: causal_conv1d(x[..., :12], weight[:12], bias[:12]),
        lambda: causal_conv1d_step(x[:, 0], before, weight, bias, out_state=before[:1]),
        lambda: causal_conv1d_step(x[:, 0], before.transpose(1, 2).contiguous().transpose(1, 2), weight, bias),
        lambda: causal_conv1d_step(before[:, 1], before, weight, bias),  # part of the state that is written
        lambda: causal_conv1d_step(x[:, 0], before.flatten()[: 48].view(1, 3, 16).expand(2, 3, 16), weight, bias),
    ):  # fmt: skip
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(RuntimeError):
        causal_conv1d(x, weight, bias, "none", before.clone().requires_grad_())
    shifted = torch.zeros(2 * 3 * 16 + 16, dtype=HALF, device="cuda")
    with pytest.raises(AssertionError):  # overlapping states
        causal_conv1d_step(x[:, 0], shifted[:96].view(2, 3, 16), weight, bias, out_state=shifted[16:].view(2, 3, 16))
    leaf = x.clone().requires_grad_()
    y = causal_conv1d(leaf, weight)
    (dx,) = torch.autograd.grad(y, leaf, dy.clone().requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivatives
        torch.autograd.grad(dx.sum(), leaf)
    twice = leaf * 1
    y = causal_conv1d(twice, weight)
    twice.add_(1)
    with pytest.raises(RuntimeError):  # what the backward pass needs has changed
        y.sum().backward()


def test_opcheck_and_compile():
    x, weight, bias, before, dy = _tensors(2, 9, 16, 4, HALF, state=True)
    xg, wg, bg = (t.clone().requires_grad_() for t in (x, weight, bias))
    torch.library.opcheck(causal_conv1d_forward, (xg, wg, bg, "silu", before, True))
    torch.library.opcheck(causal_conv1d_step_op, (x[:, 0], before, weight, bias, "silu", before.clone()))
    compiled = torch.compile(lambda x, w, b: causal_conv1d(x, w, b, "silu"), backend="aot_eager")
    got = torch.autograd.grad(compiled(xg, wg, bg), [xg, wg, bg], dy)
    expected = _train(x, weight, bias, "silu", None, dy)[1:]
    assert all(torch.equal(a, b) for a, b in zip(got, expected))


def test_captured():
    """A step of a prompt and of decoding, captured, replayed on other inputs with eager work between."""
    x, weight, bias, before, dy = _tensors(2, 40, 16, 4, BF16, state=True)
    static, state = x.clone(), before.clone()
    _train(static, weight, bias, "silu", before, dy)  # plans and kernels are made outside
    causal_conv1d_step(static[:, 0], before.clone(), weight, bias, "silu")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _train(static, weight, bias, "silu", before, dy)
        stepped = causal_conv1d_step(static[:, 0], state, weight, bias, "silu")
    eager_state = state.clone()
    for seed in range(3):
        fresh = _tensors(2, 40, 16, 4, BF16, seed=seed + 1)[0]
        static.copy_(fresh)
        graph.replay()
        expected = _train(fresh, weight, bias, "silu", before, dy)
        step = causal_conv1d_step(fresh[:, 0], eager_state, weight, bias, "silu")
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, expected))
        assert torch.equal(stepped, step) and torch.equal(state, eager_state)


def test_layer():
    torch.manual_seed(0)
    layer = CausalConv1d(24, 4, activation="silu").cuda()
    x = torch.randn(2, 6, 24, device="cuda")
    whole = layer(x)
    whole.sum().backward()
    assert layer.weight.grad.shape == (24, 4) and layer.bias.grad.shape == (24,)
    state = layer.empty_state(2)
    with torch.no_grad():
        rows = torch.stack([layer.step(x[:, t], state) for t in range(6)], 1)
    torch.testing.assert_close(rows, whole.detach(), rtol=1e-5, atol=1e-6)
