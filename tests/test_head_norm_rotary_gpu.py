"""rotary and head_norm_rotary with their gradients on the GPU against the definition in 64 bits (token_reference.py)."""

import pytest
import torch

from spio_amd.functional import head_norm_rotary, rotary, rotary_frequencies
from spio_amd.functional.head_norm_rotary_function import head_norm_rotary_forward
from spio_amd.layers import HeadNormRotary
from spio_amd.native import Bypass
from tests import token_reference as ref

pytestmark = pytest.mark.gpu
HALF, BF16, FLOAT = torch.float16, torch.bfloat16, torch.float32


def _tensors(n, l, q, k, d, dtype, norm, seed=0, gap=0):
    """Queries and keys as parts of one projection, whose heads are `gap` values apart."""
    g = torch.Generator().manual_seed(seed)
    rows = torch.randn(n, l, q + 2 * k, d + gap, generator=g).to(dtype).cuda()
    weights = [(torch.rand(d, generator=g) + 0.5).cuda() if norm else None for _ in range(2)]
    grads = [torch.randn(n, l, h, d, generator=g).to(dtype).cuda() for h in (q, k)]
    return rows[:, :, :q, :d], rows[:, :, q : q + k, :d], *weights, *grads


def _call(q, k, wq, wk, positions, frequencies, interleaved, scale):
    if wq is None:
        return rotary(q, k, positions, frequencies, interleaved, scale)
    return head_norm_rotary(q, k, wq, wk, positions, frequencies, 1e-6, interleaved, scale)


def _train(q, k, wq, wk, gq, gk, *rest):
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk) if t is not None]
    out = _call(*(leaves if wq is not None else [*leaves, None, None]), *rest)
    return [*(t.detach() for t in out), *torch.autograd.grad(out, leaves, [gq, gk])]


# heads of one lane to sixteen, some of them idle; all and a part of the channels turned; one head and several; positions
# of every sequence, or the same; far ones; heads with gaps, aligned and not (copied)
@pytest.mark.parametrize("n,l,q,k,d,pairs,dtype,norm,interleaved,start,own,scale,gap", [
    (1, 1, 1, 1, 8, 3, FLOAT, True, True, 0, True, 1.0, 0),
    (2, 5, 4, 2, 64, 32, FLOAT, True, False, 100000, True, 1.2, 0),
    (3, 7, 5, 5, 80, 40, HALF, False, False, 0, False, 1.0, 0),
    (2, 33, 3, 1, 80, 16, FLOAT, False, True, 2000000000, True, -0.5, 0),
    (1, 130, 6, 2, 128, 64, BF16, True, False, 7, False, 1.0, 16),
    (2, 9, 12, 3, 96, 8, FLOAT, True, False, 30, False, 1.0, 3),
    (1, 70, 2, 2, 256, 128, BF16, True, True, 0, True, 1.0, 0),
    (4, 300, 1, 1, 32, 16, HALF, False, False, 0, True, 2.0, 8),
])  # fmt: skip
def test_outputs_and_gradients(n, l, q, k, d, pairs, dtype, norm, interleaved, start, own, scale, gap):
    x, y, wq, wk, gq, gk = _tensors(n, l, q, k, d, dtype, norm, gap=gap)
    positions = torch.arange(l, device="cuda") + start
    if own:
        positions = positions + 3 * torch.arange(n, device="cuda")[:, None]
    if start < 1 << 20:
        positions = positions.int()
    frequencies = rotary_frequencies(2 * pairs, device="cuda")
    got = _train(x, y, wq, wk, gq, gk, positions, frequencies, interleaved, scale)
    # cosines and sines: the angle's share of a turn in 32 bits, their series, the products: less than 20 units of 1
    for i, (t, w, g) in enumerate(((x, wq, gq), (y, wk, gk))):
        expected = ref.rotary(t, w, positions, frequencies, 1e-6, interleaved, scale, g)
        ref.check("out", got[i], *expected[0], d + 60)
        ref.check("dx", got[2 + i], *expected[1], 3 * d + 120)
        if norm:
            # sums over tokens and heads: a lane's and a workgroup's in 32 bits
            ref.check("dweight", got[4 + i], *expected[2], 2 * n * l * max(q, k) + d + 120)
    with torch.no_grad():
        plain = _call(x, y, wq, wk, positions, frequencies, interleaved, scale)
    assert torch.equal(plain[0], got[0]) and torch.equal(plain[1], got[1])


def test_many_tokens_share_a_lane():
    """More tokens than a backward pass with norms has groups of lanes: these go from token to token."""
    n, l, q, k, d = 1, 33000, 1, 1, 64
    x, y, wq, wk, gq, gk = _tensors(n, l, q, k, d, FLOAT, True)
    positions, frequencies = torch.arange(l, device="cuda"), rotary_frequencies(d, device="cuda")
    got = _train(x, y, wq, wk, gq, gk, positions, frequencies, False, 1.0)
    expected = ref.rotary(x, wq, positions, frequencies, 1e-6, False, 1.0, gq)
    ref.check("dx", got[2], *expected[1], 3 * d + 120)
    ref.check("dweight", got[4], *expected[2], 200 + d)  # 3 tokens a lane, 64 lanes a workgroup, 512 of them in 64 bits


def test_no_gradient_of_one_of_the_outputs():
    for norm in (False, True):
        x, y, wq, wk, gq, gk = _tensors(2, 4, 3, 2, 32, FLOAT, norm)
        rest = (torch.arange(4, device="cuda"), rotary_frequencies(32, device="cuda"), False, 1.0)
        zero = _train(x, y, wq, wk, gq, torch.zeros_like(gk), *rest)[2:]
        for bypassed in (False, True):
            bypass = Bypass() if bypassed else None
            leaves = [t.detach().requires_grad_() for t in (x, y, wq, wk) if t is not None]
            out = _call(*(leaves if norm else [*leaves, None, None]), *rest)
            got = torch.autograd.grad(out[0], leaves, gq, allow_unused=True)
            if bypass:
                bypass.release()
            assert all(torch.equal(a if a is not None else torch.zeros_like(b), b) for a, b in zip(got, zero))


def test_rows_of_zeros_and_what_is_not_finite():
    x, y, wq, wk, gq, gk = _tensors(1, 3, 2, 2, 64, FLOAT, True)
    rest = (torch.arange(3, device="cuda"), rotary_frequencies(64, device="cuda"), False, 1.0)
    clean = _train(x, y, wq, wk, gq, gk, *rest)
    x[0, 0, 0] = 0.0
    x[0, 1, 1, 5] = float("nan")
    got = _train(x, y, wq, wk, gq, gk, *rest)
    assert not got[0][0, 0, 0].any() and got[2][0, 0, 0].isfinite().all()
    assert got[0][0, 1, 1].isnan().all() and torch.equal(got[0][0, 2], clean[0][0, 2])
    assert torch.equal(got[0][0, 1, 0], clean[0][0, 1, 0]) and torch.equal(got[3], clean[3]) and torch.equal(got[5], clean[5])


def test_python_path_is_the_same():
    x, y, wq, wk, gq, gk = _tensors(2, 21, 6, 2, 80, BF16, True)
    rest = (torch.arange(21, device="cuda") + 5, rotary_frequencies(64, device="cuda"), False, 1.1)
    native = _train(x, y, wq, wk, gq, gk, *rest)
    bypass = Bypass()
    try:
        python = _train(x, y, wq, wk, gq, gk, *rest)
    finally:
        bypass.release()
    assert all(torch.equal(a, b) for a, b in zip(native, python))


def test_empty():
    for shape in ((0, 4, 2, 32), (2, 0, 2, 32), (2, 4, 0, 32)):
        q = torch.empty(shape, device="cuda", dtype=HALF, requires_grad=True)
        k = torch.ones(*shape[:2], 1, 32, device="cuda", dtype=HALF)
        w = torch.ones(32, device="cuda", requires_grad=True)
        positions = torch.arange(shape[1], device="cuda")
        out = head_norm_rotary(q, k, w, w, positions, rotary_frequencies(32, device="cuda"))
        assert out[0].shape == shape and out[1].shape == k.shape
        dq, dw = torch.autograd.grad(out[0], [q, w], torch.empty_like(out[0]))
        assert dq.shape == shape and not dw.any()


def test_refusals():
    x, y, wq, wk, gq, gk = _tensors(2, 4, 3, 2, 32, HALF, True)
    positions, frequencies = torch.arange(4, device="cuda"), rotary_frequencies(32, device="cuda")
    for call in (
        lambda: rotary(x, y.float(), positions, frequencies),
        lambda: rotary(x, y[:, :3], positions, frequencies),
        lambda: rotary(x[..., :16], y, positions, frequencies),
        lambda: rotary(x[..., :12], y[..., :12], positions, frequencies[:4], True),
        lambda: rotary(x, y, positions[:3], frequencies),
        lambda: rotary(x, y, positions.float(), frequencies),
        lambda: rotary(x, y, positions.cpu(), frequencies),
        lambda: rotary(x, y, positions, frequencies.float()),
        lambda: rotary(x, y, positions, frequencies[:4]),
        lambda: rotary(x, y, positions, frequencies[:0]),
        lambda: rotary(x, y, positions, torch.cat([frequencies, frequencies[:8]])),
        lambda: rotary(x, y, positions, frequencies, scale=float("inf")),
        lambda: head_norm_rotary(x, y, wq, None, positions, frequencies),
        lambda: head_norm_rotary(x, y, wq, wk[:16], positions, frequencies),
        lambda: head_norm_rotary(x, y, wq, wk, positions, frequencies, eps=0.0),
        lambda: rotary(torch.zeros(1, 4, 1, 264, device="cuda"), torch.zeros(1, 4, 1, 264, device="cuda"), positions, frequencies),
    ):  # fmt: skip
        with pytest.raises(AssertionError):
            call()
    leaf = x.clone().requires_grad_()
    out = head_norm_rotary(leaf, y, wq, wk, positions, frequencies)
    (dx,) = torch.autograd.grad(out[0], leaf, gq.clone().requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivatives
        torch.autograd.grad(dx.sum(), leaf)


def test_opcheck_and_compile():
    x, y, wq, wk, gq, gk = _tensors(2, 4, 3, 2, 32, HALF, True)
    positions, frequencies = torch.arange(4, device="cuda"), rotary_frequencies(32, device="cuda")
    leaves = [t.detach().clone().requires_grad_() for t in (x, y, wq, wk)]
    torch.library.opcheck(head_norm_rotary_forward, (*leaves, positions, frequencies, 1e-6, False, 1.0))
    compiled = torch.compile(lambda *a: head_norm_rotary(*a, positions, frequencies), backend="aot_eager")
    got = torch.autograd.grad(compiled(*leaves), leaves, [gq, gk])
    expected = _train(x, y, wq, wk, gq, gk, positions, frequencies, False, 1.0)[2:]
    assert all(torch.equal(a, b) for a, b in zip(got, expected))


def test_captured():
    """A training step, captured, replayed on other inputs and positions with eager work between."""
    rest = (rotary_frequencies(64, device="cuda"), False, 1.0)
    x, y, wq, wk, gq, gk = _tensors(2, 21, 6, 2, 64, BF16, True)
    sq, sk, positions = x.clone(), y.clone(), torch.arange(21, device="cuda")
    _train(sq, sk, wq, wk, gq, gk, positions, *rest)  # plans and kernels are made outside
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _train(sq, sk, wq, wk, gq, gk, positions, *rest)
    for seed in range(3):
        x, y = _tensors(2, 21, 6, 2, 64, BF16, True, seed=seed + 1)[:2]
        sq.copy_(x)
        sk.copy_(y)
        positions += 1000
        graph.replay()
        expected = _train(x, y, wq, wk, gq, gk, positions, *rest)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, expected))


def test_layer():
    layer = HeadNormRotary(64, rotated=32, method="ramp", factor=4.0).cuda().half()
    assert layer.frequencies.dtype == torch.float64 and layer.frequencies.is_cuda and layer.q_weight.dtype == HALF
    q = torch.randn(2, 5, 4, 64, device="cuda", dtype=HALF)
    out = layer(q, q[:, :, :2])
    (out[0].sum() + out[1].sum()).backward()
    assert layer.q_weight.grad.shape == (64,) and layer.q_weight.grad.dtype == HALF
    later = layer(q[:, 3:4], q[:, 3:4, :2], torch.tensor([3], device="cuda"))
    assert torch.equal(later[0], out[0][:, 3:4]) and torch.equal(later[1], out[1][:, 3:4])
    turned = HeadNormRotary(64, norm=False, interleaved=True).cuda()
    q = q.float()
    assert turned.q_weight is None
    torch.testing.assert_close(turned(q, q)[0].norm(dim=-1), q.norm(dim=-1), rtol=1e-5, atol=1e-5)
