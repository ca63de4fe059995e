"""selective_scan, its gradients and its step on the GPU against the definition in 64 bits (token_reference.py)."""

import pytest
import torch

from spio_amd.functional import selective_scan, selective_scan_step
from spio_amd.functional.selective_scan_function import selective_scan_forward, selective_scan_step_op
from spio_amd.kernels.selective_scan_kernel import chunk_tokens
from spio_amd.layers import SelectiveScan
from spio_amd.native import Bypass
from tests import token_reference as ref

pytestmark = pytest.mark.gpu
HALF, BF16, FLOAT = torch.float16, torch.bfloat16, torch.float32
NAMES = ("u", "delta", "A", "B", "C", "D", "gate", "bias")


def _tensors(n, l, c, s, dtype, gate=True, D=True, bias=True, softplus=True, state=False, seed=0):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g)

    rows = normal(n, l, 2 * s + 5).to(dtype).cuda()  # B and C are parts of wider rows, on any byte
    both = normal(n, l, 2 * c).to(dtype).cuda()
    t = {
        "u": both[..., :c],
        "delta": (normal(n, l, c) * 0.5 if softplus else normal(n, l, c).abs() * 0.1).to(dtype).cuda(),
        "A": -(torch.arange(1, s + 1) * (0.8 + 0.4 * torch.rand(c, s, generator=g))).cuda(),
        "B": rows[..., 5 : 5 + s], "C": rows[..., 5 + s :],
        "D": normal(c).cuda() if D else None,
        "gate": both[..., c:] if gate else None,
        "bias": (normal(c) - 3 if softplus else torch.rand(c, generator=g) * 0.05).cuda() if bias else None,
    }  # fmt: skip
    before = normal(n, c, s).cuda() if state else None
    return t, before, normal(n, l, c).to(dtype).cuda()


def _train(t, softplus, before, dy):
    leaves = {k: None if v is None else v.detach().requires_grad_() for k, v in t.items()}
    y = selective_scan(*leaves.values(), softplus, before)
    present = [k for k, v in leaves.items() if v is not None]
    grads = torch.autograd.grad(y, [leaves[k] for k in present], dy)
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(present, grads)}}


# (16 states, gate, softplus) as layers have them; odd numbers of states, without what is optional; the most; lengths of
# one token, of parts of a tile (4 or 8 tokens), of one chunk and of several; channels of parts of a wave and of several.
# As many sequences as make one chunk of all tokens (1024 waves) are in the last one.
CASES = [
    (1, 1, 1, 16, FLOAT, True, True, True, True, True),
    (2, 37, 70, 16, FLOAT, True, True, True, True, True),
    (1, 300, 130, 16, BF16, True, True, True, True, False),
    (3, 66, 64, 5, HALF, False, False, False, False, True),
    (1, 41, 33, 5, FLOAT, False, True, False, False, False),
    (2, 50, 65, 32, FLOAT, True, False, True, True, False),
    (1, 100, 20, 1, BF16, False, False, True, True, False),
    (1030, 3, 40, 5, HALF, False, False, False, False, False),
]


@pytest.mark.parametrize("n,l,c,s,dtype,gate,D,bias,softplus,state", CASES)
def test_outputs_and_gradients(n, l, c, s, dtype, gate, D, bias, softplus, state):
    t, before, dy = _tensors(n, l, c, s, dtype, gate, D, bias, softplus, state)
    expected = ref.scan(*t.values(), softplus, before, dy)
    got = _train(t, softplus, before, dy)
    # a token's state has the roundings of all before it (three a token), and one more sum over the states
    terms = 3 * l + s + 80
    ref.check("y", got["y"], *expected[0], terms)
    for i, name in enumerate(NAMES):
        if t[name] is None:
            continue
        # through the states both ways; sums over channels in 32 bits, over tokens a chunk's in 32 and the chunks' in 64
        more = c if name in "BC" else l if name in ("A", "D", "bias") else 0
        ref.check("d" + name, got["d" + name], *expected[2 + i], 2 * terms + more)
        assert got["d" + name].dtype == t[name].dtype
    with torch.no_grad():
        plain, after = selective_scan(*t.values(), softplus, before, return_state=True)
    ref.check("y without gradients", plain, *expected[0], terms)
    ref.check("state", after, *expected[1], terms)


def test_cases_have_one_chunk_and_several():
    chunks = {-(-l // chunk_tokens(l, c, n, backward)) > 1 for n, l, c, *_ in CASES for backward in (False, True)}
    assert chunks == {False, True}


@pytest.mark.parametrize("dtype,s", [(FLOAT, 16), (HALF, 5)])
def test_pieces_and_steps_go_on_from_the_state(dtype, s):
    t, before, _ = _tensors(3, 45, 20, s, dtype, gate=s == 16, softplus=s == 16, state=True)
    softplus = s == 16
    expected = ref.scan(*t.values(), softplus, before, None)

    def part(first, last):
        return [v if k in ("A", "D", "bias") or v is None else v[:, first:last] for k, v in t.items()]

    first, state = selective_scan(*part(0, 40), softplus, before, return_state=True)
    second, state = selective_scan(*part(40, 41), softplus, state, return_state=True)
    rows = [first, second]
    for at in range(41, 45):
        u, *rest = [v if v is None or v.dim() < 3 else v[:, 0] for v in part(at, at + 1)]
        kept = state.clone()
        if at % 2:
            other = torch.full_like(state, float("nan"))
            rows.append(selective_scan_step(u, state, *rest, softplus, out_state=other)[:, None])
            assert torch.equal(state, kept)  # only out_state is written
            state = other
        else:
            rows.append(selective_scan_step(u, state, *rest, softplus)[:, None])
    ref.check("pieces", torch.cat(rows, 1), *expected[0], 3 * 45 + s + 80)
    ref.check("state", state, *expected[1], 3 * 45 + s + 80)


@pytest.mark.parametrize("s,dtype", [(1, BF16), (4, FLOAT), (7, FLOAT), (32, HALF)])
def test_step(s, dtype):
    """Numbers of states that are one lane's and several's, whole and odd."""
    t, before, _ = _tensors(5, 1, 37, s, dtype, state=True)
    expected = ref.scan(*t.values(), True, before, None)
    u, *rest = [v if v is None or v.dim() < 3 else v[:, 0] for v in t.values()]
    y = selective_scan_step(u, before, *rest, True)
    ref.check("y", y, expected[0][0][:, 0], expected[0][1][:, 0], s + 80)
    ref.check("state", before, *expected[1], 80)


def test_gradients_against_differences():
    """The gradients of a sum of the outputs against differences of that sum in 64 bits, at 0.001 to both sides."""
    t, _, dy = _tensors(1, 9, 3, 5, FLOAT, gate=True, softplus=True)
    got = _train(t, True, None, dy)
    rows = {k: v.detach().cpu().double() for k, v in t.items()}

    def total(values):
        return float((ref.scan(*values.values(), True, None, None)[0][0] * dy.cpu().double()).sum())

    g = torch.Generator().manual_seed(1)
    for name in NAMES:
        direction = torch.randn(rows[name].shape, generator=g).double()
        up, down = ({k: v + e * direction if k == name else v for k, v in rows.items()} for e in (1e-3, -1e-3))
        slope = (total(up) - total(down)) / 2e-3
        along = float((got["d" + name].cpu().double() * direction).sum())
        scale = float((got["d" + name].cpu().double().abs() * direction.abs()).sum())
        # third derivatives of products of exponentials of order one, times a millionth / 6
        assert abs(slope - along) <= 2e-5 * scale + 1e-6, (name, slope, along)


def test_python_path_is_the_same():
    t, before, dy = _tensors(2, 90, 70, 16, BF16, state=True)
    native = _train(t, True, before, dy)
    u, *rest = [v if v.dim() < 3 else v[:, 0] for v in t.values()]
    state, other = before.clone(), before.clone()
    stepped = selective_scan_step(u, state, *rest, True)
    bypass = Bypass()
    try:
        python = _train(t, True, before, dy)
        again = selective_scan_step(u, other, *rest, True)
    finally:
        bypass.release()
    assert all(torch.equal(native[k], python[k]) for k in native)
    assert torch.equal(stepped, again) and torch.equal(state, other)
    assert all(torch.equal(v, native[k]) for k, v in _train(t, True, before, dy).items())  # no order of atomics


def test_what_is_not_finite_stays_with_its_channel():
    """... of the tensors that have channels: sums over channels have it at their token."""
    t, _, dy = _tensors(2, 37, 70, 16, FLOAT)
    clean = _train(t, True, None, dy)
    t["u"][0, 36, 69] = float("inf")  # the last token of a part of a tile, the last channel of a part of a wave
    t["gate"][1, 20, 3] = float("nan")
    got = _train(t, True, None, dy)
    for name in ("y", "du", "ddelta", "dgate"):
        same = got[name] == clean[name]
        assert same[0, :, :69].all() and same[1, :, :3].all() and same[1, :, 4:].all(), name
    assert (got["y"] == clean["y"])[0, :36].all()
    assert (got["dC"] == clean["dC"])[0, :36].all() and not got["dB"][0, 36].isnan().any()
    assert (got["dA"] == clean["dA"])[4:69].all()


def test_large_time_steps_and_rates():
    """Steps of 0 and of 100, rates that decay at once and that grow."""
    t, _, dy = _tensors(1, 20, 10, 5, FLOAT, gate=False, D=False, bias=False, softplus=False)
    t["delta"][0, ::3], t["delta"][0, 1::7] = 0.0, 100.0
    t["A"][0] = -1e4
    t["A"][1] = 1e-3
    expected = ref.scan(*t.values(), False, None, dy)
    got = _train(t, False, None, dy)
    ref.check("y", got["y"], *expected[0], 3 * 20 + 100)
    for i, name in enumerate(NAMES):
        if t[name] is not None:
            # (rates of 1e-3 over steps of 100 make exponents of up to a tenth a token)
            ref.check("d" + name, got["d" + name], *expected[2 + i], 2 * (3 * 20 + 100) + 30)


def test_softplus_of_far_values():
    delta = torch.tensor([-200.0, -90.0, -20.0, -7.0, -1e-3, 0.0, 1e-3, 7.0, 20.0, 90.0, 200.0], device="cuda")
    zero, one = torch.zeros(11, 1, device="cuda"), torch.ones(1, 1, device="cuda")
    state = torch.zeros(1, 11, 1, device="cuda")
    y = selective_scan_step(torch.ones(1, 11, device="cuda"), state, delta[None], zero, one, one, delta_softplus=True)  # the step itself
    d = delta.cpu().double()
    expected = torch.log1p(torch.exp(-d.abs())) + d.clamp_min(0)
    # the exponential's argument is off by two units of itself; numbers below the normal ones are zero
    assert ((y[0].cpu().double() - expected).abs() <= (8 + 2 * d.abs()) * 2.0**-24 * expected + 2.0**-126).all()


def test_empty():
    for n, l in ((0, 4), (2, 0)):
        t, before, dy = _tensors(n, l, 16, 5, HALF, state=True)
        got = _train(t, True, before, dy)
        assert got["y"].shape == got["du"].shape == (n, l, 16) and got["dB"].shape == (n, l, 5)
        assert not got["dA"].any() and not got["dD"].any() and not got["dbias"].any()
        y, state = selective_scan(*t.values(), True, before, return_state=True)
        assert torch.equal(state, before)


def test_refusals():
    t, before, dy = _tensors(2, 5, 16, 5, HALF, state=True)
    for change in (
        {"delta": t["delta"].float()}, {"delta": t["delta"][:, :4]}, {"A": t["A"].cpu()}, {"A": t["A"][:8]},
        {"A": torch.zeros(16, 33, device="cuda")}, {"B": t["B"][..., :4]}, {"C": t["C"].float()}, {"D": t["D"][:3]},
        {"gate": t["gate"][..., :8]}, {"bias": t["bias"].long()}, {"u": t["u"].double(), "delta": t["delta"].double()},
    ):  # fmt: skip
        with pytest.raises(AssertionError):
            selective_scan(*{**t, **change}.values(), True)
    for state in (before.half(), before[:1], before[..., :4], before.cpu()):
        with pytest.raises(AssertionError):
            selective_scan(*t.values(), True, state)
    with pytest.raises(RuntimeError):
        selective_scan(*t.values(), True, before.clone().requires_grad_())
    u, *rest = [v if v.dim() < 3 else v[:, 0] for v in t.values()]
    flat = torch.zeros(2 * 16 * 5 + 4, device="cuda")
    for state, out in ((before, before.half()), (flat[:160].view(2, 16, 5), flat[4:].view(2, 16, 5)),
                       (flat[1:161].view(2, 16, 5), None), (before.transpose(0, 1).contiguous().transpose(0, 1), None)):  # fmt: skip
        with pytest.raises(AssertionError):
            selective_scan_step(u, state, *rest, True, out_state=out)
    leaf = t["u"].clone().requires_grad_()
    y = selective_scan(leaf, *list(t.values())[1:], True)
    (dx,) = torch.autograd.grad(y, leaf, dy.clone().requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivatives
        torch.autograd.grad(dx.sum(), leaf)


def test_opcheck_and_compile():
    t, before, dy = _tensors(2, 9, 16, 5, HALF)
    leaves = [v.clone().requires_grad_() for v in t.values()]
    torch.library.opcheck(selective_scan_forward, (*leaves, True, None, False, True))
    state = torch.zeros(2, 16, 5, device="cuda")
    u, *rest = [v if v.dim() < 3 else v[:, 0] for v in t.values()]
    torch.library.opcheck(selective_scan_step_op, (u, state, *rest, True, state.clone()))
    compiled = torch.compile(lambda *a: selective_scan(*a, True), backend="aot_eager")
    got = torch.autograd.grad(compiled(*leaves), leaves, dy)
    expected = _train(t, True, before, dy)
    assert all(torch.equal(a, expected["d" + k]) for a, k in zip(got, NAMES))


def test_captured():
    """A training step and a token of decoding, captured, replayed on other inputs with eager work between."""
    t, before, dy = _tensors(2, 90, 70, 16, BF16, state=True)
    static, state = {k: v.clone() for k, v in t.items()}, before.clone()
    step = lambda t, state: selective_scan_step(t["u"][:, 0], state, t["delta"][:, 0], t["A"], t["B"][:, 0], t["C"][:, 0], t["D"],
                                                t["gate"][:, 0], t["bias"], True)  # fmt: skip  # noqa: E731
    _train(static, True, before, dy)  # plans and kernels are made outside
    step(static, before.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _train(static, True, before, dy)
        stepped = step(static, state)
    eager_state = state.clone()
    for seed in range(3):
        fresh = _tensors(2, 90, 70, 16, BF16, seed=seed + 1)[0]
        for k, v in fresh.items():
            static[k].copy_(v)
        graph.replay()
        expected = _train(fresh, True, before, dy)
        again = step(fresh, eager_state)
        torch.cuda.synchronize()
        assert all(torch.equal(out[k], expected[k]) for k in out)
        assert torch.equal(stepped, again) and torch.equal(state, eager_state)


def test_layer():
    torch.manual_seed(0)
    layer = SelectiveScan(24, 5).cuda()
    x, delta, gate = torch.randn(3, 2, 6, 24, device="cuda")
    B, C = torch.randn(2, 2, 6, 5, device="cuda")
    whole = layer(x, delta, B, C, gate)
    whole.sum().backward()
    assert layer.log_rates.grad.shape == (24, 5) and layer.D.grad.shape == layer.delta_bias.grad.shape == (24,)
    state = layer.empty_state(2)
    with torch.no_grad():
        rows = torch.stack([layer.step(x[:, t], state, delta[:, t], B[:, t], C[:, t], gate[:, t]) for t in range(6)], 1)
    torch.testing.assert_close(rows, whole.detach(), rtol=1e-5, atol=1e-6)
