"""selective_scan and selective_scan_step on the GPU with numbers of states that are not 16: odd ones, whose last state has no
partner in the other half of a wave, those of other tiles, and idle lanes of a step."""

import pytest
import torch

from spio_amd.functional import selective_scan, selective_scan_step
from spio_amd.functional.selective_scan_function import selective_scan_backward, selective_scan_forward
from spio_amd.kernels.selective_scan_kernel import chunk_tokens
from tests import token_reference as ref
from tests.test_selective_scan_gpu import BF16, FLOAT, HALF, NAMES, _tensors, _train

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("s", [3, 5, 15])
def test_what_lies_behind_the_kept_states_is_not_read(s):
    """One tile of states, so that a row behind its last one is memory of somebody else: NaN in a tensor of which it is a part."""
    n, l, c = 1, 3, 70
    t, _, dy = _tensors(n, l, c, s, FLOAT)
    _, _, kept = selective_scan_forward(*t.values(), True, None, False, True)
    assert tuple(kept.shape) == (n, 1, s, c)
    expected = selective_scan_backward(dy, *t.values(), True, kept)
    memory = torch.full((kept.numel() + 2 * c,), float("nan"), device="cuda")
    part = memory[: kept.numel()].view(kept.shape)
    part.copy_(kept)
    got = selective_scan_backward(dy, *t.values(), True, part)
    assert all(a.isfinite().all() and torch.equal(a, b) for a, b in zip(got, expected))
    assert memory[kept.numel() :].isnan().all()


def test_chunks_whose_factor_no_number_holds():
    """Three chunks of 16 tokens, the states of which grow or decay by e^100 in the middle one: from 1e-30 and from 1e30 to numbers
    that are there, though the factor is not; gradients the same way back."""
    n, l, c, s = 1, 48, 2, 1
    assert [chunk_tokens(l, c, n, backward) for backward in (False, True)] == [16, 16]
    delta = torch.full((n, l, c), 1.0 / 64, device="cuda")
    delta[:, 16:32] = 6.25
    t = {"u": torch.zeros(n, l, c, device="cuda"), "delta": delta, "A": torch.tensor([[1.0], [-1.0]], device="cuda"),
         "B": torch.ones(n, l, s, device="cuda"), "C": torch.full((n, l, s), 0.75, device="cuda"), "D": None, "gate": None, "bias": None}  # fmt: skip
    before = torch.tensor([[[1e-30], [1e30]]], device="cuda")
    dy = torch.tensor([1e-30, 1e30], device="cuda").expand(n, l, c).contiguous()
    dy[:, :32] = 0.0
    expected = ref.scan(*t.values(), False, before, dy)
    got = _train(t, False, before, dy)
    # exponents of 100.5 in all: a product, a rate and a sum of time steps of them are off by half a unit each
    terms = 3 * l + s + 80 + 2 * 101
    ref.check("y", got["y"], *expected[0], terms)
    for i, name in enumerate(NAMES):
        if t[name] is not None:
            ref.check("d" + name, got["d" + name], *expected[2 + i], 2 * terms + l)
    assert got["y"][0, 40, 0] > 1e13 and 0 < got["y"][0, 40, 1] < 1e-12 and got["du"][0, 3, 0] > 1e11 and 0 < got["du"][0, 3, 1] < 1e-12


# Numbers of states with code of their own: tiles of eight tokens (up to 8 states) and of four; last decays held (9 to 16, odd
# ones one fewer) or none; one wave a SIMD (17 and more); odd ones; partly filled sums over lanes.  Lengths that end inside a
# tile, channels of parts of a wave; several chunks, and (more than 1023 sequences) one.
STATES = [
    (2, 37, 33, 8, FLOAT, True), (1, 85, 70, 9, FLOAT, True), (2, 41, 33, 12, BF16, False), (1, 67, 70, 15, FLOAT, True),
    (2, 35, 33, 17, FLOAT, True), (1, 53, 70, 31, HALF, False), (1, 50, 33, 3, FLOAT, True), (2, 39, 70, 21, FLOAT, False),
    (1025, 5, 33, 9, FLOAT, True), (1025, 7, 3, 15, FLOAT, False), (1025, 5, 33, 17, FLOAT, True), (1025, 11, 5, 8, FLOAT, False),
    (1025, 6, 5, 31, FLOAT, True), (1025, 9, 5, 12, HALF, False),
]  # fmt: skip


@pytest.mark.parametrize("n,l,c,s,dtype,softplus", STATES)
def test_outputs_and_gradients(n, l, c, s, dtype, softplus):
    t, before, dy = _tensors(n, l, c, s, dtype, softplus, True, True, softplus, True)
    assert (chunk_tokens(l, c, n, True) < l) == (n < 1024)
    expected = ref.scan(*t.values(), softplus, before, dy)
    got = _train(t, softplus, before, dy)
    # as for other numbers of states: three roundings a token in a state, sums over states; over channels in 32 bits; over a
    # chunk's tokens in 32 and the chunks' in 64
    terms = 3 * l + s + 80
    ref.check("y", got["y"], *expected[0], terms)
    for i, name in enumerate(NAMES):
        if t[name] is not None:
            more = c if name in "BC" else l if name in ("A", "D", "bias") else 0
            ref.check("d" + name, got["d" + name], *expected[2 + i], 2 * terms + more)
    with torch.no_grad():
        plain, after = selective_scan(*t.values(), softplus, before, return_state=True)
    ref.check("y without gradients", plain, *expected[0], terms)
    ref.check("state", after, *expected[1], terms)


@pytest.mark.parametrize("s,dtype", [(12, BF16), (17, FLOAT), (20, FLOAT), (3, HALF), (28, FLOAT)])
def test_step(s, dtype):
    """Lanes without states beside whole ones (12, 20, 28 states: three, five and seven of four and eight) and parts of one."""
    t, before, _ = _tensors(5, 1, 37, s, dtype, state=True)
    expected = ref.scan(*t.values(), True, before, None)
    u, *rest = [v if v is None or v.dim() < 3 else v[:, 0] for v in t.values()]
    y = selective_scan_step(u, before, *rest, True)
    ref.check("y", y, expected[0][0][:, 0], expected[0][1][:, 0], s + 80)
    ref.check("state", before, *expected[1], 80)
