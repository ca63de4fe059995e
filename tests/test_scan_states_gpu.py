"""selective_scan and selective_scan_step on the GPU with numbers of states that are not 16: odd ones, whose last state has no
partner in the other half of a wave, those of other tiles, and idle lanes of a step."""

import pytest
import torch

from spio_amd.functional.selective_scan_function import selective_scan_backward, selective_scan_forward
from tests.test_selective_scan_gpu import FLOAT, _tensors

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
