"""Calls of the operators over sequences of tokens as programs make them beside plain ones: limits on the native path."""

import pytest
import torch

from spio_amd import native
from spio_amd.functional import rotary, rotary_frequencies

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
