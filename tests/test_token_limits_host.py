"""Limits of the operators over sequences of tokens that their documentation names.  CPU only."""

import pytest
import torch

from spio_amd.functional import head_norm_rotary, rotary, rotary_frequencies

Q, W, POSITIONS, FREQUENCIES = torch.zeros(2, 5, 4, 32), torch.ones(32), torch.arange(5), rotary_frequencies(32)


@pytest.mark.parametrize("scale", [1e39, -1e39, float("inf"), float("nan"), 3.4028236e38])
def test_scales_that_are_no_float32_numbers_are_refused(scale):
    """The kernels multiply in float32: a sine of zero would be NaN times such a scale."""
    with pytest.raises(AssertionError, match="scale"):
        rotary(Q, Q, POSITIONS, FREQUENCIES, scale=scale)
    with pytest.raises(AssertionError, match="scale"):
        head_norm_rotary(Q, Q, W, W, POSITIONS, FREQUENCIES, scale=scale)


@pytest.mark.parametrize("scale", [0, 1e-300, -3.4028234e38])
def test_smallest_and_largest_scales_are_taken(scale):
    with pytest.raises(ValueError, match="GPU only"):
        rotary(Q, Q, POSITIONS, FREQUENCIES, scale=scale)
