"""Limits of the operators over sequences of tokens that their documentation names.  CPU only."""

import pytest
import torch

from spio_amd.functional import head_norm_rotary, rotary, rotary_frequencies
from spio_amd.kernels.causal_conv1d_kernel import slice_tokens
from spio_amd.util.math import divup

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


def test_rows_of_filter_sums():
    """Fewer than 4096 and the sequences together, and one at least of each."""
    for tokens in (1, 2, 3, 16, 17, 513, 2048, 4099, 100000, 5000000):
        for sequences in (1, 2, 127, 128, 4095, 4096, 8192, 65536):
            for channels in (8, 200, 2048):
                rows = sequences * divup(tokens, slice_tokens(tokens, channels, sequences, True))
                assert sequences <= rows < 4096 + sequences, (tokens, sequences, channels, rows)
