"""Norms of the heads of queries and keys and their rotation by position."""

import torch
from torch import nn

from ..functional.head_norm_rotary_function import head_norm_rotary, rotary, rotary_frequencies


class HeadNormRotary(nn.Module):
    """`head_norm_rotary`, or with norm=False `rotary`, of (N, L, heads, channels) queries and keys, with its weights (channels,)
    and frequencies, which `rotary_frequencies` makes of the first `rotated` channels (default: all) and `scaling`, its
    further arguments.  Positions default to 0, 1, ...
    """

    def __init__(self, channels, rotated=None, norm=True, eps=1e-6, interleaved=False, scale=1.0, device=None, dtype=None,
                 **scaling):  # fmt: skip
        super().__init__()
        self.channels, self.eps, self.interleaved, self.scale = channels, eps, interleaved, scale
        for name in ("q_weight", "k_weight"):
            weight = nn.Parameter(torch.ones(channels, device=device, dtype=dtype)) if norm else None
            self.register_parameter(name, weight)
        self.scaling = dict(channels=channels if rotated is None else rotated, **scaling)
        self.register_buffer("frequencies", rotary_frequencies(**self.scaling, device=device), persistent=False)

    def _apply(self, fn, recurse=True):
        """Frequencies go with the module to a device, but stay float64 where it is cast; those of a module without memory
        (the meta device) are made again."""
        frequencies = rotary_frequencies(**self.scaling) if self.frequencies.is_meta else self.frequencies
        super()._apply(fn, recurse)
        self.frequencies = frequencies.to(self.frequencies.device)
        return self

    def extra_repr(self) -> str:
        return f"{self.channels}, pairs={len(self.frequencies)}, norm={self.q_weight is not None}, interleaved={self.interleaved}"

    def forward(self, q: torch.Tensor, k: torch.Tensor, positions=None):
        if positions is None:
            positions = torch.arange(q.shape[1], device=q.device)
        if self.q_weight is None:
            return rotary(q, k, positions, self.frequencies, self.interleaved, self.scale)
        return head_norm_rotary(q, k, self.q_weight, self.k_weight, positions, self.frequencies, self.eps, self.interleaved,
                                self.scale)  # fmt: skip
