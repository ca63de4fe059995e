"""The selective scan of a state-space layer with its own parameters."""

import math

import torch
from torch import nn

from ..functional.selective_scan_function import selective_scan, selective_scan_step
from ..kernels.selective_scan_kernel import MAX_STATES


class SelectiveScan(nn.Module):
    """`selective_scan` with its parameters in float32: rates A = -exp(log_rates) (channels, states), the skip D and the
    bias of the time steps (channels,), which are softplus of delta and that bias.

    `forward` takes (N, L, C) inputs, delta and gate and (N, L, states) B and C; `step` the same of one token a sequence and
    the state that it updates in place, which `forward(..., return_state=True)` or `empty_state` makes.
    """

    def __init__(self, channels, states=16, min_step=1e-3, max_step=0.1, device=None):
        super().__init__()
        if channels < 1 or not 1 <= states <= MAX_STATES:
            raise ValueError(f"channels must be positive, states 1 to {MAX_STATES}")
        if not 0 < min_step <= max_step:
            raise ValueError("min_step must be positive and at most max_step")
        self.channels, self.states = channels, states
        rates = torch.arange(1, states + 1, dtype=torch.float32, device=device).log()
        self.log_rates = nn.Parameter(rates.repeat(channels, 1))
        self.D = nn.Parameter(torch.ones(channels, dtype=torch.float32, device=device))
        steps = torch.empty(channels, dtype=torch.float32, device=device).uniform_(math.log(min_step), math.log(max_step)).exp()
        self.delta_bias = nn.Parameter(steps + torch.log(-torch.expm1(-steps)))  # softplus of which the steps are

    def extra_repr(self) -> str:
        return f"{self.channels}, states={self.states}"

    def empty_state(self, sequences) -> torch.Tensor:
        """The state before the first token."""
        return self.D.new_zeros((sequences, self.channels, self.states), dtype=torch.float32).detach()

    def forward(self, x, delta, B, C, gate=None, initial_state=None, return_state=False):
        return selective_scan(x, delta, -self.log_rates.float().exp(), B, C, self.D, gate, self.delta_bias, True, initial_state,
                              return_state)  # fmt: skip

    def step(self, x, state, delta, B, C, gate=None) -> torch.Tensor:
        return selective_scan_step(x, state, delta, -self.log_rates.float().exp(), B, C, self.D, gate, self.delta_bias, True)
