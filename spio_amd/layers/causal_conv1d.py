"""A short causal convolution along the tokens, each channel by itself."""

import math

import torch
from torch import nn

from ..functional.causal_conv1d_function import causal_conv1d, causal_conv1d_step
from ..kernels.causal_conv1d_kernel import ACTIVATIONS, MAX_WIDTH, MIN_WIDTH


class CausalConv1d(nn.Module):
    """`causal_conv1d` with its filters: weight (channels, width), the last tap the token's own, and bias (channels,).

    `forward` takes (N, L, C) GPU tensors; `step` the next token of every sequence and the state that it updates in place,
    which `forward(..., return_state=True)` or `empty_state` makes.
    """

    def __init__(self, channels, width, bias=True, activation="none", device=None, dtype=None):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, not {activation!r}")
        if not MIN_WIDTH <= width <= MAX_WIDTH or channels < 8 or channels % 8:
            raise ValueError(f"width must be {MIN_WIDTH} to {MAX_WIDTH}, channels a multiple of 8")
        self.channels, self.width, self.activation = channels, width, activation
        self.weight = nn.Parameter(torch.empty((channels, width), device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.empty((channels,), device=device, dtype=dtype)) if bias else None
        self.reset_parameters()

    def reset_parameters(self):
        limit = 1 / math.sqrt(self.width)
        nn.init.uniform_(self.weight, -limit, limit)
        if self.bias is not None:
            nn.init.uniform_(self.bias, -limit, limit)

    def extra_repr(self) -> str:
        return f"{self.channels}, {self.width}, bias={self.bias is not None}, activation={self.activation}"

    def empty_state(self, sequences, dtype=None) -> torch.Tensor:
        """The state before the first token."""
        return self.weight.new_zeros((sequences, self.width - 1, self.channels), dtype=dtype).detach()

    def forward(self, x: torch.Tensor, initial_state=None, return_state=False):
        return causal_conv1d(x, self.weight, self.bias, self.activation, initial_state, return_state)

    def step(self, x: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
        return causal_conv1d_step(x, state, self.weight, self.bias, self.activation)
