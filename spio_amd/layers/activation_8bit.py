"""An activation that keeps its input for the backward pass in 8 bits."""

import torch
from torch import nn

from ..functional.activation_8bit_function import POINTWISE, activation_8bit
from ..kernels.group_norm_2d_kernel import DTYPES
from .group_norm_2d import TORCH_ACTIVATIONS


class Activation8bit(nn.Module):
    """`nn.ReLU`, `nn.SiLU` or `nn.GELU` (activation "relu", "silu", "gelu") on GPU tensors of float16, bfloat16 or
    float32; what the backward pass needs of these is kept in 8 bits a value, of relu's in one.  Tensors elsewhere and of
    other types take torch's function, which is the same and keeps its input as it is."""

    def __init__(self, activation="gelu"):
        super().__init__()
        if activation not in POINTWISE:
            raise ValueError(f"activation must be one of {POINTWISE}, not {activation!r}")
        self.activation = activation

    def extra_repr(self) -> str:
        return self.activation

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.is_cuda and x.dtype in DTYPES:
            return activation_8bit(x, self.activation)
        return TORCH_ACTIVATIONS[self.activation](x)
