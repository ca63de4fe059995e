"""Group norm with an activation over NCHW tensors."""

import torch
from torch import nn
import torch.nn.functional as F

from ..functional.group_norm_2d_function import group_norm_2d
from ..kernels.group_norm_2d_kernel import ACTIVATIONS, DTYPES, MAX_CHANNELS

TORCH_ACTIVATIONS = {"none": lambda x: x, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}


class GroupNorm2d(nn.GroupNorm):
    """`nn.GroupNorm` followed by an activation ("none", "relu", "silu", "gelu"), in one pass over the tensor.

    GPU tensors [N, C, H, W] in float16, bfloat16 or float32 whose channel count is a multiple of 8 go through the
    `group_norm_2d` kernels (channels_last in memory, float32 arithmetic, the input's type out, under autocast too);
    everything else takes torch's group_norm and activation, which are the same function.  `checkpoint_8bit`
    keeps the kernels' input for the backward pass in 8 bits.
    """

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, device=None, dtype=None, activation="none",
                 checkpoint_8bit=False):  # fmt: skip
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, not {activation!r}")
        super().__init__(num_groups, num_channels, eps, affine, device, dtype)
        self.activation = activation
        self.checkpoint_8bit = checkpoint_8bit

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, activation={self.activation}, checkpoint_8bit={self.checkpoint_8bit}"

    def forward(self, x: torch.Tensor) -> torch.Tensor:  # pylint: disable=arguments-renamed
        if (x.is_cuda and x.dim() == 4 and x.dtype in DTYPES and x.shape[1] == self.num_channels
                and x.shape[1] % 8 == 0 and x.shape[1] <= MAX_CHANNELS and 0 < self.eps < float("inf")):  # fmt: skip
            return group_norm_2d(x, self.num_groups, self.weight, self.bias, self.eps, self.activation,
                                 self.checkpoint_8bit)  # fmt: skip
        y = F.group_norm(x, self.num_groups, self.weight, self.bias, self.eps)
        return TORCH_ACTIVATIONS[self.activation](y)
