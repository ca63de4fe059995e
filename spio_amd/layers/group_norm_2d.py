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
    everything else takes torch's group_norm (with weight and bias outside it where its gradients of them would be wrong)
    and activation, which are the same function.  `checkpoint_8bit` keeps the kernels' input for the backward pass in 8 bits.
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
        return TORCH_ACTIVATIONS[self.activation](self._torch_group_norm(x))

    def _torch_group_norm(self, x: torch.Tensor) -> torch.Tensor:
        """torch's group_norm.  On the GPU its gradients of weight and bias are wrong here for more than 128 images (float32
        200n 9c 5x4 is off by 0.4 of the largest, 128n by 2e-7), so that these are applied to its normalised values then."""
        wants_sums = self.affine and torch.is_grad_enabled() and (self.weight.requires_grad or self.bias.requires_grad)
        if not (x.is_cuda and x.dim() > 1 and x.shape[0] > 128 and wants_sums):
            return F.group_norm(x, self.num_groups, self.weight, self.bias, self.eps)
        narrow = x.dtype in (torch.float16, torch.bfloat16)
        y = F.group_norm(x.float() if narrow else x, self.num_groups, None, None, self.eps)
        shape = (1, self.num_channels) + (1,) * (x.dim() - 2)
        y = torch.addcmul(self.bias.to(y.dtype).view(shape), y, self.weight.to(y.dtype).view(shape))
        return y if torch.is_autocast_enabled("cuda") else y.to(x.dtype)
