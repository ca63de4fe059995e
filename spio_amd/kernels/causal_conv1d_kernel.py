"""Causal convolution along tokens (csrc/causal_conv1d.hip): parameters, factories, and how sequences are cut into slices.

Specialised by types, width and activation; everything else is an argument (SpioConv1dArgs), and the grid follows from it.
"""

from dataclasses import dataclass

from ..util.math import divup
from .group_norm_2d_kernel import DTYPE_NAMES
from .kernel import KernelSpec
from .kernel_factory import KernelFactory
from .launch_params import LaunchParams

SOURCE = "causal_conv1d.hip"
MIN_WIDTH, MAX_WIDTH = 2, 8
ACTIVATIONS = {"none": 0, "silu": 2}  # the numbers that group_norm_2d_kernel has for them
UNROLL = 4


def slice_tokens(tokens: int, channels: int, sequences: int, backward: bool) -> int:
    """Tokens that a lane walks along: as many as leave 2^17 lanes, from 4 to 32, or 16 to 256 backward, where a lane also leaves
    a row of sums and reads the tokens beside its slice again (us: 8n 2048l 2048c forward with 4, 8, 16, 32, 64 tokens 40, 30, 28,
    25, 24, backward with 16, 32, 64, 128 60, 53, 50, 81; 1n 2051l 1536c forward with 4, 8, 16, 32 8.2, 7.8, 8.7, 12.1); and so many
    that there are fewer rows of sums than 4096 and the sequences together, of which each leaves one at least: a lane stays
    within its sequence."""
    lanes = channels // 8 * sequences
    if backward:
        return max(16, min(256, divup(tokens * lanes, 1 << 17)), divup(tokens * sequences, 4096))
    return max(4, min(32, divup(tokens * lanes, 1 << 17)))


@dataclass(frozen=True)
class CausalConv1dParams:
    """Width and activation, and the numbers of the tensors' type and that of weight and bias."""

    width: int
    dtype: int = 0
    weight_dtype: int = 2
    activation: int = 0

    def encode(self) -> str:
        act = next(name for name, number in ACTIVATIONS.items() if number == self.activation)
        return f"{self.width}w_{DTYPE_NAMES[self.dtype]}_{DTYPE_NAMES[self.weight_dtype]}_{act}"

    def validate(self):
        assert MIN_WIDTH <= self.width <= MAX_WIDTH and 0 <= self.dtype <= 2 and 0 <= self.weight_dtype <= 2
        assert self.activation in ACTIVATIONS.values()


@dataclass(frozen=True)
class CausalConv1dConfig:
    """Tokens that a lane requests at once."""

    unroll: int = UNROLL


def _spec(mode, threads):
    def spec(params: CausalConv1dParams, config: CausalConv1dConfig, _device_attr=None) -> KernelSpec:
        params.validate()
        defines = {"SPIO_MODE": mode, "SPIO_WIDTH": params.width, "SPIO_DTYPE": params.dtype, "SPIO_WDTYPE": params.weight_dtype,
                   "SPIO_ACT": params.activation, "SPIO_UNROLL": config.unroll}  # fmt: skip
        return KernelSpec(defines, LaunchParams(grid=1, block=threads), SOURCE, takes_structure=True)

    return spec


def _factory(name, mode, threads):
    return KernelFactory(
        CausalConv1dParams,
        CausalConv1dConfig,
        None,
        kernel_name=name,
        configs=lambda params, device_attr=None: [CausalConv1dConfig()],
        kernel_spec=_spec(mode, threads),
        args_checker=None,
    )


causal_conv1d_kernel_factory = _factory("spio_causal_conv1d", 0, 256)
causal_conv1d_bwd_kernel_factory = _factory("spio_causal_conv1d_bwd", 1, 256)
causal_conv1d_sums_kernel_factory = _factory("spio_causal_conv1d_sums", 2, 256)
causal_conv1d_step_kernel_factory = _factory("spio_causal_conv1d_step", 3, 64)
