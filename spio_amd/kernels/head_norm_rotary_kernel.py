"""Rotary positions with or without a norm of every head (csrc/head_norm_rotary.hip): parameters, factories, grids.

Specialised by type, channels of a head and layout of the pairs; everything else is an argument (SpioRotaryArgs).
"""

from dataclasses import dataclass

from ..util.math import divup
from .group_norm_2d_kernel import DTYPE_NAMES
from .kernel import KernelSpec
from .kernel_factory import KernelFactory
from .launch_params import LaunchParams

SOURCE = "head_norm_rotary.hip"
MAX_HEAD = 256
THREADS = 256
# Workgroups of a backward pass with norms, each of which leaves a row of sums: two a compute unit (4n 2048l 24q 8k 128d 48 us,
# with 1024 as long and twice the rows)
SUMMED_WORKGROUPS = 512


def lanes_of(head: int, norm: bool) -> int:
    """Lanes of a head: one for two units of eight channels, with norms, whose sums cross them, a power of two."""
    return divup(head, 16) if not norm else 1 << (divup(head, 16) - 1).bit_length()


def parts_of(tokens: int, heads: int, head: int, norm: bool) -> int:
    """Parts that the heads of a token are split into: lanes that share a token's cosines take every parts-th head.  A power
    of two, for four to seven heads a lane (us with 1, 2, 4 and 8 parts, forward: 2n 4097l 16 heads of 80 channels 34, 32,
    28, 28; 4n 2048l 24q 8k 128d with norms 37, 36, 37, 38, backward 49, 49, 48, 51; 1n 16385l 32q 8k 81, 74, 73, 73; 400
    tokens, 24q 8k 13.9, 10.4, 9.6, 11.7).  Two heads a lane where all lanes then are fewer waves than compute units, as
    with one token a sequence (8n 12q 12k 64d with 2, 4, 6 parts 5.6, 5.0, 4.2; 8n 32q 8k 128d with norms, 8 and 16, 6.1 and
    5.2)."""
    most = divup(heads, 2)
    if divup(tokens * lanes_of(head, norm), 64) * most < 256:
        return most
    return 1 << max(0, (heads // 4).bit_length() - 1)


def grid_of(tokens: int, parts: int, head: int, norm: bool, summed: bool) -> int:
    grid = divup(tokens * parts, THREADS // lanes_of(head, norm))
    return min(grid, SUMMED_WORKGROUPS) if summed else grid


@dataclass(frozen=True)
class HeadNormRotaryParams:
    """Channels of a head, the number of the tensors' type, whether heads are normed, and whether pairs are neighbours."""

    head: int
    dtype: int = 0
    norm: bool = True
    interleaved: bool = False

    def encode(self) -> str:
        return f"{self.head}d_{DTYPE_NAMES[self.dtype]}_{'norm' if self.norm else 'turn'}" + ("_pairs" if self.interleaved else "")

    def validate(self):
        assert self.head % 8 == 0 and 8 <= self.head <= MAX_HEAD and 0 <= self.dtype <= 2


@dataclass(frozen=True)
class HeadNormRotaryConfig:
    """Heads that a lane requests at once (4n 2048l 24q 8k 128d with norms, forward and backward, us: one 39 and 49, two 37 and
    48, four 38 and 60)."""

    heads: int = 2


def _spec(mode):
    def spec(params: HeadNormRotaryParams, config: HeadNormRotaryConfig, _device_attr=None) -> KernelSpec:
        params.validate()
        defines = {"SPIO_MODE": mode, "SPIO_HEAD": params.head, "SPIO_DTYPE": params.dtype, "SPIO_NORM": int(params.norm),
                   "SPIO_INTERLEAVED": int(params.interleaved), "SPIO_HEADS": config.heads}  # fmt: skip
        return KernelSpec(defines, LaunchParams(grid=1, block=THREADS), SOURCE, takes_structure=True)

    return spec


def _factory(name, mode):
    return KernelFactory(
        HeadNormRotaryParams,
        HeadNormRotaryConfig,
        None,
        kernel_name=name,
        configs=lambda params, device_attr=None: [HeadNormRotaryConfig()],
        kernel_spec=_spec(mode),
        args_checker=None,
    )


head_norm_rotary_kernel_factory = _factory("spio_head_norm_rotary", 0)
head_norm_rotary_bwd_kernel_factory = _factory("spio_head_norm_rotary_bwd", 1)
head_norm_rotary_sums_kernel_factory = _factory("spio_head_norm_rotary_sums", 2)
