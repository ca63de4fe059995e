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
SUMMED_WORKGROUPS = 512  # of a backward pass with norms, each of which leaves a row of sums


def lanes_of(head: int) -> int:
    """Lanes of a head: two units of eight channels each, a power of two."""
    lanes = 1
    while lanes * 16 < head:
        lanes *= 2
    return lanes


def parts_of(tokens: int, heads: int, head: int) -> int:
    """Parts that the heads of a token are split into: lanes that share a token's cosines take every parts-th head.  About
    eight heads a lane, fewer where waves are few (us with 1, 2, 4, 8 and 16 parts, forward: 2n 4097l 16 heads of 80
    channels 39, 32, 29, 31, 38; 1n 16385l 32q 8k 128d 90, 80, 77, 89, 113)."""
    waves = divup(tokens * lanes_of(head), 64)
    return min(divup(heads, 2), max(divup(heads, 8), divup(4096, waves)))


def grid_of(tokens: int, parts: int, head: int, summed: bool) -> int:
    grid = divup(tokens * parts * lanes_of(head), THREADS)
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
    """Heads that a lane requests at once: two, or one in a forward pass with norms, which so has registers for more waves
    (4n 2048l 24q 8k 128d 38 us, with two 41; without norms 2n 4097l 16q 16k 80d 39, with two 36)."""

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
        configs=lambda params, device_attr=None: [HeadNormRotaryConfig(1 if params.norm and mode == 0 else 2)],
        kernel_spec=_spec(mode),
        args_checker=None,
    )


head_norm_rotary_kernel_factory = _factory("spio_head_norm_rotary", 0)
head_norm_rotary_bwd_kernel_factory = _factory("spio_head_norm_rotary_bwd", 1)
head_norm_rotary_sums_kernel_factory = _factory("spio_head_norm_rotary_sums", 2)
