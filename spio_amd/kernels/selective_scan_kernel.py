"""Selective scan (csrc/selective_scan.hip): parameters, factories, and how sequences are cut into chunks.

Specialised by type and number of states; everything else is an argument (SpioScanArgs), and the grid follows from it.
"""

from dataclasses import dataclass

from ..util.math import divup
from .group_norm_2d_kernel import DTYPE_NAMES
from .kernel import KernelSpec
from .kernel_factory import KernelFactory
from .launch_params import LaunchParams

SOURCE = "selective_scan.hip"
MAX_STATES = 32
LANES = 64  # channels of a workgroup


def tile_tokens(states: int) -> int:
    """Tokens of a tile: those whose states the backward pass holds in registers at once, and the distance of the states
    that the forward pass keeps for it."""
    return 8 if states <= 8 else 6 if states <= 16 else 4


def chunk_tokens(tokens: int, channels: int, sequences: int, states: int) -> int:
    """Tokens of a chunk, whole tiles: all of them where sequences and channels alone give every SIMD a wave."""
    waves = divup(channels, LANES) * sequences
    tile = tile_tokens(states)
    chunks = max(1, min(1024 // waves, tokens // 32))
    return divup(divup(tokens, chunks), tile) * tile


@dataclass(frozen=True)
class SelectiveScanParams:
    """States of a channel, and the number of the tensors' type (group_norm_2d_kernel.DTYPES)."""

    states: int
    dtype: int = 0

    def encode(self) -> str:
        return f"{self.states}s_{DTYPE_NAMES[self.dtype]}"

    def validate(self):
        assert 1 <= self.states <= MAX_STATES and 0 <= self.dtype <= 2


@dataclass(frozen=True)
class SelectiveScanConfig:
    """Tokens of a tile."""

    tile: int


def _spec(mode, threads):
    def spec(params: SelectiveScanParams, config: SelectiveScanConfig, _device_attr=None) -> KernelSpec:
        params.validate()
        defines = {"SPIO_MODE": mode, "SPIO_STATES": params.states, "SPIO_DTYPE": params.dtype, "SPIO_T": config.tile,
                   "SPIO_WAVES": 2 if params.states <= 16 else 1}  # fmt: skip
        return KernelSpec(defines, LaunchParams(grid=1, block=threads), SOURCE, takes_structure=True)

    return spec


def _factory(name, mode, threads):
    return KernelFactory(
        SelectiveScanParams,
        SelectiveScanConfig,
        None,
        kernel_name=name,
        configs=lambda params, device_attr=None: [SelectiveScanConfig(tile_tokens(params.states))],
        kernel_spec=_spec(mode, threads),
        args_checker=None,
    )


selective_scan_ends_kernel_factory = _factory("spio_selective_scan_ends", 0, 64)
selective_scan_kernel_factory = _factory("spio_selective_scan", 1, 64)
selective_scan_ends_bwd_kernel_factory = _factory("spio_selective_scan_ends_bwd", 2, 64)
selective_scan_bwd_kernel_factory = _factory("spio_selective_scan_bwd", 3, 64)
selective_scan_sums_kernel_factory = _factory("spio_selective_scan_sums", 4, 256)
selective_scan_step_kernel_factory = _factory("spio_selective_scan_step", 5, 256)
