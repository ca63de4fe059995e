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
ENDS, OUT, ENDS_BACK = 0, 1, 2  # modes of the kernel


def tile_tokens(states: int) -> int:
    """Tokens of a tile: those whose states the backward pass holds in registers at once, and the distance of the states
    that the forward pass keeps for it.  Longer tiles keep less, but 16 states of five tokens and more have no room in half a
    SIMD's registers (4n 2048l 2048c backward: 239 us with 4 tokens, 275 with 5, 397 with 6, 542 with 8)."""
    return 8 if states <= 8 else 4


def chunk_tokens(tokens: int, channels: int, sequences: int, backward: bool) -> int:
    """Tokens of a chunk.  All of them where sequences and channels alone give most SIMDs a wave: a first pass over chunks
    costs as much as it brings then (forward, us whole and in chunks: 1024 waves 49 and 69, 1536 waves 115 and 142; backward
    1024 waves 138 and 134).  Else as many chunks as fill the device, whose SIMDs hold two waves of the backward pass,
    once or, where chunks then keep 48 tokens, twice (4n 2048l 2048c backward: 2048 waves 241 us, 4096 217), but
    none of fewer than 16 tokens."""
    waves = divup(channels, LANES) * sequences
    if waves >= (1024 if backward else 700):
        return tokens
    chunks = 4096 // waves
    if tokens < 48 * chunks:
        chunks = max(1, min(2048 // waves, tokens // 16))
    return divup(divup(tokens, chunks), 8) * 8


@dataclass(frozen=True)
class SelectiveScanParams:
    """States of a channel, the number of the tensors' type (group_norm_2d_kernel.DTYPES), and what the kernel does of what
    is optional: gate, softplus of the time steps, keeping states for the backward pass."""

    states: int
    dtype: int = 0
    gate: bool = False
    softplus: bool = False
    keep: bool = False

    def encode(self) -> str:
        flags = ("_gate" if self.gate else "") + ("_softplus" if self.softplus else "") + ("_keep" if self.keep else "")
        return f"{self.states}s_{DTYPE_NAMES[self.dtype]}{flags}"

    def validate(self):
        assert 1 <= self.states <= MAX_STATES and 0 <= self.dtype <= 2


@dataclass(frozen=True)
class SelectiveScanConfig:
    """Tokens of a tile, and how many of its last ones the backward pass holds the decays of, as many as the registers have
    room for (4n 2048l 2048c with 16 states: none 233 us, two 224, three 215, four, of which some are kept in memory, 238)."""

    tile: int
    held: int = 0


def _config(mode, params):
    """The tile between kept states where these are written or read, else eight tokens (1n 4099l 1536c 73.0 us, with four 75.1)."""
    if mode in (ENDS, ENDS_BACK) or (mode == OUT and not params.keep):
        return SelectiveScanConfig(8)
    return SelectiveScanConfig(tile_tokens(params.states), (3 - params.states % 2) * (8 < params.states <= 16))


def _spec(mode, threads):
    def spec(params: SelectiveScanParams, config: SelectiveScanConfig, _device_attr=None) -> KernelSpec:
        params.validate()
        defines = {"SPIO_MODE": mode, "SPIO_STATES": params.states, "SPIO_DTYPE": params.dtype, "SPIO_T": config.tile,
                   "SPIO_HELD": config.held, "SPIO_WAVES": 2 if params.states <= 16 else 1, "SPIO_GATE": int(params.gate),
                   "SPIO_SOFTPLUS": int(params.softplus), "SPIO_KEEP": int(params.keep)}  # fmt: skip
        return KernelSpec(defines, LaunchParams(grid=1, block=threads), SOURCE, takes_structure=True)

    return spec


def _factory(name, mode, threads):
    return KernelFactory(
        SelectiveScanParams,
        SelectiveScanConfig,
        None,
        kernel_name=name,
        configs=lambda params, device_attr=None: [_config(mode, params)],
        kernel_spec=_spec(mode, threads),
        args_checker=None,
    )


selective_scan_ends_kernel_factory = _factory("spio_selective_scan_ends", 0, 64)
selective_scan_kernel_factory = _factory("spio_selective_scan", 1, 64)
selective_scan_ends_bwd_kernel_factory = _factory("spio_selective_scan_ends_bwd", 2, 64)
selective_scan_bwd_kernel_factory = _factory("spio_selective_scan_bwd", 3, 64)
selective_scan_sums_kernel_factory = _factory("spio_selective_scan_sums", 4, 256)
selective_scan_step_kernel_factory = _factory("spio_selective_scan_step", 5, 256)
selective_scan_join_kernel_factory = _factory("spio_selective_scan_join", 6, 64)
selective_scan_join_bwd_kernel_factory = _factory("spio_selective_scan_join_bwd", 7, 64)
