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
    SIMD's registers (4n 2048l 2048c, backward and the forward pass that keeps, no decays held: with 4 tokens 231 and 99 us, with
    5 247 and 100, with 6 261 and 97, with 8 320 and 85)."""
    return 8 if states <= 8 else 4


def chunk_tokens(tokens: int, channels: int, sequences: int, backward: bool) -> int:
    """Tokens of a chunk.  All of them where sequences and channels alone give most of the 1024 SIMDs a wave, else as many chunks
    as fill the device, whose SIMDs hold two waves of the backward pass, once or, where chunks then keep 48 tokens, twice (4n
    2048l 2048c backward: 2048 waves 225 us, 4096 213), but none of fewer than 16 tokens.

    Sequences of 1024 tokens of 2048 channels, us whole / in the chunks of the second rule (two chunks from 1536 waves on):

        waves                        512           704            1024           1536
        16 states, a prompt          415 / 232     442 / 360      456 / 452      578 / 789
                   keeping states    582 / 289     604 / 416      649 / 567      762 / 885
                   backward          1041 / 517    1045 / 770     1059 / 1000    1478 / 1598
        8 states, a prompt           286 / 154     318 / 239      334 / 299      391 / 516
                   backward          732 / 349     731 / 514      744 / 668      993 / 1072
        32 states, a prompt          1096 / 519    1206 / 758     1218 / 982     1368 / 1365
                   backward          1888 / 1184   1903 / 1770    1908 / 2228    3814 / 3438
        1 state, a prompt            207 / 100     249 / 153      276 / 206      272 / 312
                   backward          500 / 228     507 / 318      529 / 425      625 / 594

    The borders, 700 waves forward and 1024 backward, are one for all numbers of states and on the side of whole sequences, which
    take no workspace: forward from 700 to 1023 waves chunks are faster by a fifth to two fifths, at 1024 by up to a quarter,
    backward at 1024 with up to 16 states by 6 to 20 %."""
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
    room for (4n 2048l 2048c with 16 states: none 231 us, one 224, two 220, three 213, four, of which some are kept in memory,
    236)."""

    tile: int
    held: int = 0


def _config(mode, params):
    """The tile between kept states where these are written or read, else eight tokens (1n 4099l 1536c, the call 73.0 us,
    with four 75.1)."""
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
