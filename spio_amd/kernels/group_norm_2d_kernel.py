"""Group norm with an activation over NHWC tensors: parameters, configurations, factories.

The kernels (csrc/group_norm_2d.hip, csrc/group_norm_2d_bwd.hip) are specialised by channels, groups, types and
activation, not by the number and size of the images, which are arguments: the names of the kernels leave those out, so
that the compiled code is one file for all that get the same configuration.

Arguments, forward:  (output, codes, exponents, stats, input, weight, bias, pixels, images)
          backward:  (sums, grad_input, input or codes, exponents, grad_output, stats, weight, bias, pixels, images)
`stats` is float32 [n][groups][2] (mean, rstd), `sums` float32 [2][c] (0 = grad_weight, 1 = grad_bias), absent where
there are neither.  Codes and exponents are the input in the 8-bit form of csrc/spio_pointwise.h (relu's exponents with a
bit a value more: kept_shapes).
"""

from dataclasses import dataclass
from math import gcd
from typing import List

import torch

from ..util.math import divup
from .kernel import KernelSpec
from .kernel_factory import KernelFactory
from .launch_params import LaunchParams

SOURCE = "group_norm_2d.hip"
BWD_SOURCE = "group_norm_2d_bwd.hip"
MAX_CHANNELS = 4096

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
DTYPE_NAMES = ("f16", "bf16", "f32")


@dataclass(frozen=True)
class GroupNorm2dParams:
    """One group norm: input [n, c, h, w] with channels_last strides; `dtype` and `activation` are the numbers of
    DTYPES and ACTIVATIONS; `kept`: the input is written (forward) or read (backward) in 8 bits."""

    n: int
    c: int
    h: int
    w: int
    groups: int
    dtype: int = 0
    activation: int = 0
    eps: float = 1e-5
    has_weight: bool = True
    has_bias: bool = True
    kept: bool = False

    def encode(self) -> str:
        """What the compiled code depends on besides the configuration, in characters of an identifier (eps as in
        LayerNorm2dParams).  Recorded choices are filed under it, so that one for images of another size may be found:
        the factories have no other configuration than the chosen one, and such a record is passed over."""
        eps = repr(float(self.eps)).replace(".", "p").replace("-", "m").replace("+", "")
        flags = ("w" if self.has_weight else "nw") + ("b" if self.has_bias else "nb") + ("_8bit" if self.kept else "")
        act = list(ACTIVATIONS)[self.activation]
        return f"{self.c}c_{self.groups}g_{DTYPE_NAMES[self.dtype]}_{act}_{eps}eps_{flags}"

    def validate(self):
        assert self.n > 0 and self.h > 0 and self.w > 0
        assert self.c % 8 == 0 and 0 < self.c <= MAX_CHANNELS, f"channels must be a multiple of 8 up to {MAX_CHANNELS}"
        assert self.groups > 0 and self.c % self.groups == 0, "channels must be a multiple of the groups"
        assert 0 <= self.dtype <= 2 and 0 <= self.activation <= 3 and 0 < self.eps < float("inf")
        assert self.pixels < 1 << 31, "at most 2^31 pixels an image"

    @property
    def pixels(self) -> int:
        return self.h * self.w

    @property
    def kernel_eps(self) -> float:
        """eps as the kernels add it: the nearest to it that float32 has a normal number for.  As less (or nothing) it would
        leave a group without a deviation an infinite rstd, and NaN."""
        info = torch.finfo(torch.float32)
        return min(max(float(self.eps), info.tiny), info.max)

    @property
    def shape(self):
        return (self.n, self.c, self.h, self.w)


@dataclass(frozen=True)
class GroupNorm2dConfig:
    """Threads of a workgroup, units of eight channels that a lane holds, channels of a workgroup, and whether images
    are cut into stretches of pixels (two launches) or held whole (one)."""

    threads: int
    units: int
    slice: int
    split: int


def _granule(params: GroupNorm2dParams) -> int:
    """Slices of an image are multiples of this many channels: whole groups, whole blocks of 32."""
    group = params.c // params.groups
    step = group * 32 // gcd(group, 32)
    return min(step, params.c)


def _lane_units(params: GroupNorm2dParams, width: int) -> int:
    """Lanes that a pixel's slice takes."""
    return divup(width // 8, 4) * 4 if params.kept else width // 8


def _rows(params: GroupNorm2dParams, threads: int, width: int) -> int:
    """Pixels that a workgroup's threads have one unit each of: all that there are lanes for, or, where that idles no
    more than a sixteenth of them, as many as make whole lines."""
    rows = threads // _lane_units(params, width)
    pixel = params.c * (4 if params.dtype == 2 else 2)
    lines = rows - rows % (128 // gcd(128, pixel))
    return lines if width == params.c and 16 * (rows - lines) <= rows else rows


def is_legal(params: GroupNorm2dParams, config: GroupNorm2dConfig) -> bool:
    return (
        config.threads in (256, 512, 1024)
        and 1 <= config.units <= 16
        and 0 < config.slice <= params.c
        and (config.slice == params.c or config.slice % _granule(params) == 0)
        and config.threads >= _lane_units(params, config.slice)
        and (config.split == 1 or _span(params, config) >= params.pixels)
    )


def _span(params: GroupNorm2dParams, config: GroupNorm2dConfig) -> int:
    """Pixels that a workgroup holds."""
    return _rows(params, config.threads, config.slice) * config.units


# How a configuration is chosen.  The times of its two kinds were fitted to sweeps of 200 shapes in both directions (1 to
# 256 images, 48 to 1280 channels, 5x5 to 224x224): a launch, and for every round of workgroups over the device what the
# units of a workgroup take.  us = LAUNCH + PER_UNIT * rounds * threads * units for whole images, us = LAUNCH +
# PER_UNIT * units of the tensor / compute units + PER_JOIN * (joins - 1) in stretches, where the input is read twice; both for
# 16-byte units.  Over 120 more random shapes the choice took 1.02 times the best of ten others on average, at most 1.39 (with
# stretches of four or five lengths; any number of units since, which _best_stretches measures).
# Whole images win where there are enough of them, us whole and in stretches: forward 128n 384c 14x14 9.5 and 12, 64n
# 128c 28x28 9.6 and 11.3, 8n 1280c 8x8 5.6 and 6.9, but 4n 256c 32x32 8.5 and 7.1, 64n 192c 20x20 with one group 9.4 and 8.9;
# backward 128n 384c 14x14 14.7 and 19.4, 32n 192c 28x28 float32 17.9 and 21.2, 64n 128c 28x28 13.8 and 14.7, but 4n 256c
# 32x32 15 and 7.6.
_WHOLE = {False: (3.3, 1.1e-3), True: (6.0, 1.65e-3)}  # forward; backward, whose sums over images are a launch
_STRETCHES = {False: (6.2, 1.75e-3, 0.67), True: (6.6, 3.0e-3, 0.39)}


def _shared_lines(params: GroupNorm2dParams, width: int, bwd: bool) -> float:
    """How much longer a pass takes where slices of `width` channels share lines of 128 bytes, which every one of them
    touches, or sectors of 32, which none can write whole.  Fitted to 450 measurements (45 shapes), all with workgroups in
    the order of gn::place, whose neighbours are on different XCDs.  us: 128n 384c 14x14 in slices of 96 channels 10.4, of
    192 9.5; with a checkpoint 64n 128c 28x28 in slices of 32 channels 15.6, of 64, half as many workgroups, 11.4; 103n 328c
    27x27 in slices of 64 75, in stretches 32.  Less where the caches hold it all: 10n 112c 10x10 in slices of 32 channels
    3.8, of 64 5.3."""
    if width == params.c:
        return 1.0
    value = 4 if params.dtype == 2 else 2
    pixel = params.c * value
    lines = 0 if width * value % 128 == 0 and pixel % 128 == 0 else 112 / (width * value)  # more than its own, of each
    code_lines = 0 if not params.kept or (width % 128 == 0 and params.c % 128 == 0) else 120 / width
    sectors, code_sectors = pixel % 32 != 0, params.kept and params.c % 32 != 0
    if bwd:
        more = 0.5 * lines + 0.1 * code_lines + 0.3 * code_sectors
    else:
        more = 0.42 * lines + 0.34 * code_lines + 0.36 * sectors + 0.24 * code_sectors
    return 1.0 + more * (0.3 if params.n * params.pixels * pixel < 8 << 20 else 1.0)


def _best_whole(params: GroupNorm2dParams, cus: int, bwd: bool):
    """(cost, configuration) that holds whole images, or None; the cost is rounds * threads * units."""
    wide = params.dtype == 2
    # units in a lane's registers, of which 1024 threads have 128 each: 8 backward and 4 forward (16-bit types)
    most = ((8, 3) if wide else (13, 5)) if bwd else ((12, 6) if wide else (16, 12))
    granule = _granule(params)
    gelu = 1.25 if params.activation == 3 and not bwd else 1.0
    best = None
    for width in [*range(granule, params.c, granule), params.c]:
        lanes = _lane_units(params, width)
        groups = params.n * divup(params.c, width)
        shared = _shared_lines(params, width, bwd)
        for threads in (256, 512, 1024) if groups >= 2 * cus else (512, 256, 1024):
            if threads < lanes:
                continue
            units = divup(params.pixels, _rows(params, threads, width))
            if units > most[threads == 1024]:
                continue
            # a workgroup is faster where others leave it more of the memory's rate, and slower by gelu's instructions
            cost = divup(groups, cus) * threads * units * shared * (0.7 + 0.3 * min(1.0, groups / cus)) * gelu
            if best is None or cost < best[0]:
                best = (cost, GroupNorm2dConfig(threads, units, width, 0))
    return best


def _joins(params: GroupNorm2dParams, config: GroupNorm2dConfig) -> int:
    """Times that a lane of the second launch waits for partial results: the lanes of a group load those of four
    stretches each at once."""
    lanes = 64
    while lanes > 1 and lanes * params.groups > config.threads:
        lanes //= 2
    return divup(params.groups, config.threads // lanes) * divup(params.pixels, _span(params, config) * 4 * lanes)


def _best_stretches(params: GroupNorm2dParams, cus: int, bwd: bool) -> GroupNorm2dConfig:
    """The stretch that leaves the least of the last round of workgroups idle; a workgroup costs what 256 units do
    besides its own, and one of 512 threads takes 8 % longer where the input is kept (128n 96c 56x56 backward 61 and 65 us,
    23n 112c 110x110 81 and 84).  Over 46 shapes it is within 1 % of the best on average, 12 % at worst.  With four
    or five lengths to choose from instead of all it was 3.5 % slower: backward 32n 256c 56x56 62.6 -> 53.4 us, 9n 296c 109x109
    67.2 -> 54.4.  The forward pass holds its units, the backward pass lets them follow each other."""
    if bwd:
        kinds = [(t, u) for t in (256, 512) for u in range(16, 1, -1)]
    else:
        most = 8 if params.dtype == 2 else 12
        kinds = [(t, u) for t in (512, 256) for u in (8, 7, 6, 12, 11, 10, 9, 5, 4, 3, 2) if u <= most]
    best = None
    for threads, units in kinds:
        lanes = _lane_units(params, params.c)
        if threads < lanes:
            continue
        # no more units than stretches of equal length need
        rows = _rows(params, threads, params.c)
        stretches = divup(params.pixels, rows * units)
        units = divup(params.pixels, rows * stretches)
        grid = params.n * divup(params.pixels, rows * units)
        config = GroupNorm2dConfig(threads, units, params.c, 1)
        cost = divup(grid, cus) * (threads * units + 256) * (1.08 if params.kept and threads == 512 else 1.0)
        cost += (125 if bwd else 400) * (_joins(params, config) - 1)
        if best is None or cost < best[0]:
            best = (cost, config)
    return best[1]


def _choose(params: GroupNorm2dParams, device_attr, bwd: bool) -> List[GroupNorm2dConfig]:
    params.validate()
    cus = getattr(device_attr, "multiprocessor_count", 256) or 256
    whole, split = _best_whole(params, cus, bwd), _best_stretches(params, cus, bwd)
    if whole is not None:
        size = 2 if params.dtype == 2 else 1
        total = params.n * params.pixels * params.c / 8 / cus
        launch, per_unit = _WHOLE[bwd]
        launches, per_unit_twice, per_join = _STRETCHES[bwd]
        stretches = launches + per_unit_twice * size * total + per_join * (_joins(params, split) - 1)
        if launch + per_unit * size * whole[0] <= stretches:
            return [whole[1]]
    return [split]


def _get_configs(params: GroupNorm2dParams, device_attr=None) -> List[GroupNorm2dConfig]:
    return _choose(params, device_attr, False)


def _get_bwd_configs(params: GroupNorm2dParams, device_attr=None) -> List[GroupNorm2dConfig]:
    return _choose(params, device_attr, True)


def _defines(params: GroupNorm2dParams, config: GroupNorm2dConfig):
    return {
        "SPIO_GN_C": params.c, "SPIO_GN_GROUPS": params.groups, "SPIO_GN_SLICE": config.slice,
        "SPIO_GN_THREADS": config.threads, "SPIO_GN_UNITS": config.units, "SPIO_GN_SPLIT": config.split,
        "SPIO_GN_ROWS": _rows(params, config.threads, config.slice), "SPIO_GN_EPS": f"{params.kernel_eps!r}f",
        "SPIO_GN_HAS_WEIGHT": int(params.has_weight), "SPIO_GN_HAS_BIAS": int(params.has_bias),
        "SPIO_GN_KEPT": int(params.kept), "SPIO_DTYPE": params.dtype, "SPIO_ACT": params.activation,
    }  # fmt: skip


def _grid(params: GroupNorm2dParams, config: GroupNorm2dConfig):
    """(workgroups, stretches of an image)"""
    params.validate()
    assert is_legal(params, config), f"illegal configuration {config} of {params}"
    stretches = divup(params.pixels, _span(params, config)) if config.split else 1
    grid = params.n * stretches * divup(params.c, config.slice)
    assert (grid + 2 * params.c) * config.threads < 1 << 32, "more workgroups than a launch can have"
    return grid, stretches


def _get_kernel_spec(params: GroupNorm2dParams, config: GroupNorm2dConfig, _device_attr=None) -> KernelSpec:
    grid, stretches = _grid(params, config)
    launch = LaunchParams(grid=grid, block=config.threads)
    spec = KernelSpec(_defines(params, config), launch, SOURCE)
    if config.split:
        spec.workspace_bytes = params.n * params.groups * stretches * 8
        spec.workspace_arg = 3
        spec.epilogue_suffix = "_apply"
        spec.epilogue_launch_params = launch
        spec.epilogue_extra_args = (0, 1, 2, 4, 5, 6, 7, 8)
    return spec


def _get_bwd_kernel_spec(params: GroupNorm2dParams, config: GroupNorm2dConfig, _device_attr=None) -> KernelSpec:
    grid, stretches = _grid(params, config)
    affine = params.has_weight or params.has_bias
    launch = LaunchParams(grid=grid, block=config.threads)
    spec = KernelSpec(dict(_defines(params, config), SPIO_GN_AFFINE=int(affine)), launch, BWD_SOURCE)
    spec.overwrites_output = bool(config.split)  # grad_input and all sums are the second launch's
    adding = divup(2 * params.c, 32) if affine else 0
    rows = params.n * stretches * 2 * params.c * 4 if affine else 0
    if config.split:
        spec.workspace_bytes = rows + params.n * stretches * 2 * params.groups * 4
        spec.epilogue_suffix = "_apply"
        spec.epilogue_launch_params = LaunchParams(grid=grid + adding, block=config.threads)
        spec.epilogue_extra_args = (1, 2, 3, 4, 5, 6, 7, 8, 9)
    elif affine:
        spec.workspace_bytes = rows
        spec.epilogue_suffix = "_reduce"
        spec.epilogue_launch_params = LaunchParams(grid=adding, block=config.threads)
        spec.epilogue_extra_args = (9,)
    return spec


def _torch_dtype(params):
    return list(DTYPES)[params.dtype]


def _vectors(params, device):
    return [torch.randn(params.c, device=device) if there else None for there in (params.has_weight, params.has_bias)]


def _images(params, device):
    x = torch.randn(params.shape, device=device).to(_torch_dtype(params))
    return x.contiguous(memory_format=torch.channels_last)


def kept_shapes(n, c, h, w, activation=0):
    """Shapes of the codes and exponents of an input that is kept in 8 bits (channels innermost); relu's exponents are
    followed by a byte for every eight channels, whether the gradient of each output passes."""
    return (n, h, w, c), (n, h, w, divup(c, 32) + (c // 8 if activation == ACTIVATIONS["relu"] else 0))


def _make_test_args(params: GroupNorm2dParams, device):
    codes, exponents = (torch.empty(s, device=device, dtype=torch.uint8) if params.kept else None
                        for s in kept_shapes(*params.shape, params.activation))  # fmt: skip
    x = _images(params, device)
    stats = torch.empty((params.n, params.groups, 2), device=device)
    return (torch.empty_like(x), codes, exponents, stats, x, *_vectors(params, device), params.pixels, params.n)


def _make_bwd_test_args(params: GroupNorm2dParams, device):
    dy = _images(params, device)
    if params.kept:
        codes, exponents = kept_shapes(*params.shape, params.activation)
        x = torch.randint(0, 256, codes, device=device, dtype=torch.uint8)
        exponents = torch.full(exponents, 126, device=device, dtype=torch.uint8)
    else:
        x, exponents = _images(params, device), None
    stats = torch.ones((params.n, params.groups, 2), device=device)
    sums = torch.empty((2, params.c), device=device) if params.has_weight or params.has_bias else None
    return (sums, torch.empty_like(dy), x, exponents, dy, stats, *_vectors(params, device), params.pixels, params.n)


group_norm_2d_kernel_factory = KernelFactory(
    GroupNorm2dParams,
    GroupNorm2dConfig,
    None,
    kernel_name="spio_group_norm_2d",
    configs=_get_configs,
    kernel_spec=_get_kernel_spec,
    make_test_args=_make_test_args,
    args_checker=None,
)

group_norm_2d_bwd_kernel_factory = KernelFactory(
    GroupNorm2dParams,
    GroupNorm2dConfig,
    None,
    kernel_name="spio_group_norm_2d_bwd",
    configs=_get_bwd_configs,
    kernel_spec=_get_bwd_kernel_spec,
    make_test_args=_make_bwd_test_args,
    args_checker=None,
)
