"""Group norm with an activation over NHWC tensors: parameters, configurations, factories.

The kernels (csrc/group_norm_2d.hip, csrc/group_norm_2d_bwd.hip) are specialised by channels, groups, types and
activation, not by the number and size of the images, which are arguments: the names of the kernels leave those out, so
that the compiled code is one file for all of them.

Arguments, forward:  (output, codes, exponents, stats, input, weight, bias, pixels, images)
          backward:  (sums, grad_input, input or codes, exponents, grad_output, stats, weight, bias, pixels, images)
`stats` is float32 [n][groups][2] (mean, rstd), `sums` float32 [2][c] (0 = grad_weight, 1 = grad_bias), absent where
there are neither.  Codes and exponents are the input in the 8-bit form of csrc/spio_pointwise.h.
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
        """What the compiled code depends on, in characters of an identifier (eps as in LayerNorm2dParams)."""
        eps = repr(float(self.eps)).replace(".", "p").replace("-", "m").replace("+", "")
        flags = ("w" if self.has_weight else "nw") + ("b" if self.has_bias else "nb") + ("_8bit" if self.kept else "")
        act = list(ACTIVATIONS)[self.activation]
        return f"{self.c}c_{self.groups}g_{DTYPE_NAMES[self.dtype]}_{act}_{eps}eps_{flags}"

    def validate(self):
        assert self.n > 0 and self.h > 0 and self.w > 0
        assert self.c % 8 == 0 and 0 < self.c <= MAX_CHANNELS, f"channels must be a multiple of 8 up to {MAX_CHANNELS}"
        assert self.groups > 0 and self.c % self.groups == 0, "channels must be a multiple of the groups"
        assert 0 <= self.dtype <= 2 and 0 <= self.activation <= 3 and self.eps > 0
        assert self.pixels < 1 << 31, "at most 2^31 pixels an image"

    @property
    def pixels(self) -> int:
        return self.h * self.w

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
    return config.threads // _lane_units(params, config.slice) * config.units


def _choose(params: GroupNorm2dParams, cus: int, most: int, bwd: bool) -> GroupNorm2dConfig:
    """`most`: units that a lane holds without its registers running out at 1024 threads."""
    granule = _granule(params)
    widths = [w for w in range(granule, params.c, granule)] + [params.c]
    best = None
    for width in widths:
        lanes = _lane_units(params, width)
        for threads in (256, 512, 1024):
            if threads < lanes:
                continue
            units = divup(params.pixels, threads // lanes)
            if units <= (8 if threads < 1024 else most):
                groups = params.n * divup(params.c, width)
                key = (groups >= 2 * cus, width if groups >= 2 * cus else -width, -threads)
                if best is None or key > best[0]:
                    best = (key, GroupNorm2dConfig(threads, units, width, 0))
                break
    if best is not None:
        return best[1]
    return GroupNorm2dConfig(512, min(8, most), params.c, 1)


def _get_configs(params: GroupNorm2dParams, device_attr=None) -> List[GroupNorm2dConfig]:
    cus = getattr(device_attr, "multiprocessor_count", 256) or 256
    return [_choose(params, cus, 6 if params.dtype == 2 else 12, False)]


def _get_bwd_configs(params: GroupNorm2dParams, device_attr=None) -> List[GroupNorm2dConfig]:
    cus = getattr(device_attr, "multiprocessor_count", 256) or 256
    return [_choose(params, cus, 3 if params.dtype == 2 else 6, True)]


def _defines(params: GroupNorm2dParams, config: GroupNorm2dConfig):
    params.validate()
    assert is_legal(params, config), f"illegal configuration {config} of {params}"
    return {
        "SPIO_GN_C": params.c, "SPIO_GN_GROUPS": params.groups, "SPIO_GN_SLICE": config.slice,
        "SPIO_GN_THREADS": config.threads, "SPIO_GN_UNITS": config.units, "SPIO_GN_SPLIT": config.split,
        "SPIO_GN_EPS": f"{float(params.eps)!r}f", "SPIO_GN_HAS_WEIGHT": int(params.has_weight),
        "SPIO_GN_HAS_BIAS": int(params.has_bias), "SPIO_GN_KEPT": int(params.kept),
        "SPIO_DTYPE": params.dtype, "SPIO_ACT": params.activation,
    }  # fmt: skip


def _grid(params: GroupNorm2dParams, config: GroupNorm2dConfig):
    """(workgroups, stretches of an image)"""
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


def kept_shapes(n, c, h, w):
    """Shapes of the codes and exponents of an input that is kept in 8 bits (channels innermost)."""
    return (n, h, w, c), (n, h, w, divup(c, 32))


def _make_test_args(params: GroupNorm2dParams, device):
    codes, exponents = (torch.empty(s, device=device, dtype=torch.uint8) if params.kept else None
                        for s in kept_shapes(*params.shape))  # fmt: skip
    x = _images(params, device)
    stats = torch.empty((params.n, params.groups, 2), device=device)
    return (torch.empty_like(x), codes, exponents, stats, x, *_vectors(params, device), params.pixels, params.n)


def _make_bwd_test_args(params: GroupNorm2dParams, device):
    dy = _images(params, device)
    if params.kept:
        codes, exponents = kept_shapes(*params.shape)
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
    is_legal=is_legal,
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
    is_legal=is_legal,
)
