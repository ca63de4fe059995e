"""The compiled kernels of the group norm and of the 8-bit form hold no 64-bit shift by a vector register, which the
hardware gets wrong where that register is a wave's last one: images held whole and in stretches, both directions, and the
four element-wise kernels.  CPU only."""

import os
import re
import subprocess

import pytest

from spio_amd.build import CSRC_DIR, HIPCC_DEVICE_FLAGS, ROCM_HOME
from spio_amd.hip import DeviceAttributes
from spio_amd.kernels import (
    Activation8bitConfig,
    Activation8bitParams,
    GroupNorm2dParams,
    activation_8bit_bwd_kernel_factory,
    activation_8bit_kernel_factory,
    group_norm_2d_bwd_kernel_factory,
    group_norm_2d_kernel_factory,
    pack_8bit_kernel_factory,
    unpack_8bit_kernel_factory,
)

WIDE_SHIFT = re.compile(r"v_(?:lshl|lshr|ashr)rev_[bi]64\S* v\[\d+:\d+\], v\d+")
NORMS = [
    GroupNorm2dParams(128, 768, 7, 7, 32),  # whole
    GroupNorm2dParams(32, 192, 28, 28, 24, 2, 2),  # whole, in slices
    GroupNorm2dParams(64, 64, 14, 13, 8, 1, 1, kept=True),
    GroupNorm2dParams(16, 24, 144, 144, 4, 1, 3, kept=True),  # stretches
    GroupNorm2dParams(1, 8, 200, 200, 8, 2, 1, kept=True),
]
CASES = [(factory, params) for params in NORMS for factory in (group_norm_2d_kernel_factory, group_norm_2d_bwd_kernel_factory)]
CASES += [(factory, Activation8bitParams(dtype, activation))
          for factory, activation in ((activation_8bit_kernel_factory, 1), (activation_8bit_bwd_kernel_factory, 1),
                                      (activation_8bit_kernel_factory, 3), (activation_8bit_bwd_kernel_factory, 3),
                                      (pack_8bit_kernel_factory, 0), (unpack_8bit_kernel_factory, 0))
          for dtype in (0, 2)]  # fmt: skip


@pytest.mark.parametrize("factory,params", CASES, ids=lambda v: v.encode() if hasattr(v, "encode") else "")
def test_no_shift_of_64_bits_by_a_vector_register(factory, params, tmp_path):
    attr = DeviceAttributes()
    config = Activation8bitConfig() if isinstance(params, Activation8bitParams) else factory.configs(params, attr)[0]
    kernel = factory.make_kernel(params, config, attr)
    out = str(tmp_path / "kernel.s")
    subprocess.run([os.path.join(ROCM_HOME, "bin", "hipcc"), "-S", "--cuda-device-only", *HIPCC_DEVICE_FLAGS, f"-I{CSRC_DIR}",
                    *[f"-D{k}={v}" for k, v in kernel.defines.items()], "-o", out,
                    os.path.join(CSRC_DIR, kernel.kernel_source_file)], check=True, capture_output=True)  # fmt: skip
    code = open(out).read()
    assert "buffer_" in code and not WIDE_SHIFT.findall(code)
