"""Element-wise kernels with an 8-bit checkpoint (csrc/activation_8bit.hip): parameters and factories.

Specialised by type and activation; the number of values is an argument, and the grid follows from it.  Arguments:
  activation_8bit      (output, codes or None, exponents or None, input, n)
  activation_8bit_bwd  (grad_input, codes, exponents, grad_output, n)
  pack_8bit            (codes, exponents, input, n)
  unpack_8bit          (output, codes, exponents, n)
"""

from dataclasses import dataclass

import torch

from .group_norm_2d_kernel import ACTIVATIONS, DTYPE_NAMES, DTYPES
from .kernel import KernelSpec
from .kernel_factory import KernelFactory
from .launch_params import LaunchParams

SOURCE = "activation_8bit.hip"
BLOCK = 32  # values of a block of the 8-bit form


@dataclass(frozen=True)
class Activation8bitParams:
    """Type and activation (numbers of DTYPES and ACTIVATIONS), and whether the forward pass keeps its input."""

    dtype: int = 0
    activation: int = 0
    kept: bool = True

    def encode(self) -> str:
        return f"{DTYPE_NAMES[self.dtype]}_{list(ACTIVATIONS)[self.activation]}" + ("_8bit" if self.kept else "")

    def validate(self):
        assert 0 <= self.dtype <= 2 and 0 <= self.activation <= 3


@dataclass(frozen=True)
class Activation8bitConfig:
    """Threads of a workgroup and units of eight values that a lane has in flight.

    Two units everywhere: with four, gelu of float16 tensors takes as long at 2 million values (9.4 us) and up to a
    tenth longer above (us forward / backward, two units and four: 19 million values 19.5 / 19.0 and 21.7 / 20.3, 77 million
    65.5 / 63.6 and 70.1 / 67.0, 154 million 129.7 / 130.9 and 131.4 / 133.6); one unit, 512 and 1024 threads are in between.
    """

    threads: int = 256
    units: int = 2


def _spec(mode):
    def spec(params: Activation8bitParams, config: Activation8bitConfig, _device_attr=None) -> KernelSpec:
        params.validate()
        defines = {
            "SPIO_MODE": mode, "SPIO_THREADS": config.threads, "SPIO_UNROLL": config.units,
            "SPIO_DTYPE": params.dtype, "SPIO_ACT": params.activation, "SPIO_KEEP": int(params.kept),
        }  # fmt: skip
        return KernelSpec(defines, LaunchParams(grid=1, block=config.threads), SOURCE,
                          values_per_workgroup=config.threads * config.units * 8)  # fmt: skip

    return spec


def _test_args(mode):
    def args(params: Activation8bitParams, device):
        n = 1 << 24
        values = torch.randn(n, device=device).to(list(DTYPES)[params.dtype])
        codes = torch.randint(0, 256, (n,), device=device, dtype=torch.uint8)
        exponents = torch.full((n // BLOCK,), 126, device=device, dtype=torch.uint8)
        kept = (codes, exponents) if params.kept else (None, None)
        return {
            0: (torch.empty_like(values), *kept, values, n),
            1: (torch.empty_like(values), codes, exponents, values, n),
            2: (codes, exponents, values, n),
            3: (values, codes, exponents, n),
        }[mode]

    return args


def _factory(name, mode):
    return KernelFactory(
        Activation8bitParams,
        Activation8bitConfig,
        None,
        kernel_name=name,
        configs=lambda params, device_attr=None: [Activation8bitConfig()],
        kernel_spec=_spec(mode),
        make_test_args=_test_args(mode),
        args_checker=None,
    )


activation_8bit_kernel_factory = _factory("spio_activation_8bit", 0)
activation_8bit_bwd_kernel_factory = _factory("spio_activation_8bit_bwd", 1)
pack_8bit_kernel_factory = _factory("spio_pack_8bit", 2)
unpack_8bit_kernel_factory = _factory("spio_unpack_8bit", 3)
