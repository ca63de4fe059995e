"""relu between tensors that are kept in 8 bits: its gradient is that of the input as it was.

The derivative jumps at zero, so half a step of the 8-bit form is a whole gradient: activation_8bit keeps a bit a value for
it, group_norm_2d one beside the codes.  The expected gradients go by the inputs themselves.
"""

import pytest
import torch

from spio_amd import native
from spio_amd.functional import activation_8bit, group_norm_2d
from spio_amd.functional.activation_8bit_function import activation_8bit_forward
from spio_amd.functional.group_norm_2d_function import group_norm_2d_forward
from spio_amd.hip import get_device_attributes
from spio_amd.kernels.group_norm_2d_kernel import DTYPES as NUMBERS
from spio_amd.kernels.group_norm_2d_kernel import GroupNorm2dParams, _get_bwd_configs
from spio_amd.layers import Activation8bit
from tests.pointwise_reference import CL, assert_within, group_norm, pack_rows, rounding, values

pytestmark = pytest.mark.gpu
HALF, BF16, FLOAT = torch.float16, torch.bfloat16, torch.float32
DTYPES = [HALF, BF16, FLOAT]


def _with_outliers(n, dtype, seed=0):
    """Every block has one value 100 times the others: most of these are less than half a step."""
    g = torch.Generator().manual_seed(seed + n)
    x = torch.randn(n, generator=g)
    x[::32] *= 100
    return x.to(dtype)


@pytest.fixture(params=["native", "python"])
def path(request):
    held = native.Bypass() if request.param == "python" else None
    yield request.param
    if held:
        held.release()


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_small_values(dtype, path):
    for n in (1, 7, 8, 9, 31, 33, 4095, 4096, 4097, 100_003):
        x, dy = _with_outliers(n, dtype), torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dtype)
        assert n < 4000 or ((x > 0) & (values(*pack_rows(x)) == 0)).any()
        xg = x.cuda().requires_grad_()
        y = activation_8bit(xg, "relu")
        (dx,) = torch.autograd.grad(y, xg, dy.cuda())
        assert torch.equal(y.cpu(), torch.relu(x))
        assert torch.equal(dx.cpu(), torch.where(x > 0, dy, torch.zeros_like(dy)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_beside_infinities_and_nan(dtype, path):
    """A value's gradient depends on nothing but the value; NaN passes it on, as torch's relu has it."""
    x = _with_outliers(32 * 5 + 3, dtype)
    x[5], x[40], x[41], x[70], x[162] = float("inf"), float("-inf"), 0.0, float("nan"), float("inf")
    dy = torch.arange(1.0, x.numel() + 1).to(dtype)
    for function in (lambda t: activation_8bit(t, "relu"), Activation8bit("relu"), torch.relu):
        xg = x.cuda().requires_grad_()
        (dx,) = torch.autograd.grad(function(xg), xg, dy.cuda())
        assert torch.equal(dx.cpu(), torch.where(x <= 0, torch.zeros_like(dy), dy))


def test_layouts_and_empty_tensors(path):
    x = _with_outliers(2 * 24 * 5 * 7, HALF).reshape(2, 24, 5, 7).cuda()
    for t in (x.contiguous(memory_format=CL), x.transpose(1, 3), x[:, :, ::2], x[:1].expand(3, 24, 5, 7), x.reshape(-1)[1:], x[:0]):
        t = t.detach().requires_grad_()
        dy = torch.randn(t.shape, device="cuda", dtype=HALF)
        (dx,) = torch.autograd.grad(activation_8bit(t, "relu"), t, dy)
        assert torch.equal(dx, torch.where(t > 0, dy, 0))


def test_what_is_kept_and_the_operator():
    """A bit a value."""
    x = _with_outliers(1003, HALF).cuda().requires_grad_()
    y, bits, exponents = activation_8bit_forward(x, "relu", True)
    assert bits.shape == (126,) and exponents.shape == (0,)
    shifts = torch.arange(8, device="cuda")
    seen = (bits.to(torch.int32)[:, None] >> shifts & 1).reshape(-1)
    assert torch.equal(seen[:1003].bool(), x > 0) and not seen[1003:].any()
    torch.library.opcheck(activation_8bit_forward, (x, "relu", True))
    compiled = torch.compile(lambda t: activation_8bit(t, "relu"), backend="aot_eager")
    (dx,) = torch.autograd.grad(compiled(x), x, torch.ones_like(x))
    assert torch.equal(dx, (x > 0).to(HALF))


def _norm_tensors(shape, dtype, affine):
    g = torch.Generator().manual_seed(sum(shape))
    n, c, h, w = shape
    x = torch.randn(shape, generator=g)
    x[:, ::8] *= 30  # blocks have values far larger than most
    x, dy = x.to(dtype), torch.randn(shape, generator=g).to(dtype)
    weight = torch.rand(c, generator=g) + 0.5 if "w" in affine else None
    bias = torch.rand(c, generator=g) - 0.5 if "b" in affine else None
    return x, dy, weight, bias


def _norm_exact(x, dy, groups, weight, bias):
    """Gradients of the norm of the kept values with relu's mask of the values as they were: dz is dy where z of the
    input is positive, and the rest is the norm without activation of the kept values.  With the sums of the terms."""
    (z,) = group_norm(x, groups, weight, bias, 1e-5, "none")
    dz = torch.where(z > 0, dy.double(), 0.0)
    out, _, w_terms, b_terms = group_norm(x, groups, weight, bias, 1e-5, "none", dz, True)
    return z, out[1:], w_terms, b_terms


# whole images and stretches, a last block of 24 and of 8 channels, units that make no whole block
NORM_CASES = [
    ((3, 24, 9, 7), 4, HALF, "wb", 0), ((2, 64, 14, 13), 8, BF16, "wb", 0), ((2, 320, 13, 11), 32, FLOAT, "w", 0),
    ((1, 72, 60, 57), 9, HALF, "wb", 1), ((2, 96, 56, 56), 32, BF16, "", 1), ((1, 40, 75, 61), 10, FLOAT, "b", 1),
]  # fmt: skip
