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


# images that the backward pass holds whole (all channels and slices of 32) and in stretches, a last block of 24 and of 8 channels
NORM_CASES = [
    ((3, 24, 9, 7), 4, HALF, "wb", 0), ((2, 64, 14, 13), 8, BF16, "wb", 1), ((24, 320, 13, 11), 10, FLOAT, "w", 0),
    ((1, 72, 60, 57), 9, HALF, "wb", 1), ((2, 96, 56, 56), 32, BF16, "", 1), ((1, 40, 75, 61), 10, FLOAT, "b", 1),
]  # fmt: skip


@pytest.mark.parametrize("shape,groups,dtype,affine,split", NORM_CASES)
def test_norm_with_relu_and_a_checkpoint(shape, groups, dtype, affine, split, path):
    """Tolerances as in the tests of the norm: 2^-16 of a tensor's largest value, 2^-17 of a sum's terms."""
    x, dy, weight, bias = _norm_tensors(shape, dtype, affine)
    params = GroupNorm2dParams(*shape, groups, NUMBERS[dtype], 1, 1e-5, weight is not None, bias is not None, True)
    assert _get_bwd_configs(params, get_device_attributes(0))[0].split == split
    z, *_ = _norm_exact(x, dy, groups, weight, bias)
    dy = torch.where(z.abs() < 2.0**-12 * z.abs().max(), 0, dy)  # where the arithmetic decides the sign
    z, exact, w_terms, b_terms = _norm_exact(x, dy, groups, weight, bias)
    rounded = values(*pack_rows(x.permute(0, 2, 3, 1))).permute(0, 3, 1, 2)
    assert ((rounded > 0) != (x > 0)).any()
    leaves = [None if t is None else t.cuda().requires_grad_() for t in (x.cuda().contiguous(memory_format=CL), weight, bias)]
    y = group_norm_2d(leaves[0], groups, leaves[1], leaves[2], 1e-5, "relu", True)
    wanted = z.clamp_min(0)
    assert_within(y.detach(), wanted, 2.0**-16 * wanted.max() + rounding(wanted, dtype), "y")
    dx, *rest = torch.autograd.grad(y, [t for t in leaves if t is not None], dy.cuda())
    assert_within(dx, exact[0], 2.0**-16 * exact[0].abs().max() + rounding(exact[0], dtype), "dx")
    sums = [(exact[1], w_terms), (exact[2], b_terms)]
    for got, (e, terms) in zip(rest, [s for s, v in zip(sums, (weight, bias)) if v is not None]):
        assert_within(got, e, 2.0**-17 * terms + 2.0**-40, "sums")


def test_the_norms_operator():
    """A pixel's row of exponents ends with a byte for every eight channels."""
    x, dy, weight, bias = _norm_tensors((2, 72, 5, 6), HALF, "wb")
    xg, wg, bg = (t.cuda().requires_grad_() for t in (x.cuda().contiguous(memory_format=CL), weight, bias))
    y, _, codes, exponents = group_norm_2d_forward(xg, 9, wg, bg, 1e-5, "relu", True)
    assert codes.shape == (2, 5, 6, 72) and exponents.shape == (2, 5, 6, 3 + 9)
    expected_codes, expected_exponents = pack_rows(x.permute(0, 2, 3, 1))
    assert torch.equal(codes.cpu(), expected_codes) and torch.equal(exponents[..., :3].cpu(), expected_exponents)
    bits = (exponents[..., 3:, None].to(torch.int32) >> torch.arange(8, device="cuda") & 1).flatten(-2).bool()
    assert torch.equal(bits, (y > 0).permute(0, 2, 3, 1))
    torch.library.opcheck(group_norm_2d_forward, (xg, 9, wg, bg, 1e-5, "relu", True))
    compiled = torch.compile(lambda x, w, b: group_norm_2d(x, 9, w, b, 1e-5, "relu", True), backend="aot_eager")
    got = torch.autograd.grad(compiled(xg, wg, bg), [xg, wg, bg], dy.cuda())
    expected = torch.autograd.grad(group_norm_2d(xg, 9, wg, bg, 1e-5, "relu", True), [xg, wg, bg], dy.cuda())
    assert all(torch.equal(a, b) for a, b in zip(got, expected))


def test_replays_of_a_captured_pass():
    x = _with_outliers(3 * 24 * 9 * 7, HALF).reshape(3, 24, 9, 7).cuda().contiguous(memory_format=CL).requires_grad_()
    dy = torch.randn_like(x)

    def step():
        y = activation_8bit(group_norm_2d(x, 3, activation="relu", checkpoint_8bit=True) - 0.5, "relu")
        return [y.detach(), torch.autograd.grad(y, x, dy)[0]]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for seed in range(3):
        torch.manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn(3, 24, 9, 7, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))
