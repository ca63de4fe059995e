"""group_norm_2d where float32 arithmetic comes to its ends: constant groups, means far above the deviation, rows of
sums of very many images, the smallest eps."""

import pytest
import torch

from spio_amd import native
from spio_amd.functional import group_norm_2d
from spio_amd.hip import get_device_attributes
from spio_amd.kernels.group_norm_2d_kernel import GroupNorm2dParams, _get_bwd_configs, _get_configs, DTYPES
from spio_amd.layers import GroupNorm2d
from tests.pointwise_reference import CL, assert_within, group_norm, rounding

pytestmark = pytest.mark.gpu
HALF, BF16, FLOAT = torch.float16, torch.bfloat16, torch.float32
# (shape, groups, whether the image is cut into stretches); no group has a power of two of values
SHAPES = [((2, 16, 7, 7), 2, 0), ((1, 72, 9, 5), 8, 0), ((1, 64, 57, 55), 32, 1), ((2, 48, 75, 61), 8, 1)]


def _is_split(shape, groups, dtype, configs=_get_configs, **more):
    (config,) = configs(GroupNorm2dParams(*shape, groups, DTYPES[dtype], **more), get_device_attributes(0))
    return config.split


@pytest.mark.parametrize("value,dtype", [(3.0, HALF), (1000.0, HALF), (0.203125, BF16), (1.0e5, FLOAT), (2.0**65, BF16),
                                         (-1.625 * 2.0**70, BF16), (1.25 * 2.0**66, FLOAT)])  # fmt: skip
@pytest.mark.parametrize("shape,groups,split", SHAPES)
def test_a_constant_group_is_its_bias(shape, groups, split, value, dtype):
    """The values have at most ten bits and a stretch less than 2^14 of them: every sum is exact in 24 bits, the mean is
    the value, and no difference is left, whatever the size of the value."""
    assert _is_split(shape, groups, dtype, has_weight=False) == split
    c = shape[1]
    x = torch.full(shape, value, dtype=dtype, device="cuda").contiguous(memory_format=CL)
    bias = torch.arange(c, dtype=torch.float32) / 8
    y = group_norm_2d(x, groups, None, bias.cuda()).cpu().float()
    assert torch.equal(y, bias[:, None, None].expand(shape))


@pytest.mark.parametrize("shape,groups,split", SHAPES)
def test_a_mean_whose_square_overflows(shape, groups, split):
    """Values around 1.2 * 2^64, 2^-9 of that apart: the squares of the differences stay finite, that of the mean does not.
    A mean is off by 2^-19 of itself at most (chains of 128 values, then trees), which is 2^-10 of a deviation."""
    assert _is_split(shape, groups, FLOAT, has_weight=False, has_bias=False) == split
    g = torch.Generator().manual_seed(0)
    x = (1.2 * 2.0**64 * (1 + 2.0**-9 * torch.randn(shape, generator=g, dtype=torch.float64))).float()
    (exact,) = group_norm(x, groups, None, None, 1e-5, "none")
    y = group_norm_2d(x.cuda().contiguous(memory_format=CL), groups)
    assert_within(y, exact, 2.0**-10 + 2.0**-16 * exact.abs().max() + rounding(exact, FLOAT))


@pytest.mark.parametrize("shape,split", [((65536, 8, 1, 1), 1), ((33000, 16, 2, 1), 1), ((16384, 64, 8, 8), 0)])
def test_sums_over_very_many_images(shape, split):
    """Rows of sums are added in trees and in 64 bits: grad_bias is within 2^-19 of the sum of the terms' magnitudes (the
    workgroups' own chains and trees 2^-20), also where all terms are equal and roundings of a long chain all go one
    way.  One image's share is 2^-16 or more."""
    n, c, h, w = shape
    assert _is_split(shape, 2, FLOAT, _get_bwd_configs, has_weight=False) == split
    bias = torch.zeros(c, device="cuda", requires_grad=True)
    x = torch.randn(n, h, w, c, device="cuda", dtype=FLOAT).permute(0, 3, 1, 2)
    y = group_norm_2d(x, 2, None, bias)
    same = torch.full((n, h, w, c), 0.1, device="cuda", dtype=FLOAT).permute(0, 3, 1, 2)
    g = torch.Generator("cuda").manual_seed(1)
    mixed = torch.empty(n, h, w, c, device="cuda", dtype=FLOAT).normal_(generator=g).permute(0, 3, 1, 2)
    for dy in (same, mixed):
        (db,) = torch.autograd.grad(y, bias, dy, retain_graph=True)
        terms = dy.permute(0, 2, 3, 1).reshape(-1, c).double()
        assert_within(db, terms.sum(0).cpu(), 2.0**-19 * terms.abs().sum(0).cpu())


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("eps", [1e-37, 1e-40, 1e-60, 1e-300, 1e40])
def test_eps_beyond_the_normal_numbers(eps, python):
    """One that float32 has no normal number for counts as the nearest that it has one for: a constant group still is its
    bias, and a group with a deviation what it is without eps (or, with the largest, its bias)."""
    held = native.Bypass() if python else None
    bias = torch.arange(16.0) / 8
    for hw in ((8, 8), (64, 64)):
        x = torch.full((1, 16, *hw), 3.0)
        y = group_norm_2d(x.cuda().contiguous(memory_format=CL), 2, None, bias.cuda(), eps).cpu()
        assert torch.equal(y, bias[:, None, None].expand(y.shape))
        x = torch.randn(1, 16, *hw, generator=torch.Generator().manual_seed(2))
        (exact,) = group_norm(x, 2, None, bias, eps, "none")
        y = group_norm_2d(x.cuda().contiguous(memory_format=CL), 2, None, bias.cuda(), eps)
        assert_within(y, exact, 2.0**-16 * exact.abs().max())
    if held:
        held.release()


@pytest.mark.parametrize("shape", [(128, 9, 5, 4), (200, 9, 5, 4), (129, 15, 7), (1000, 12), (300, 20, 1, 1)])
@pytest.mark.parametrize("dtype", [HALF, FLOAT, torch.float64])
def test_the_layer_on_more_images_than_torch_sums_right(shape, dtype):
    """Tensors that the kernels do not take, against the same layer in 64 bits on the CPU.  Of the largest value: four steps of the
    type for the roundings of norm, activation, their gradients and the result, and 2^-12 for float32 arithmetic on groups of
    as few as three values, whose deviation may be a hundredth of them."""
    g = torch.Generator().manual_seed(3)
    n, c = shape[:2]
    layer = GroupNorm2d(c // 3 if c % 3 == 0 else 4, c, activation="silu")
    with torch.no_grad():
        for p in layer.parameters():
            p.copy_((torch.rand(c, generator=g) + 0.5).to(dtype))
    x, dy = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    exact = GroupNorm2d(layer.num_groups, c, activation="silu").double()
    exact.load_state_dict(layer.state_dict())
    xe, xg = x.double().requires_grad_(), x.cuda().requires_grad_()
    expected = [exact(xe), *torch.autograd.grad(exact(xe), [xe, *exact.parameters()], dy.double())]
    layer = layer.to(dtype).cuda()
    y = layer(xg)
    got = [y, *torch.autograd.grad(y, [xg, *layer.parameters()], dy.cuda())]
    for a, e, name in zip(got, expected, ("y", "dx", "dw", "db")):
        assert a.dtype == dtype and a.shape == e.shape
        assert_within(a.detach(), e.detach(), (2.0**-12 + 4 * torch.finfo(dtype).eps) * e.detach().abs().max(), name)
    with torch.autocast("cuda", dtype=HALF):
        y = layer(xg)
    assert y.dtype == (FLOAT if dtype == HALF else dtype)
