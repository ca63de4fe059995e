"""group_norm_2d and its backward against the formula in 64 bits on the CPU.

Tolerances.  The kernels compute in float32 (units of 2^-24): a mean is a sum of chains of at most 16 * 8 values, then
a tree, off by at most 2^-19 of the mean magnitude, which here is at most four deviations: 2^-17 of xhat.  A handful of
further roundings, the activations (2^-22 of their argument) and the sums of the backward pass stay below as much
again, so results are within 2^-16 of the largest magnitude of theirs, plus half a step of the type they are rounded to.  Sums
over images and pixels: 2^-17 of the sum of the magnitudes of their terms.
"""

import pytest
import torch

from spio_amd.functional import group_norm_2d
from spio_amd.functional.group_norm_2d_function import group_norm_2d_backward, group_norm_2d_forward
from spio_amd.hip import get_device_attributes
from spio_amd.kernels.group_norm_2d_kernel import (
    GroupNorm2dConfig,
    GroupNorm2dParams,
    group_norm_2d_bwd_kernel_factory,
    group_norm_2d_kernel_factory,
    is_legal,
    kept_shapes,
)
from spio_amd.layers import GroupNorm2d
from tests.pointwise_reference import CL, assert_within, group_norm, rounding, pack_rows

pytestmark = pytest.mark.gpu
HALF, BF16, FLOAT = torch.float16, torch.bfloat16, torch.float32


def _tensors(n, c, h, w, dtype, affine="wb", seed=0):
    g = torch.Generator().manual_seed(seed + n + c + h + w)
    scale, shift = torch.rand(c, 1, 1, generator=g) * 1.5 + 0.5, torch.rand(c, 1, 1, generator=g) * 2 - 1
    x = (torch.randn(n, c, h, w, generator=g) * scale + shift).to(dtype)
    dy = torch.randn(n, c, h, w, generator=g).to(dtype)
    weight = torch.rand(c, generator=g) + 0.5 if "w" in affine else None
    bias = torch.rand(c, generator=g) - 0.5 if "b" in affine else None
    return x, dy, weight, bias


def _on_gpu(t, grad=True):
    if t is None:
        return None
    t = t.cuda().contiguous(memory_format=CL) if t.dim() == 4 else t.cuda()
    return t.requires_grad_(grad)


def _check(got, x, dy, groups, weight, bias, act, kept, dtype, what=""):
    """got: y, grad_input and the vectors' gradients that there are."""
    exact, z, w_terms, b_terms = group_norm(x, groups, weight, bias, 1e-5, act, dy, kept)
    if act == "relu":  # the gradient jumps at zero: nothing comes in where that is closer than the arithmetic is exact
        assert not dy[z.abs() < 2.0**-16 * z.abs().max()].any()
    names = ["y", "dx"] + [name for name, v in (("dw", weight), ("db", bias)) if v is not None]
    for g, name in zip(got, names):
        e = exact[["y", "dx", "dw", "db"].index(name)]
        if name in ("y", "dx"):
            assert g.dtype == dtype and g.is_contiguous(memory_format=CL)
            assert_within(g, e, 2.0**-16 * e.abs().max() + rounding(e, dtype), f"{what} {name}")
        else:
            assert_within(g, e, 2.0**-17 * (w_terms if name == "dw" else b_terms) + 2.0**-40, f"{what} {name}")
    assert len(got) == len(names)


# (n, c, h, w), groups, type, activation, kept, affine.  Group widths 1, 2, 3, 4, 6, 8, 10, 24 and all channels; images of one
# pixel, whole in one workgroup and in stretches; a last slice with fewer channels; lanes without channels.
CASES = [
    ((2, 96, 56, 56), 32, HALF, "silu", True, "wb"),
    ((3, 72, 49, 33), 9, BF16, "gelu", False, "wb"),
    ((4, 768, 7, 7), 32, HALF, "none", False, "wb"),
    ((2, 192, 28, 28), 24, FLOAT, "silu", False, "wb"),
    ((2, 24, 90, 71), 4, BF16, "gelu", True, "w"),
    ((1, 64, 57, 55), 32, HALF, "relu", False, "b"),
    ((3, 40, 5, 9), 40, FLOAT, "gelu", True, "wb"),
    ((2, 320, 13, 11), 32, HALF, "silu", True, ""),
    ((2, 72, 1, 1), 3, FLOAT, "none", False, "wb"),
    ((2, 128, 30, 17), 1, BF16, "silu", True, "wb"),
    ((1, 4096, 3, 2), 16, HALF, "gelu", False, "wb"),
    ((5, 8, 3, 1), 2, FLOAT, "relu", True, "wb"),
    ((1, 48, 130, 101), 8, FLOAT, "silu", True, ""),
]


@pytest.mark.parametrize("shape,groups,dtype,act,kept,affine", CASES)
def test_forward_and_gradients(shape, groups, dtype, act, kept, affine):
    x, dy, weight, bias = _tensors(*shape, dtype, affine)
    if act == "relu":
        _, z, *_ = group_norm(x, groups, weight, bias, 1e-5, act, dy, kept)
        dy = torch.where(z.abs() < 2.0**-12 * z.abs().max(), 0, dy)
    leaves = [_on_gpu(x), _on_gpu(weight), _on_gpu(bias)]
    y = group_norm_2d(leaves[0], groups, leaves[1], leaves[2], 1e-5, act, kept)
    got = [y.detach(), *torch.autograd.grad(y, [t for t in leaves if t is not None], _on_gpu(dy, False))]
    _check(got, x, dy, groups, weight, bias, act, kept, dtype)
    with torch.no_grad():  # without a checkpoint (whose blocks may divide the sums otherwise)
        plain = group_norm_2d(leaves[0], groups, leaves[1], leaves[2], 1e-5, act, kept)
        exact = group_norm(x, groups, weight, bias, 1e-5, act)[0]
        assert_within(plain, exact, 2.0**-16 * exact.abs().max() + rounding(exact, dtype))
        assert kept or torch.equal(plain, y)
    y2 = group_norm_2d(leaves[0], groups, leaves[1], leaves[2], 1e-5, act, kept)
    again = [y2.detach(), *torch.autograd.grad(y2, [t for t in leaves if t is not None], _on_gpu(dy, False))]
    assert all(torch.equal(a, b) for a, b in zip(got, again))  # sums in the same order always


@pytest.mark.parametrize("units,kept", [(1, True), (2, True), (2, False), (3, True), (4, True)])
def test_more_stretches_than_lanes_of_a_group(units, kept):
    """Each lane joins several stretches' statistics, the last of which there are not everywhere."""
    x, dy, weight, bias = _tensors(5, 768, 14, 20, FLOAT, "w")
    params = GroupNorm2dParams(5, 768, 14, 20, 32, 2, 2, has_bias=False, kept=kept)
    xg, wg, dyg = _on_gpu(x, False), _on_gpu(weight, False), _on_gpu(dy, False)
    y, dx, stats, sums = torch.empty_like(xg), torch.empty_like(xg), torch.empty(5, 32, 2).cuda(), torch.empty(2, 768).cuda()
    codes, exponents = (torch.empty(s, dtype=torch.uint8, device="cuda") if kept else None for s in kept_shapes(5, 768, 14, 20))
    attr = get_device_attributes(0)
    for threads in (256, 512):
        kernels = [f.make_kernel(params, GroupNorm2dConfig(threads, units, 768, 1), attr)
                   for f in (group_norm_2d_kernel_factory, group_norm_2d_bwd_kernel_factory)]  # fmt: skip
        for kernel in kernels:
            kernel.compile()
            kernel.load(0)
        for _ in range(3):
            y.fill_(-42)
            kernels[0](y, codes, exponents, stats, xg, wg, None, params.pixels, 5)
            kernels[1](sums, dx, codes if kept else xg, exponents, dyg, stats, wg, None, params.pixels, 5)
            _check([y, dx, sums[0]], x, dy, 32, weight, None, "silu", kept, FLOAT, f"{threads} {units}")
        for kernel in kernels:
            kernel.unload()


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("shape,groups", [((2, 160, 19, 11), 16), ((3, 40, 17, 9), 10)])
def test_every_kind_of_configuration(shape, groups, kept):
    """Whole images and stretches, slices and all channels, each number of threads: through the kernels themselves, with
    outputs and workspaces that hold other values before."""
    n, c, h, w = shape
    x, dy, weight, bias = _tensors(*shape, HALF)
    xg, dyg, wg, bg = (_on_gpu(t, False) for t in (x, dy, weight, bias))
    params = GroupNorm2dParams(n, c, h, w, groups, activation=2, kept=kept)
    codes, exponents = pack_rows(x.permute(0, 2, 3, 1))
    tried = 0
    for threads in (256, 512, 1024):
        for units in (1, 3, 8, 11):
            for width in sorted({32, 64, 160, c}):
                for split in (0, 1):
                    config = GroupNorm2dConfig(threads, units, width, split)
                    if not is_legal(params, config) or (threads, units) not in ((256, 1), (256, 8), (512, 3), (512, 11), (1024, 3)):
                        continue
                    tried += 1
                    forward = group_norm_2d_kernel_factory.make_kernel(params, config)
                    backward = group_norm_2d_bwd_kernel_factory.make_kernel(params, config)
                    for kernel in (forward, backward):
                        kernel.compile()
                        kernel.load(0)
                    y, dx = torch.full_like(xg, -42.0), torch.full_like(xg, -42.0)
                    stats = torch.full((n, groups, 2), float("nan"), device="cuda")
                    sums = torch.full((2, c), float("nan"), device="cuda")
                    kc = torch.full((n, h, w, c), 77, dtype=torch.int8, device="cuda") if kept else None
                    ke = torch.full((n, h, w, -(-c // 32)), 7, dtype=torch.uint8, device="cuda") if kept else None
                    forward(y, kc, ke, stats, xg, wg, bg, params.pixels, n)
                    if kept:
                        assert torch.equal(kc.cpu(), codes) and torch.equal(ke.cpu(), exponents), config
                    backward(sums, dx, kc if kept else xg, ke, dyg, stats, wg, bg, params.pixels, n)
                    _check([y, dx, sums[0], sums[1]], x, dy, groups, weight, bias, "silu", kept, HALF, str(config))
                    for kernel in (forward, backward):
                        kernel.unload()
    assert tried >= 6


def _call(x, groups, weight, bias, dy, act="silu", kept=False):
    y = group_norm_2d(x, groups, weight, bias, 1e-5, act, kept)
    return [y.detach(), *torch.autograd.grad(y, [x, weight, bias], dy)]


@pytest.mark.parametrize("kept", [False, True])
def test_layouts_alignment_and_types_of_the_vectors(kept):
    """Tensors in NCHW order, with gaps, off 16 bytes, a gradient that is one number seen everywhere, and vectors in
    float16 or with gaps give what the tensors in order give."""
    shape, groups = (2, 48, 9, 10), 6
    x, dy, weight, bias = _tensors(*shape, HALF)
    weight, bias = weight.half(), bias.half()
    dy = dy[:1, :1, :1, :1].expand(shape)
    expected = _call(_on_gpu(x), groups, _on_gpu(weight), _on_gpu(bias), dy.contiguous().cuda(), kept=kept)

    def off(t):  # one value behind a 16-byte border
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:]
        return torch.as_strided(flat, t.shape, t.cuda().contiguous(memory_format=CL).stride()).copy_(t)

    ways = [
        (x.cuda(), weight.cuda(), bias.cuda()),
        (off(x), weight.cuda(), bias.cuda()),
        (torch.stack([x, x], -1).cuda()[..., 0], torch.stack([weight, weight], -1).cuda()[:, 0], bias.cuda()),
        (x.cuda().contiguous(memory_format=CL), weight.cuda(), torch.cat([bias[:1], bias]).cuda()[1:]),
    ]
    for tensors in ways:
        leaves = [t.requires_grad_() for t in tensors]
        got = _call(leaves[0], groups, leaves[1], leaves[2], dy.cuda(), kept=kept)
        assert [g.dtype for g in got] == [HALF] * 4
        assert all(torch.equal(a, b) for a, b in zip(got, expected))


@pytest.mark.parametrize("split", [False, True])
def test_infinities_and_nan_stay_in_their_group(split):
    n, c, h, w, groups = (2, 64, 60, 57, 8) if split else (2, 64, 9, 10, 8)
    x, dy, weight, bias = _tensors(n, c, h, w, HALF)
    expected = _call(_on_gpu(x), groups, _on_gpu(weight), _on_gpu(bias), _on_gpu(dy, False))
    x[0, 9, 3, 4], x[1, 63, 8, 8] = float("inf"), float("nan")
    got = _call(_on_gpu(x), groups, _on_gpu(weight), _on_gpu(bias), _on_gpu(dy, False))
    touched = torch.zeros(n, groups, dtype=torch.bool)
    touched[0, 1] = touched[1, 7] = True
    for g, e in zip(got[:2], expected[:2]):
        g, e = (t.reshape(n, groups, -1).cpu() for t in (g, e))
        assert torch.isnan(g[touched]).all() and torch.equal(g[~touched], e[~touched])
    channels = touched.any(0).repeat_interleave(8)
    for g, e in zip(got[2:], expected[2:]):
        assert torch.equal(g.cpu()[~channels], e.cpu()[~channels])


def test_a_constant_group_and_the_lowest_value():
    """No variance: rstd is 1/sqrt(eps), the output the bias; and values at the type's end do not overflow on the way."""
    x = torch.full((1, 16, 4, 4), 3.0).to(BF16)
    y = group_norm_2d(x.cuda(), 2, None, torch.arange(16.0).cuda())
    assert torch.equal(y.float().cpu(), torch.arange(16.0)[:, None, None].expand(1, 16, 4, 4))
    x = torch.full((1, 16, 4, 4), -65504.0).half()
    x[:, ::2] = 65504.0
    y = group_norm_2d(x.cuda(), 2).float().cpu()
    assert torch.equal(y, torch.where(x > 0, 1.0, -1.0))


def test_gradient_against_differences():
    """Along a random direction, in float32: the difference of the outputs 2^-6 apart has an error of that squared times
    the third derivative, which is of the order of the gradient itself here, and rounding of 2^-24 * 2^6 of the
    outputs' norm: together below 2^-9 of the product of norms."""
    x, dy, weight, bias = _tensors(2, 32, 6, 5, FLOAT)
    g = torch.Generator().manual_seed(1)
    leaves = [_on_gpu(t) for t in (x, weight, bias)]
    grads = _call(leaves[0], 4, leaves[1], leaves[2], dy.cuda(), "gelu")[1:]
    for i, t in enumerate((x, weight, bias)):
        v = torch.randn(t.shape, generator=g)
        ends = []
        for sign in (1, -1):
            moved = [x, weight, bias]
            moved[i] = t + sign * 2.0**-6 * v
            y = group_norm_2d(moved[0].cuda(), 4, moved[1].cuda(), moved[2].cuda(), activation="gelu")
            ends.append((y.cpu().double() * dy.double()).sum())
        slope = (ends[0] - ends[1]) / 2.0**-5
        product = (grads[i].cpu().double() * v.double()).sum()
        assert abs(slope - product) <= 2.0**-9 * grads[i].double().norm().cpu() * v.double().norm()


def test_images_that_pass_32_bits():
    """More than 2^31 values: the first and the last images are the same, and those of a small call, which adds in
    another order (a step of the result's type, and 2^-15 of the largest, apart at most)."""
    x, dy, weight, bias = _tensors(3, 64, 32, 32, HALF)
    n = 3 * 11000  # 2.16e9 values
    weight, bias = weight.cuda(), bias.cuda()
    xs, dys = _on_gpu(x, False), _on_gpu(dy, False)
    y, stats, codes, exponents = group_norm_2d_forward(xs, 16, weight, bias, 1e-5, "silu", True)
    dx, sums = group_norm_2d_backward(dys, codes, exponents, stats, 16, weight, bias, 1e-5, "silu")
    big = [xs.permute(0, 2, 3, 1).repeat(n // 3, 1, 1, 1).permute(0, 3, 1, 2)]
    big_y, big_stats, big_codes, big_exponents = group_norm_2d_forward(big[0], 16, weight, bias, 1e-5, "silu", True)

    def close(a, b):
        bound = torch.finfo(a.dtype).eps * b.abs().double() + 2.0**-15 * float(b.abs().max())
        return bool(((a.double() - b.double()).abs() <= bound).all())

    for whole, part in ((big_y, y), (big_stats, stats)):
        assert torch.equal(whole[:3], whole[-3:]) and close(whole[-3:], part)
    for whole, part in ((big_codes, codes), (big_exponents, exponents)):
        assert torch.equal(whole[:3], part) and torch.equal(whole[-3:], part)
    del big_y
    big[0] = dys.permute(0, 2, 3, 1).repeat(n // 3, 1, 1, 1).permute(0, 3, 1, 2)
    big_dx, big_sums = group_norm_2d_backward(big[0], big_codes, big_exponents, big_stats, 16, weight, bias, 1e-5, "silu")
    assert torch.equal(big_dx[:3], big_dx[-3:]) and close(big_dx[-3:], dx)
    # 11000 times the small sums, added in another order
    scale = sums.abs().max() * (n // 3)
    assert (big_sums - sums * (n // 3)).abs().max() <= 2.0**-14 * scale


@pytest.mark.parametrize("kept", [False, True])
def test_replays_of_a_captured_pass(kept):
    """Both passes in a HIP graph on a stream of its own, replayed on new data between eager calls; two graphs that were
    captured one after the other do not share memory that both still need."""
    shapes = [((2, 96, 14, 14), 32), ((1, 64, 60, 57), 8)]  # one launch and two
    runs = []
    for shape, groups in shapes:
        x, dy, weight, bias = _tensors(*shape, HALF)
        leaves = [_on_gpu(t) for t in (x, weight, bias)]
        dyg = _on_gpu(dy, False)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _call(leaves[0], groups, leaves[1], leaves[2], dyg, kept=kept)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = _call(leaves[0], groups, leaves[1], leaves[2], dyg, kept=kept)
        runs.append((graph, leaves, dyg, groups, out))
    for seed in range(1, 4):
        for (shape, _), (graph, leaves, dyg, groups, out) in zip(shapes, runs):
            x, dy, *_ = _tensors(*shape, HALF, seed=100 * seed)
            with torch.no_grad():
                leaves[0].copy_(x)
                dyg.copy_(dy)
            graph.replay()
        torch.cuda.synchronize()
        for graph, leaves, dyg, groups, out in runs:
            expected = _call(leaves[0], groups, leaves[1], leaves[2], dyg, kept=kept)
            assert all(torch.equal(a, b) for a, b in zip(out, expected))


def test_streams():
    """The kernels run on the current stream: behind work that is queued there."""
    x, dy, weight, bias = _tensors(4, 96, 56, 56, HALF)
    wg, bg = weight.cuda(), bias.cuda()
    expected = group_norm_2d(_on_gpu(x, False), 32, wg, bg)
    side = torch.cuda.Stream()
    a = torch.randn(4096, 4096, device="cuda")
    xg = torch.zeros_like(expected)
    source = _on_gpu(x, False)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            a = a @ a * 1e-3
        xg.copy_(source)
        y = group_norm_2d(xg, 32, wg, bg)
    side.synchronize()
    assert torch.equal(y, expected)


def test_empty_tensors():
    for shape in ((0, 32, 4, 4), (2, 32, 0, 4)):
        x = torch.empty(shape, device="cuda", dtype=HALF).requires_grad_()
        w = torch.ones(32, device="cuda", requires_grad=True)
        y = group_norm_2d(x, 4, w)
        assert y.shape == shape and y.dtype == HALF
        dx, dw = torch.autograd.grad(y, [x, w], torch.empty_like(y))
        assert dx.shape == shape and torch.equal(dw, torch.zeros_like(w))


def test_refusals_on_the_gpu():
    x = torch.zeros(2, 32, 4, 4, device="cuda", dtype=HALF)
    with pytest.raises(AssertionError):
        group_norm_2d(x, 5)
    with pytest.raises(AssertionError):
        group_norm_2d(x.double(), 4)
    with pytest.raises(AssertionError):
        group_norm_2d(x, 4, torch.ones(16, device="cuda"))
    with pytest.raises(AssertionError):
        group_norm_2d(x, 4, torch.ones(32))  # on the CPU
    with pytest.raises(AssertionError):
        group_norm_2d(torch.zeros(1, 4104, 1, 1, device="cuda"), 4)  # more channels than the kernels take
    y = group_norm_2d(x.requires_grad_(), 4)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivatives
        torch.autograd.grad(dx.sum(), x)
    leaf = torch.zeros(2, 32, 4, 4, device="cuda", dtype=HALF)
    moved = leaf.clone().requires_grad_()
    y = group_norm_2d(moved * 1, 4)
    twice = moved * 1
    y = group_norm_2d(twice, 4)
    twice.add_(1)  # what the backward pass needs has changed
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_opcheck_and_compile():
    x, dy, weight, bias = _tensors(2, 48, 5, 6, HALF)
    xg, wg, bg = (_on_gpu(t) for t in (x, weight, bias))
    for kept in (False, True):
        torch.library.opcheck(group_norm_2d_forward, (xg, 6, wg, bg, 1e-5, "silu", kept))
        compiled = torch.compile(lambda x, w, b: group_norm_2d(x, 6, w, b, 1e-5, "silu", kept), backend="aot_eager")  # pylint: disable=cell-var-from-loop
        got = torch.autograd.grad(compiled(xg, wg, bg), [xg, wg, bg], _on_gpu(dy, False))
        expected = _call(xg, 6, wg, bg, _on_gpu(dy, False), kept=kept)[1:]
        assert all(torch.equal(a, b) for a, b in zip(got, expected))


def test_layer():
    """The layer on GPU tensors, under autocast, and on tensors that the kernels do not take."""
    torch.manual_seed(0)
    layer = GroupNorm2d(4, 40, activation="gelu", checkpoint_8bit=True)
    with torch.no_grad():
        layer.weight.uniform_(0.5, 1.5)
        layer.bias.uniform_(-0.5, 0.5)
    x = torch.randn(2, 40, 6, 7)
    expected = layer(x)  # torch's, on the CPU
    layer = layer.cuda()
    with torch.autocast("cuda", dtype=torch.float16):
        y = layer(x.cuda().contiguous(memory_format=CL))
    assert y.dtype == FLOAT
    torch.testing.assert_close(y.cpu(), expected, rtol=1e-5, atol=1e-5)
    y.sum().backward()
    assert layer.weight.grad.shape == (40,) and torch.isfinite(layer.weight.grad).all()
    odd = GroupNorm2d(3, 9, activation="relu").cuda()
    assert odd(torch.randn(2, 9, 4, 4, device="cuda")).shape == (2, 9, 4, 4)
    flat = GroupNorm2d(4, 40, activation="silu").cuda()
    assert flat(torch.randn(2, 40, 11, device="cuda")).shape == (2, 40, 11)
