"""pack_8bit, unpack_8bit, activation_8bit and conv2d_gw8_8bit against their definitions in 64 bits on the CPU.

Codes and exponents are whole numbers and have to be equal; so are the values they stand for, which 16 bits hold.
Activations and their gradients: float32 arithmetic, 2^-20 of the largest magnitude of an argument's neighbourhood (an
exponential's argument is rounded to 2^-24 of itself, up to 2^4), and half a step of the type they are rounded to.
"""

import pytest
import torch

from spio_amd.convnext_gw8 import ConvNeXtGw8
from spio_amd.functional import activation_8bit, conv2d_gw8, conv2d_gw8_8bit, pack_8bit, unpack_8bit
from spio_amd.functional.activation_8bit_function import activation_8bit_forward, pack_8bit_op
from spio_amd.functional.conv2d_gw8_8bit_function import conv2d_gw8_8bit_forward
from spio_amd.layers import Activation8bit, Conv2dGw8, GroupNorm2d
from tests.pointwise_reference import CL, activate, assert_within, rounding, pack_rows, slope, values

pytestmark = pytest.mark.gpu
HALF, BF16, FLOAT = torch.float16, torch.bfloat16, torch.float32
DTYPES = [HALF, BF16, FLOAT]


def _values(n, dtype, seed=0):
    """n values whose blocks differ in size by many powers of two."""
    g = torch.Generator().manual_seed(n + seed)
    size = torch.exp2(torch.randint(-12, 9, (-(-n // 32),), generator=g).float()).repeat_interleave(32)[:n]
    return (torch.randn(n, generator=g) * size).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 31, 32, 33, 40, 1000, 8192, 8193, 100_003])
def test_pack_and_unpack(n, dtype):
    x = _values(n, dtype)
    packed = pack_8bit(x.cuda())
    codes, exponents = pack_rows(x)
    assert torch.equal(packed.codes.cpu(), codes) and torch.equal(packed.exponents.cpu(), exponents)
    for target in DTYPES:
        back = unpack_8bit(packed, None if target == dtype else target)
        assert back.dtype == target and back.shape == x.shape
        exact = values(codes, exponents)
        assert torch.equal(back.cpu(), exact.to(target))


@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_at_the_ends_of_the_types(dtype):
    """Zeros, the smallest values, the largest, 127.5 steps (which are 64 of the next), ties, and blocks with an
    infinity or a NaN, which are lost whole and leave their neighbours alone."""
    info = torch.finfo(dtype)
    smallest = {HALF: 2.0**-24, BF16: 2.0**-133, FLOAT: 2.0**-149}[dtype]
    x = torch.zeros(9, 32)
    x[1, 5] = smallest
    x[2, :3] = torch.tensor([info.max, -info.max, 1.0])
    x[3, :4] = torch.tensor([127.5, 2.0, 3.0, -1.0])
    x[4, :5] = torch.tensor([127.0, 2.5, 3.5, -0.5, 0.5])
    x[5, :2] = torch.tensor([127.0, float("inf")])
    x[6, :2] = torch.tensor([1.0, -2.0])
    x[7, 31] = float("nan")
    x[8, :2] = torch.tensor([127.25, 126.75]) if dtype != BF16 else torch.tensor([127.0, 126.5])
    x = x.to(dtype)
    packed = pack_8bit(x.cuda())
    finite = torch.isfinite(x).all(1)
    codes, exponents = pack_rows(x[finite].reshape(-1))
    assert torch.equal(packed.codes.cpu().reshape(9, 32)[finite].reshape(-1), codes)
    assert torch.equal(packed.exponents.cpu()[finite], exponents)
    assert (packed.exponents.cpu()[~finite] == 255).all()
    back = unpack_8bit(packed).cpu().double()
    assert torch.isnan(back[~finite]).all() and torch.isfinite(back[finite]).all()
    exact = values(codes, exponents).clamp(-info.max, info.max).reshape(-1, 32)  # the largest may round up
    assert torch.equal(back[finite], exact)
    # half a step, where the largest value has at least 63.75 of them, or half of the smallest step, 2**-126
    bound = x[finite].double().abs().amax(1, True) / 127 + 2.0**-127
    assert ((back[finite] - x[finite].double()).abs() <= bound).all()


def test_layouts():
    """Blocks are neighbours in memory, whatever the strides; tensors with gaps are packed as their copies."""
    x = _values(2 * 24 * 5 * 7, HALF).reshape(2, 24, 5, 7).cuda()
    for t in (x, x.contiguous(memory_format=CL), x.transpose(1, 3), x[:, :, ::2], x[:1].expand(3, 24, 5, 7),
              x.reshape(-1)[1:], x.reshape(-1)[3:100]):  # fmt: skip
        packed = pack_8bit(t)
        back = unpack_8bit(packed)
        assert back.shape == t.shape
        seen = t if back.stride() == t.stride() else t.contiguous()
        flat = torch.as_strided(seen, (t.numel(),), (1,)).cpu()
        assert torch.equal(torch.as_strided(back, (t.numel(),), (1,)).cpu().double(), values(*pack_rows(flat)))
    empty = unpack_8bit(pack_8bit(x[:0]))
    assert empty.shape == (0, 24, 5, 7)


@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_activation_and_gradient(dtype, act):
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(3, 37, 5, 11, generator=g) * 4).to(dtype)
    dy = torch.randn(3, 37, 5, 11, generator=g).to(dtype)
    xg = x.cuda().requires_grad_()
    y = activation_8bit(xg, act)
    (dx,) = torch.autograd.grad(y, xg, dy.cuda())
    assert y.dtype == dx.dtype == dtype
    exact = activate(x.double(), act)
    assert_within(y.detach(), exact, rounding(exact, dtype) + 2.0**-20, "y")
    kept = values(*pack_rows(x.reshape(-1))).reshape(x.shape)
    exact = dy.double() * slope(kept, act)
    assert_within(dx, exact, rounding(exact, dtype) + 2.0**-20 * dy.double().abs(), "dx")
    with torch.no_grad():
        assert torch.equal(activation_8bit(xg, act), y)


def test_activation_far_out():
    """Where exponentials overflow and vanish: the ends of the type, infinity (z times a factor of one) and NaN."""
    x = torch.tensor([-65504.0, -100.0, -20.0, -14.0, 0.0, 14.0, 100.0, 65504.0, float("inf"), float("nan")])
    for dtype in DTYPES:
        xd = x.to(dtype)
        for act in ("relu", "silu", "gelu"):
            got = activation_8bit(xd.cuda(), act).cpu().double()
            torch.testing.assert_close(got, activate(xd.double(), act), rtol=1e-2, atol=1e-6, equal_nan=True)


@pytest.mark.parametrize("layout", ["channels_last", "strided", "off"])
def test_activation_layouts(layout):
    g = torch.Generator().manual_seed(5)
    x, dy = torch.randn(2, 16, 6, 9, generator=g).half(), torch.randn(2, 16, 6, 9, generator=g).half()
    xg = {"channels_last": lambda: x.cuda().contiguous(memory_format=CL),
          "strided": lambda: torch.stack([x, x], -1).cuda()[..., 1],
          "off": lambda: torch.cat([x.reshape(-1)[:1], x.reshape(-1)]).cuda()[1:].reshape(x.shape)}[layout]()  # fmt: skip
    xg.requires_grad_()
    y = activation_8bit(xg, "gelu")
    (dx,) = torch.autograd.grad(y, xg, dy.cuda())
    order = (0, 2, 3, 1) if layout == "channels_last" else (0, 1, 2, 3)
    kept = values(*pack_rows(x.permute(order).reshape(-1))).reshape(x.permute(order).shape)
    exact = dy.permute(order).double() * slope(kept, "gelu")
    assert_within(dx.permute(order), exact, rounding(exact, HALF) + 2.0**-20 * dy.permute(order).double().abs())


def test_tensors_that_pass_32_bits():
    x = _values(1 << 20, HALF).cuda()
    n = (1 << 31) + (1 << 20) + 8
    big = torch.cat([x.repeat(n >> 20), x[:8]])
    assert big.numel() > 1 << 31
    packed, part = pack_8bit(big), pack_8bit(x)
    back = unpack_8bit(packed)
    assert torch.equal(packed.codes[-(1 << 20) - 8 : -8], part.codes)
    assert torch.equal(back[-(1 << 20) - 8 : -8], unpack_8bit(part)) and torch.equal(back[: 1 << 20], unpack_8bit(part))
    del back, packed
    y, codes, exponents = activation_8bit_forward(big, "silu", True)
    assert torch.equal(y[-(1 << 20) - 8 : -8], activation_8bit(x, "silu"))
    assert torch.equal(codes[-(1 << 20) - 8 : -8], part.codes)


def test_convolution_with_a_checkpoint_in_8_bits():
    """Output and grad_input are conv2d_gw8's; grad_weight is its on the values that the checkpoint stands for."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(3, 40, 13, 11, generator=g).half().cuda().contiguous(memory_format=CL).requires_grad_()
    w = (torch.randn(40, 8, 3, 3, generator=g) * 0.1).half().cuda().contiguous(memory_format=CL).requires_grad_()
    b = torch.randn(40, generator=g).cuda().requires_grad_()
    dy = torch.randn(3, 40, 13, 11, generator=g).half().cuda().contiguous(memory_format=CL)
    y = conv2d_gw8_8bit(x, w, b, padding_y=1, padding_x=1, groups=5)
    assert torch.equal(y, conv2d_gw8(x, w, b, padding_y=1, padding_x=1, groups=5))
    got = torch.autograd.grad(y, [x, w, b], dy)
    kept = unpack_8bit(pack_8bit(x)).requires_grad_()
    expected = torch.autograd.grad(conv2d_gw8(kept, w, b, padding_y=1, padding_x=1, groups=5), [kept, w, b], dy)
    for a, e in zip(got, expected):  # (sums with atomics: their order differs)
        assert a.dtype == e.dtype
        torch.testing.assert_close(a.float(), e.float(), rtol=1e-3, atol=1e-4 * float(e.float().abs().max()))
    (dx,) = torch.autograd.grad(conv2d_gw8_8bit(x, w, b, padding_y=1, padding_x=1, groups=5), [x], dy)
    torch.testing.assert_close(dx, expected[0], rtol=1e-3, atol=1e-3)
    with torch.no_grad():
        assert torch.equal(conv2d_gw8_8bit(x, w, b, padding_y=1, padding_x=1, groups=5), y)
    with pytest.raises(AssertionError):
        conv2d_gw8_8bit(x.float(), w, b, padding_y=1, padding_x=1, groups=5)


def test_opcheck_and_compile():
    x = torch.randn(2, 16, 6, 9, device="cuda").half().contiguous(memory_format=CL).requires_grad_()
    w = torch.randn(16, 8, 3, 3, device="cuda").half().contiguous(memory_format=CL).requires_grad_()
    torch.library.opcheck(pack_8bit_op, (x.detach(),))
    torch.library.opcheck(activation_8bit_forward, (x, "gelu", True))
    torch.library.opcheck(conv2d_gw8_8bit_forward, (x, w, None, 1, 1), test_utils=("test_schema", "test_faketensor"))
    compiled = torch.compile(lambda t: activation_8bit(t, "silu"), backend="aot_eager")
    dy = torch.randn_like(x)
    got = torch.autograd.grad(compiled(x), x, dy)
    assert torch.equal(got[0], torch.autograd.grad(activation_8bit(x, "silu"), x, dy)[0])


def test_replays_of_a_captured_pass():
    x = torch.randn(3, 50, 33, device="cuda").half().requires_grad_()
    dy = torch.randn_like(x)

    def step():
        y = activation_8bit(x, "gelu")
        return [y.detach(), torch.autograd.grad(y, x, dy)[0], unpack_8bit(pack_8bit(x))]

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
            x.copy_(torch.randn(3, 50, 33, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_hooks_on_saved_tensors():
    """Codes and exponents are one-dimensional: hooks that pack and unpack them otherwise change nothing."""
    x = torch.randn(2, 16, 6, 9, device="cuda").half().contiguous(memory_format=CL).requires_grad_()
    dy = torch.randn_like(x)
    norm = GroupNorm2d(4, 16, activation="silu", checkpoint_8bit=True).cuda()

    def run():
        y = activation_8bit(norm(x), "gelu")
        return torch.autograd.grad(y, [x, *norm.parameters()], dy)

    expected = run()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().cpu(), lambda t: t.cuda()):
        got = run()
    assert all(torch.equal(a, b) for a, b in zip(got, expected))


def test_network_with_checkpoints_in_8_bits():
    """The ConvNeXt-shaped network with the three operators together: it keeps less between its passes, its logits
    are those without checkpoints but for the norms' kernels, and its gradients are close to them.  The checkpoints are
    off by 1/127.5 of a block's largest value at most, a relative error of about 2^-8 in the middle: gradients of the
    whole network by less than a tenth of their norm."""

    def build(kept):
        torch.manual_seed(0)

        def conv(dim):
            layer = Conv2dGw8(dim, dim, 3, padding=1, groups=dim // 8)
            layer.checkpoint_8bit = kept
            return layer

        return ConvNeXtGw8(conv, widths=(32, 64), depths=(2, 1), classes=10,
                           norm2d=lambda d: GroupNorm2d(4, d, activation="silu", checkpoint_8bit=kept),
                           make_act=Activation8bit if kept else torch.nn.GELU).cuda().to(memory_format=CL)  # fmt: skip

    x = torch.randn(4, 3, 64, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    grads, logits, kept_bytes = [], [], []
    for kept in (False, True):
        model = build(kept)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        with torch.autocast("cuda", dtype=torch.float16):
            y = model(x.contiguous(memory_format=CL))
        kept_bytes.append(torch.cuda.memory_allocated() - before)
        y.float().square().sum().backward()
        logits.append(y.detach().float())
        grads.append([p.grad for p in model.parameters()])
    assert kept_bytes[1] < 0.8 * kept_bytes[0]
    torch.testing.assert_close(logits[1], logits[0], rtol=1e-2, atol=1e-2 * float(logits[0].abs().max()))
    for a, e in zip(grads[1], grads[0]):
        assert (a - e).norm() <= 0.1 * e.norm() + 1e-6
