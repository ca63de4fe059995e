"""The group norm, the activations and the 8-bit form in 64 bits on the CPU, from their definitions."""

import math

import torch

CL = torch.channels_last


def activate(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    return z


def slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def pack_blocks(blocks):
    """(codes, exponent bytes) of finite blocks [..., values], by the definition: the smallest step 2**k, k >= -126, of
    which the largest magnitude is less than 127.5; codes by rounding to even, 127 at most."""
    b = blocks.double()
    top = b.abs().amax(-1)
    k = torch.full(top.shape, -126, dtype=torch.int64)
    for candidate in range(-126, 122):
        k = torch.where(top >= 127.5 * 2.0**candidate, candidate + 1, k)
    k = k.clamp_max(121)  # byte 254
    codes = torch.round(b / torch.pow(torch.tensor(2.0, dtype=torch.float64), k.double())[..., None]).clamp(-127, 127)
    return codes.to(torch.int8), (k + 6 + 127).to(torch.uint8)


def _in_blocks(rows, function):
    """function of blocks of 32 of the last dimension, the last block with what is left, for a list of outputs."""
    length = rows.shape[-1]
    whole = length // 32 * 32
    parts = []
    if whole:
        parts.append(function(rows[..., :whole].unflatten(-1, (-1, 32))))
    if whole < length:
        parts.append(function(rows[..., None, whole:]))
    codes = torch.cat([p[0].flatten(-2) for p in parts], -1)
    exponents = torch.cat([p[1] for p in parts], -1)
    return codes, exponents


def pack_rows(rows):
    """Codes and exponent bytes of blocks of 32 along the last dimension."""
    return _in_blocks(rows, pack_blocks)


def values(codes, exponents):
    """What they stand for, in 64 bits; NaN in blocks with byte 255."""
    steps = torch.pow(torch.tensor(2.0, dtype=torch.float64), exponents.double() - 133)
    steps = torch.where(exponents == 255, float("nan"), steps)
    return codes.double() * steps.repeat_interleave(32, -1)[..., : codes.shape[-1]]


def group_norm(x, groups, weight, bias, eps, act, dy=None, kept=False):
    """y and, with dy, grad_input, grad_weight, grad_bias (always made) of NCHW tensors, and what z is in the backward
    pass.  `kept`: the backward pass has the values of the 8-bit form of x, mean and deviation are those of x."""
    x = x.double()
    n, c = x.shape[:2]

    def spread(per_group):  # [n, groups] -> [n, c, 1, 1]
        return per_group.repeat_interleave(c // groups, 1)[:, :, None, None]

    grouped = x.reshape(n, groups, -1)
    mean = grouped.mean(-1)
    rstd = 1 / (((grouped - mean[..., None]) ** 2).mean(-1) + eps).sqrt()
    w = torch.ones(c, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(c, dtype=torch.float64) if bias is None else bias.double()
    w, b = w[:, None, None], b[:, None, None]
    z = (x - spread(mean)) * spread(rstd) * w + b
    out = [activate(z, act)]
    if dy is None:
        return out
    if kept:
        x = values(*pack_rows(x.permute(0, 2, 3, 1))).permute(0, 3, 1, 2)
    xhat = (x - spread(mean)) * spread(rstd)
    z = xhat * w + b
    dz = dy.double() * slope(z, act)
    g = dz * w
    mean_g = spread(g.reshape(n, groups, -1).mean(-1))
    mean_gx = spread((g * xhat).reshape(n, groups, -1).mean(-1))
    out += [spread(rstd) * (g - mean_g - xhat * mean_gx), (dz * xhat).sum((0, 2, 3)), dz.sum((0, 2, 3))]
    return out, z, (dz * xhat).abs().sum((0, 2, 3)), dz.abs().sum((0, 2, 3))


def rounding(exact, dtype):
    """Half of the distance between neighbouring values: eps/2 of the value, and below the smallest normal one, where they
    are as far apart as there (2**-24 in float16), half of that."""
    info = torch.finfo(dtype)
    return info.eps / 2 * exact.abs() + info.smallest_normal * info.eps / 2


def assert_within(got, exact, tolerance, what=""):
    """|got - exact| <= tolerance everywhere (tensors or a number); both in 64 bits."""
    error = (got.double().cpu() - exact).abs()
    bad = ~(error <= tolerance)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, the worst by {float(error[bad].max())}"
