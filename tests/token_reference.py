"""The operators over sequences of tokens by their definitions, token by token in 64 bits on the CPU, with the sums of the
magnitudes of what is added: what the kernels' 32 bits can be off by is a share of these.

A kernel's multiply-adds, products and exponentials are each off by at most a few units of 2^-24 of their result (an
exponential's argument x by a few |x| of them, which e^-|x| outweighs; a softplus by 8 and twice its argument), so that a sum of k such terms, each the product of up to m
factors, is off by at most (k + 4 m + 16) 2^-24 of the sum of their magnitudes; what is stored is rounded by half a step more.
"""

import torch

U = 2.0**-24


def tolerance(actual, expected, magnitudes, terms):
    """Differences allowed at every element: half a step of the type, and `terms` units of the magnitudes."""
    half = torch.finfo(actual.dtype).eps / 2
    tiny = torch.finfo(actual.dtype).smallest_normal
    return half * expected.abs() * (1 + 2 * half) + terms * U * magnitudes * (1 + half) + tiny * half


def check(what, actual, expected, magnitudes, terms):
    actual, dtype = actual.detach().cpu(), actual.dtype
    assert actual.shape == expected.shape, (what, actual.shape, expected.shape)
    off = (actual.double() - expected).abs()
    allowed = tolerance(actual, expected, magnitudes, terms)
    bad = ~(off <= allowed)
    assert not bad.any(), f"{what} ({dtype}): {int(bad.sum())} of {bad.numel()} off, worst {float((off / allowed)[bad].max()):.2f} times"


def sigmoid(z):
    return 1 / (1 + torch.exp(-z))


def double(*tensors):
    return [None if t is None else t.detach().cpu().double() for t in tensors]


def conv1d(x, weight, bias, act, before, dy):
    """Outputs, state behind, and gradients for x, weight, bias, each with its magnitudes."""
    x, weight, bias, before, dy = double(x, weight, bias, before, dy)
    n, l, c = x.shape
    width = weight.shape[1]
    before = torch.zeros(n, width - 1, c, dtype=torch.float64) if before is None else before
    window = torch.cat([before, x], 1)

    def sums(window, weight, bias):
        z = torch.zeros(n, l, c, dtype=torch.float64) + (0 if bias is None else bias)
        for i in range(width):
            z = z + window[:, i : i + l] * weight[:, i]
        return z

    z = sums(window, weight, bias)
    zm = sums(window.abs(), weight.abs(), None if bias is None else bias.abs())
    s = sigmoid(z) if act == "silu" else torch.ones_like(z)
    y = z * s
    slope = s * (1 + z * (1 - s)) if act == "silu" else s
    # silu's slope is at most 1.1, its own at most 0.5
    out = [(y, 1.1 * zm), (window[:, l:], torch.zeros_like(window[:, l:]))]
    if dy is None:
        return out
    dz, dzm = dy * slope, dy.abs() * (1.1 + (0.5 * zm if act == "silu" else 0))

    def back(dz, window, weight):
        dx = torch.zeros_like(x)
        dw = torch.zeros_like(weight)
        for i in range(width):
            shift = width - 1 - i
            dx[:, : l - shift if shift < l else 0] += (dz * weight[:, i])[:, shift:]
            dw[:, i] = (dz * window[:, i : i + l]).sum((0, 1))
        return dx, dw, dz.sum((0, 1))

    return out + list(zip(back(dz, window, weight), back(dzm, window.abs(), weight.abs())))


def _scan(u, dl, A, B, C, D, before, dy, rate):
    """y, last state, and gradients for u, dl, A, B, C, D; `rate` multiplies where A does so itself."""
    n, l, c = u.shape
    h = [before]
    y = torch.zeros_like(u)
    for t in range(l):
        h.append(torch.exp(dl[:, t, :, None] * A) * h[-1] + (dl[:, t] * u[:, t])[..., None] * B[:, t, None])
        y[:, t] = (h[-1] * C[:, t, None]).sum(-1) + D * u[:, t]
    if dy is None:
        return y, h[-1], ()
    du, ddl, dA, dB, dC = (torch.zeros_like(v) for v in (u, dl, A, B, C))
    r = torch.zeros_like(before)
    for t in range(l - 1, -1, -1):
        g = C[:, t, None] * dy[:, t, :, None] + r
        a = torch.exp(dl[:, t, :, None] * A)
        dC[:, t] = (dy[:, t, :, None] * h[t + 1]).sum(1)
        dB[:, t] = (g * (dl[:, t] * u[:, t])[..., None]).sum(1)
        gB = (g * B[:, t, None]).sum(-1)
        w = g * a * h[t]
        du[:, t] = gB * dl[:, t] + D * dy[:, t]
        ddl[:, t] = gB * u[:, t] + (w * rate).sum(-1)
        dA += (w * dl[:, t, :, None]).sum(0)
        r = a * g
    return y, h[-1], (du, ddl, dA, dB, dC, (dy * u).sum((0, 1)))


def scan(u, delta, A, B, C, D, gate, bias, softplus, before, dout):
    """Outputs, last state, and gradients for u, delta, A, B, C, D, gate, bias, each with its magnitudes."""
    u, delta, A, B, C, D, gate, bias, before, dout = double(u, delta, A, B, C, D, gate, bias, before, dout)
    n, l, c = u.shape
    D = torch.zeros(c, dtype=torch.float64) if D is None else D
    raw = delta if bias is None else delta + bias
    dl = torch.log1p(torch.exp(-raw.abs())) + raw.clamp_min(0) if softplus else raw
    before = torch.zeros(n, c, A.shape[1], dtype=torch.float64) if before is None else before
    s = torch.ones_like(u) if gate is None else sigmoid(gate)
    v = torch.ones_like(u) if gate is None else gate * s
    dy = None if dout is None else dout * v
    y, h, grads = _scan(u, dl, A, B, C, D, before, dy, A)
    # (dl may be negative without softplus: its magnitude where it multiplies, itself in the decays)
    sign = torch.where(dl < 0, -1.0, 1.0)
    ym, hm, gradsm = _scan(u.abs() * sign, dl, A, B.abs(), C.abs(), D.abs() * 0, before.abs(), None if dy is None else dy.abs(), A.abs())
    ym = ym + D.abs() * u.abs()
    out = [(y * v, ym * v.abs()), (h, hm)]
    if dout is None:
        return out
    du, ddl, dA, dB, dC, dD = grads
    dum, ddlm, dAm, dBm, dCm, dDm = (g.abs() for g in gradsm)
    dum = dum + D.abs() * dy.abs()
    dDm = (dy.abs() * u.abs()).sum((0, 1))
    slope = sigmoid(raw) if softplus else torch.ones_like(raw)
    slope_of_gate = torch.zeros_like(u) if gate is None else s * (1 + gate * (1 - s))
    ddelta, ddeltam = ddl * slope, ddlm * slope
    return out + [(du, dum), (ddelta, ddeltam), (dA, dAm), (dB, dBm), (dC, dCm), (dD, dDm),
                  (dout * y * slope_of_gate, dout.abs() * ym * 1.1), (ddelta.sum((0, 1)), ddeltam.sum((0, 1)))]  # fmt: skip


def rotary(x, weight, positions, frequencies, eps, interleaved, scale, dy):
    """Outputs and gradients for x and the weight of one tensor [n, l, heads, d], each with its magnitudes."""
    x, weight, dy = double(x, weight, dy)
    positions, frequencies = positions.detach().cpu().double(), frequencies.detach().cpu()
    angles = (positions[..., None] * frequencies)[..., None, :]
    cos, sin = torch.cos(angles) * scale, torch.sin(angles) * scale
    pairs = frequencies.shape[0]

    def turned(x, cos, sin, minus):
        out = x.clone()
        first = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
        second = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
        out[..., first] = x[..., first] * cos + minus * x[..., second] * sin
        out[..., second] = x[..., second] * cos - minus * x[..., first] * sin
        return out

    def pair_sums(x):  # of both channels of a pair, whatever the angle
        out = x.clone()
        first = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
        second = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
        both = (x[..., first] + x[..., second]) * abs(scale)
        out[..., first], out[..., second] = both, both
        return out

    if weight is None:
        n = x
    else:
        rstd = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        xhat = x * rstd
        n = xhat * weight
    out = [(turned(n, cos, sin, -1), pair_sums(n.abs()))]
    if dy is None:
        return out
    dn, dnm = turned(dy, cos, -sin, -1), pair_sums(dy.abs())
    if weight is None:
        return out + [(dn, dnm)]
    g, gm = dn * weight, dnm * weight.abs()
    dx = rstd * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    dxm = rstd * (gm + xhat.abs() * (gm * xhat.abs()).mean(-1, keepdim=True))
    return out + [(dx, dxm), ((dn * xhat).sum((0, 1, 2)), (dnm * xhat.abs()).sum((0, 1, 2)))]
