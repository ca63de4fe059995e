"""What the operators of token-mixing layers are timed on: those of state-space layers (a short causal convolution and
the selective scan behind it) and those of attention layers (rotary positions, alone and behind the norm of each head).

A case is one pass through a public operator on tensors that are already on the GPU, tokens by channels in memory:

  conv    causal_conv1d with an activation, or causal_conv1d_step
  scan    selective_scan with its gate, or selective_scan_step
  rotary  rotary on queries and keys
  norm    head_norm_rotary on queries and keys

with "mode" "infer" (a prompt, without gradients; the convolution and the scan return the state that decoding goes on
from), "train" (outputs and all gradients) or "step" (one token a sequence; the state goes to a second buffer, so that a
pass can be repeated).

Sizes are those of the package's network (widths 192 to 1536, its images as sequences of 196 to 3136 pixels), or generic
ones of language models' layers, and odd ones between them.

The plain forms are elementary torch operations in 32 bits; `exact` is the definition in 64.
"""

import math

import torch

own = False

EPS = 1e-6


def _conv(mode, n, l, c, w=4, dtype="bfloat16", act="silu", name=None):
    case = {"op": "conv", "mode": mode, "n": n, "l": l, "c": c, "w": w, "dtype": dtype, "act": act}
    return case if name is None else dict(case, name=name)


def _scan(mode, n, l, c, s=16, dtype="bfloat16", gate=True, name=None):
    case = {"op": "scan", "mode": mode, "n": n, "l": l, "c": c, "s": s, "dtype": dtype, "gate": gate}
    return case if name is None else dict(case, name=name)


def _rotary(op, mode, n, l, q, k, d, r, dtype="bfloat16", interleaved=False, start=0, factor=1.0, name=None):
    case = {"op": op, "mode": mode, "n": n, "l": l, "q": q, "k": k, "d": d, "r": r, "dtype": dtype,
            "interleaved": interleaved, "start": start, "factor": factor}  # fmt: skip
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # one sequence's next token: nothing but the latency of a call
        _conv("step", 1, 1, 1536, name="conv step 1n 1536c"),
        # one prompt of odd length
        _conv("infer", 1, 2051, 1536, dtype="float16", name="conv prompt 1n 2051l 1536c f16"),
        # training at an ordinary batch
        _conv("train", 8, 2048, 2048, name="conv train 8n 2048l 2048c"),
        # the next tokens of a served batch: as much state as fits the caches
        _scan("step", 64, 1, 1536, name="scan step 64n 1536c 16s"),
        # one long prompt of odd length: few channels behind each other's tokens
        _scan("infer", 1, 4099, 1536, dtype="float16", name="scan prompt 1n 4099l 1536c f16"),
        # training on text
        _scan("train", 4, 2048, 2048, name="scan train 4n 2048l 2048c"),
        # training on images of 14x14 pixels: short sequences, many of them
        _scan("train", 128, 196, 768, dtype="float16", name="scan train 128n 196l 768c f16"),
        # a small ragged layer in float32, eight states a channel
        _scan("train", 2, 777, 200, 8, "float32", name="scan train 2n 777l 200c 8s f32"),
        # the next tokens of eight sequences of different lengths, far into a long context
        _rotary("rotary", "infer", 8, 1, 12, 12, 64, 64, start=20000, name="rotary step 8n 12q 12k 64d"),
        # training with a rotation of the first 32 of 80 channels, in neighbouring pairs
        _rotary("rotary", "train", 2, 4097, 16, 16, 80, 32, "float16", True,
                name="rotary train 2n 4097l 80d f16"),  # fmt: skip
        # training with normed heads, three queries a key
        _rotary("norm", "train", 4, 2048, 24, 8, 128, 128, name="norm train 4n 2048l 24q 8k 128d"),
        # a long prompt in a context that the frequencies were scaled for
        _rotary("norm", "infer", 1, 16385, 32, 8, 128, 128, start=100000, factor=8.0,
                name="norm prompt 1n 16385l 32q 8k 128d"),  # fmt: skip
    ]


def _log_uniform(rng, low, high):
    return math.exp(rng.uniform(math.log(low), math.log(high)))


def draw(rng):
    sizes = [work(c) for c in listed()]
    least, most = min(w["bytes"] for w in sizes), {k: max(w[k] for w in sizes) for k in ("bytes", "flops")}
    while True:
        op = rng.choices(("conv", "scan", "rotary", "norm"), weights=(3, 5, 2, 3))[0]
        dtype = rng.choices(("bfloat16", "float16", "float32"), weights=(4, 3, 2))[0]
        n = round(_log_uniform(rng, 1, 128))
        if op in ("conv", "scan"):
            mode = rng.choices(("infer", "train", "step"), weights=(3, 4, 2))[0]
            l = 1 if mode == "step" else round(_log_uniform(rng, 1, 8192))
            c = round(_log_uniform(rng, 8, 4096))
            if op == "conv":
                case = _conv(mode, n, l, -(-c // 8) * 8, rng.choice((2, 3, 4, 4, 4, 5)), dtype,
                             rng.choice(("none", "silu", "silu")))  # fmt: skip
            else:
                states = rng.choice((16, 16, 16, 8, rng.randint(1, 32)))
                case = _scan(mode, n, l, c, states, dtype, rng.random() < 0.8)
        else:
            mode = rng.choice(("infer", "train"))
            l = 1 if mode == "infer" and rng.random() < 0.3 else round(_log_uniform(rng, 1, 16384))
            d = rng.choice((32, 64, 64, 80, 96, 128, 128, 128, 192, 256))
            k = round(_log_uniform(rng, 1, 32))
            q = k * rng.choice([g for g in (1, 2, 3, 4, 8) if k * g <= 64])
            interleaved = rng.random() < 0.4
            r = rng.choice((d, d, d // 2 // 16 * 16, d // 4 // 16 * 16)) or d
            r = r if interleaved else r // 16 * 16
            case = _rotary(op, mode, n, l, q, k, d, r, dtype, interleaved, rng.choice((0, 0, round(_log_uniform(rng, 1, 500000)))),
                           rng.choice((1.0, 1.0, 4.0, 8.0)))  # fmt: skip
        w = work(case)
        if least <= w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return case


def _frequencies(case):
    """Radians a position of each rotated pair; `factor` scales the low ones for a context that many times as long."""
    base = 10000.0
    f = base ** (-2.0 * torch.arange(case["r"] // 2, dtype=torch.float64) / case["r"])
    turns = f * 8192 / (2 * math.pi)  # of the context that was trained on
    keep = ((turns - 1) / 31).clamp(0, 1)  # all of the fast ones, none of those that do not make a turn
    return f * keep + f / case["factor"] * (1 - keep)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, op, mode = getattr(torch, case["dtype"]), case["op"], case["mode"]
    n, l = case["n"], case["l"]

    def uniform(shape, low, high, dt=torch.float32):
        return torch.empty(shape, device="cuda").uniform_(low, high, generator=gen).to(dt)

    def normal(*shape, dt=dtype):
        return torch.empty(shape, device="cuda", dtype=dt).normal_(generator=gen)

    state = {"case": case}
    leaves = []
    if op == "conv":
        c, w = case["c"], case["w"]
        state["x"] = normal(n, l, c).mul_(uniform((c,), 0.5, 2.0, dtype))
        limit = 1 / math.sqrt(w)
        # weights of a served model are in its type, those of a trained one in float32
        state["weight"] = uniform((c, w), -limit, limit, torch.float32 if mode == "train" else dtype)
        state["bias"] = uniform((c,), -limit, limit, torch.float32 if mode == "train" else dtype)
        leaves = ["x", "weight", "bias"]
        state["dy"] = normal(n, l, c)
        if mode == "step":
            state["x"] = state["x"].reshape(n, c)
            state["before"] = normal(n, w - 1, c)
            state["after"] = torch.empty_like(state["before"])
    elif op == "scan":
        c, s = case["c"], case["s"]
        state["u"] = normal(n, l, c)
        state["delta"] = normal(n, l, c).mul_(0.5)
        # as a trained layer has them: rates around 1..s, time steps from 0.001 to 0.1
        state["A"] = -torch.arange(1, s + 1, device="cuda").float() * uniform((c, s), 0.8, 1.25)
        step = torch.exp(uniform((c,), math.log(1e-3), math.log(0.1)))
        state["delta_bias"] = step + torch.log(-torch.expm1(-step))
        state["D"] = uniform((c,), 0.5, 1.5)
        # one projection makes the rank of delta, B and C: rows of a wider tensor
        rows = normal(n, l, 2 * s + 24)
        state["B"], state["C"] = rows[..., 24 : 24 + s], rows[..., 24 + s :]
        state["gate"] = normal(n, l, c) if case["gate"] else None
        state["dy"] = normal(n, l, c)
        leaves = ["u", "delta", "A", "B", "C", "D", "delta_bias"] + (["gate"] if case["gate"] else [])
        if mode == "step":
            for key in ("u", "delta", "B", "C", "gate"):
                state[key] = None if state[key] is None else state[key][:, 0]
            state["before"] = normal(n, c, s, dt=torch.float32)
            state["after"] = torch.empty_like(state["before"])
    else:
        q, k, d = case["q"], case["k"], case["d"]
        # one projection makes queries, keys and values
        rows = normal(n, l, (q + 2 * k) * d).mul_(uniform(((q + 2 * k) * d,), 0.5, 2.0, dtype))
        state["q"] = rows[..., : q * d].unflatten(-1, (q, d))
        state["k"] = rows[..., q * d : (q + k) * d].unflatten(-1, (k, d))
        first = torch.randint(0, case["start"] + 1, (n, 1), device="cuda", generator=gen) if l == 1 else case["start"]
        state["positions"] = torch.arange(l, device="cuda") + first
        state["frequencies"] = _frequencies(case).cuda()
        state["scale"] = 0.1 * math.log(case["factor"]) + 1
        state["dq"], state["dk"] = normal(n, l, q, d), normal(n, l, k, d)
        leaves = ["q", "k"]
        if op == "norm":
            state["q_weight"], state["k_weight"] = uniform((d,), 0.5, 1.5), uniform((d,), 0.5, 1.5)
            leaves += ["q_weight", "k_weight"]
    if mode == "train":
        for key in leaves:
            state[key] = state[key].detach().requires_grad_()
        state["leaves"] = [state[key] for key in leaves]
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from spio_amd import functional as F

    case = state["case"]
    mode = case["mode"]
    if case["op"] == "conv":
        if mode == "step":
            y = F.causal_conv1d_step(state["x"], state["before"], state["weight"], state["bias"], case["act"],
                                     out_state=state["after"])  # fmt: skip
            return [y, state["after"]]
        y = F.causal_conv1d(state["x"], state["weight"], state["bias"], case["act"], return_state=mode == "infer")
        if mode == "infer":
            return list(y)
        return [y.detach(), *torch.autograd.grad(y, state["leaves"], state["dy"])]
    if case["op"] == "scan":
        args = [state[key] for key in ("u", "delta", "A", "B", "C", "D", "gate", "delta_bias")]
        if mode == "step":
            y = F.selective_scan_step(state["u"], state["before"], *args[1:], delta_softplus=True, out_state=state["after"])
            return [y, state["after"]]
        y = F.selective_scan(*args, delta_softplus=True, return_state=mode == "infer")
        if mode == "infer":
            return list(y)
        return [y.detach(), *torch.autograd.grad(y, state["leaves"], state["dy"])]
    rest = dict(interleaved=case["interleaved"], scale=state["scale"])
    if case["op"] == "norm":
        out = F.head_norm_rotary(state["q"], state["k"], state["q_weight"], state["k_weight"], state["positions"],
                                 state["frequencies"], eps=EPS, **rest)  # fmt: skip
    else:
        out = F.rotary(state["q"], state["k"], state["positions"], state["frequencies"], **rest)
    if mode == "infer":
        return list(out)
    return [*(t.detach() for t in out), *torch.autograd.grad(out, state["leaves"], [state["dq"], state["dk"]])]


# ---- plain form: elementary operations in 32 bits, rounded once at the end ----


def _silu(z):
    """(value, derivative)"""
    s = 1 / (1 + torch.exp(-z))
    return z * s, s * (1 + z * (1 - s))


def _run_plain(state):
    with torch.no_grad():
        if state["case"]["op"] == "conv":
            return _plain_conv(state)
        if state["case"]["op"] == "scan":
            return _plain_scan(state)
        return _plain_rotary(state)


def _plain_conv(state):
    case = state["case"]
    x, w, dtype = state["x"], state["weight"].float(), state["x"].dtype
    width, c = case["w"], case["c"]
    xf = (x[:, None] if case["mode"] == "step" else x).float()
    n, l = xf.shape[:2]
    before = state["before"].float() if case["mode"] == "step" else xf.new_zeros(n, width - 1, c)
    padded = torch.cat([before, xf], 1)
    z = sum(padded[:, i : i + l] * w[:, i] for i in range(width)) + state["bias"].float()
    y, slope = _silu(z) if case["act"] == "silu" else (z, torch.ones_like(z))
    if case["mode"] == "step":
        return [y[:, 0].to(dtype), padded[:, 1:].to(dtype)]
    if case["mode"] == "infer":
        return [y.to(dtype), padded[:, l:].to(dtype)]
    dz = state["dy"].float() * slope
    behind = torch.cat([dz, dz.new_zeros(n, width - 1, c)], 1)
    dx = sum(behind[:, width - 1 - i : width - 1 - i + l] * w[:, i] for i in range(width))
    # sequence by sequence first: sums over all tokens at once are long for 32 bits
    dw = torch.stack([(dz * padded[:, i : i + l]).sum(1).sum(0) for i in range(width)], -1)
    return [y.to(dtype), dx.to(dtype), dw, dz.sum(1).sum(0)]


def _doubled(a, b):
    """h with h[t] = a[t] h[t-1] + b[t] along the second dimension, by spans of doubling length."""
    span, length = 1, b.shape[1]
    while span < length:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1) if 2 * span < length else a
        span *= 2
    return b


def _plain_scan(state):
    case = state["case"]
    step, dtype = case["mode"] == "step", state["u"].dtype

    def f(key):
        t = state[key]
        return None if t is None else (t[:, None] if step else t).float()

    u, raw, B, C, gate = f("u"), f("delta"), f("B"), f("C"), f("gate")
    A, D = state["A"], state["D"]
    raw = raw + state["delta_bias"]
    delta = torch.where(raw > 20, raw, torch.log1p(torch.exp(raw.clamp(max=20))))
    a = torch.exp(delta[..., None] * A)
    b = (delta * u)[..., None] * B[:, :, None]
    h = a * state["before"][:, None] + b if step else _doubled(a, b)
    y = (h * C[:, :, None]).sum(-1) + D * u
    out = y if gate is None else y * _silu(gate)[0]
    if step:
        return [out[:, 0].to(dtype), h[:, 0]]
    if case["mode"] == "infer":
        return [out.to(dtype), h[:, -1].clone()]
    dout = state["dy"].float()
    dgate = None
    if gate is not None:
        value, slope = _silu(gate)
        dgate = (dout * y * slope).to(dtype)
        dout = dout * value
    # the same recurrence from the last token to the first
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _doubled(later.flip(1), (dout[..., None] * C[:, :, None]).flip(1)).flip(1)
    dC = (dout[..., None] * h).sum(2)
    dB = (g * (delta * u)[..., None]).sum(2)
    gb = (g * B[:, :, None]).sum(-1)
    du = gb * delta + dout * D
    da = g[:, 1:] * h[:, :-1] * a[:, 1:]
    dA = (da * delta[:, 1:, :, None]).sum(1).sum(0)
    ddelta = gb * u
    ddelta[:, 1:] += (da * A).sum(-1)
    ddelta = ddelta / (1 + torch.exp(-raw))
    out = [out.to(dtype), du.to(dtype), ddelta.to(dtype), dA, dB.to(dtype), dC.to(dtype), (dout * u).sum(1).sum(0),
           ddelta.sum(1).sum(0)]  # fmt: skip
    return out if dgate is None else [*out, dgate]


def _rotated(x, cos, sin, interleaved):
    """x [n, l, h, d] with cosines and sines [*, l, 1, r / 2] of its first r channels' pairs."""
    r = 2 * cos.shape[-1]
    if interleaved:
        first, second = x[..., 0:r:2], x[..., 1:r:2]
    else:
        first, second = x[..., : r // 2], x[..., r // 2 : r]
    pair = first * cos - second * sin, second * cos + first * sin
    turned = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
    return torch.cat([turned, x[..., r:]], -1)


def _plain_rotary(state):
    case = state["case"]
    # angles of far positions are rounded by whole parts of a turn in 32 bits
    angles = (state["positions"].double()[..., None] * state["frequencies"])[..., None, :]
    cos, sin = (torch.cos(angles) * state["scale"]).float(), (torch.sin(angles) * state["scale"]).float()
    outputs, gradients, sums = [], [], []
    for key in ("q", "k"):
        x = state[key]
        y = x.float()
        if case["op"] == "norm":
            weight = state[key + "_weight"]
            rstd = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
            xhat = y * rstd
            y = xhat * weight
        outputs.append(_rotated(y, cos, sin, case["interleaved"]).to(x.dtype))
        if case["mode"] == "train":
            dx = _rotated(state["d" + key].float(), cos, -sin, case["interleaved"])
            if case["op"] == "norm":
                sums.append((dx * xhat).sum(2).sum(1).sum(0))
                dx = dx * weight
                dx = rstd * (dx - xhat * (dx * xhat).mean(-1, keepdim=True))
            gradients.append(dx.to(x.dtype))
    return outputs + gradients + sums


# ---- the definition in 64 bits ----


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "conv":
        return _exact_conv(state)
    if case["op"] == "scan":
        return _exact_scan(state)
    return _exact_rotary(state)


def _leaf(t):
    return None if t is None else t.detach().double().requires_grad_()


def _exact_conv(state):
    case = state["case"]
    x, w, b = (_leaf(state[k]) for k in ("x", "weight", "bias"))
    tokens = x[:, None] if case["mode"] == "step" else x
    n, l, c = tokens.shape
    keep = case["w"] - 1
    past = state["before"].double() if case["mode"] == "step" else tokens.new_zeros(n, keep, c)
    window = torch.cat([past, tokens], 1)
    z = torch.matmul(window.unfold(1, case["w"], 1).unsqueeze(-2), w.unsqueeze(-1)).squeeze(-1).squeeze(-1) + b
    y = torch.nn.functional.silu(z) if case["act"] == "silu" else z
    if case["mode"] == "train":
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), state["dy"].double())]
    after = window[:, window.shape[1] - keep :].detach()
    return [(y[:, 0] if case["mode"] == "step" else y).detach(), after]


def _exact_scan(state):
    """Token by token; the gradients by torch's differentiation of each token's step, from the last to the first."""
    case = state["case"]
    if case["n"] * case["l"] * case["c"] * case["s"] > 1 << 30 or (case["mode"] == "train" and case["l"] > 4096):
        return None
    names = ("u", "delta", "A", "B", "C", "D", "delta_bias", "gate")
    u, delta, A, B, C, D, bias, gate = (None if state[k] is None else state[k].detach().double() for k in names)
    if case["mode"] == "step":
        u, delta, B, C, gate = (None if t is None else t[:, None] for t in (u, delta, B, C, gate))

    def advance(h, u, delta, A, B, C, D, bias, gate):
        dt = torch.nn.functional.softplus(delta + bias, threshold=1e9)
        h = torch.exp(dt[..., None] * A) * h + dt[..., None] * u[..., None] * B[:, None]
        y = (h * C[:, None]).sum(-1) + D * u
        return h, y if gate is None else y * torch.nn.functional.silu(gate)

    def token(t):
        return u[:, t], delta[:, t], A, B[:, t], C[:, t], D, bias, None if gate is None else gate[:, t]

    n, l, c = u.shape
    before = state["before"].double() if case["mode"] == "step" else u.new_zeros(n, c, case["s"])
    states, outputs = [before], []
    train = case["mode"] == "train"
    for t in range(l):
        h, y = advance(states[-1], *token(t))
        if not train:
            states.clear()
        states.append(h)
        outputs.append(y)
    out = torch.stack(outputs, 1)
    if not train:
        return [out[:, 0] if case["mode"] == "step" else out, states[-1]]
    grads = [None if v is None else torch.zeros_like(v) for v in (u, delta, A, B, C, D, bias, gate)]
    dh = torch.zeros_like(before)
    for t in range(l - 1, -1, -1):
        given = [None if v is None else v.detach().requires_grad_() for v in (states[t], *token(t))]
        with torch.enable_grad():
            h, y = advance(*given)
        wanted = [v for v in given if v is not None]
        got = iter(torch.autograd.grad((h, y), wanted, (dh, state["dy"][:, t].double())))
        dh = next(got)
        for i, total in enumerate(grads):
            if total is None:
                continue
            if i in (2, 5, 6):  # of all tokens
                total += next(got)
            else:
                total[:, t] = next(got)
    return [out, *(g for g in grads if g is not None)]


def _exact_rotary(state):
    case = state["case"]
    angles = state["positions"].double()[..., None, None] * state["frequencies"].double()
    turn = torch.polar(torch.full_like(angles, state["scale"]), angles)
    names = ["q", "k"] + (["q_weight", "k_weight"] if case["op"] == "norm" else [])
    leaves = [_leaf(state[k]) for k in names]
    r, outputs = case["r"], []
    for i in range(2):
        x = leaves[i]
        if case["op"] == "norm":
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * leaves[2 + i]
        head = x[..., :r]
        pairs = head.unflatten(-1, (r // 2, 2)) if case["interleaved"] else head.unflatten(-1, (2, r // 2)).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        turned = turned if case["interleaved"] else turned.transpose(-1, -2)
        outputs.append(torch.cat([turned.flatten(-2), x[..., r:]], -1))
    if case["mode"] == "infer":
        return [y.detach() for y in outputs]
    grads = torch.autograd.grad(outputs, leaves, [state["dq"].double(), state["dk"].double()])
    return [*(y.detach() for y in outputs), *grads]


def work(case):
    """Inputs once and outputs once, a position or a state's rate counted as nothing beside them; additions, products and
    exponentials."""
    size = 4 if case["dtype"] == "float32" else 2
    n, l = case["n"], case["l"]
    train = case["mode"] == "train"
    if case["op"] == "conv":
        values = n * l * case["c"]
        kept = 0 if train else n * (case["w"] - 1) * case["c"]
        kept *= 2 if case["mode"] == "step" else 1
        params = case["c"] * (case["w"] + 1) * (8 if train else size)
        products = 2 * case["w"] + (4 if case["act"] == "silu" else 0)
        return {"bytes": ((4 if train else 2) * values + kept) * size + params,
                "flops": values * products * (4 if train else 1)}  # fmt: skip
    if case["op"] == "scan":
        values, rows = n * l * case["c"], n * l * case["s"]
        # u, delta, out, and dy with the gradients of the first two; the gate and its own
        tensors = (6 if train else 3) + case["gate"] * (2 if train else 1)
        state_bytes = 0 if train else n * case["c"] * case["s"] * 4 * (2 if case["mode"] == "step" else 1)
        params = case["c"] * (case["s"] + 2) * 4 * (2 if train else 1)
        return {"bytes": (tensors * values + rows * (4 if train else 2)) * size + state_bytes + params,
                "flops": values * case["s"] * (24 if train else 7)}  # fmt: skip
    values = n * l * (case["q"] + case["k"]) * case["d"]
    norm = case["op"] == "norm"
    return {"bytes": values * size * (4 if train else 2) + n * l * 8,
            "flops": values * (3 + 4 * norm) * (3 if train else 1)}  # fmt: skip
