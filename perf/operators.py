"""What the channels-last group norm and the 8-bit activation checkpoints are timed on.

A case is one pass through a public operator on tensors that are already on the GPU:

  norm_infer  group_norm_2d with an activation, without gradients (serving, evaluation)
  norm_train  group_norm_2d with an activation and its gradients; with "bits": 8 the backward pass reads the
              input from the 8-bit checkpoint that the forward pass wrote
  act_infer   activation_8bit without gradients
  act_train   activation_8bit and its gradient: the forward pass keeps its input in 8 bits
  pack        pack_8bit and unpack_8bit: what a layer with an 8-bit checkpoint adds to its two passes

Sizes are those of the package's network (widths 96/192/384/768 at 56/28/14/7, its MLPs four times as wide), of
its benchmark and kernel tests, and odd ones between them.

The plain forms are elementary torch operations in 32 bits; `exact` is the definition in 64.
"""

import math

import torch

own = False

CL = torch.channels_last
EPS = 1e-5


def _norm(op, n, c, groups, h, w, dtype="float16", act="silu", bits=16, affine=True, name=None):
    case = {"op": op, "n": n, "c": c, "groups": groups, "h": h, "w": w, "dtype": dtype, "act": act, "bits": bits,
            "affine": affine}  # fmt: skip
    return case if name is None else dict(case, name=name)


def _flat(op, n, c, h, w, dtype="float16", act="gelu", name=None):
    case = {"op": op, "n": n, "c": c, "h": h, "w": w, "dtype": dtype, "act": act}
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # one image: what a request costs when nothing is batched; two channels a group
        _norm("norm_infer", 1, 64, 32, 56, 56, name="norm infer 1n 64c 56x56"),
        # a small ragged batch, image and channel count
        _norm("norm_infer", 3, 72, 9, 49, 33, "bfloat16", "gelu", name="norm infer 3n 72c 49x33 bf16"),
        # first layers of a network on large images, six channels a group: many pixels behind each mean
        _norm("norm_infer", 32, 48, 8, 224, 224, name="norm infer 32n 48c 224x224"),
        # first stage at the benchmark's batch, three channels a group, input kept in 8 bits
        _norm("norm_train", 128, 96, 32, 56, 56, bits=8, name="norm train 128n 96c 56x56 8 bits"),
        # last stage: few pixels, many channels, the norm alone
        _norm("norm_train", 128, 768, 32, 7, 7, act="none", name="norm train 128n 768c 7x7"),
        # second stage on a float32 residual stream
        _norm("norm_train", 32, 192, 24, 28, 28, "float32", name="norm train 32n 192c 28x28 float32"),
        # early layer of an EfficientNet-like network, bfloat16, input kept in 8 bits
        _norm("norm_train", 16, 24, 4, 144, 144, "bfloat16", "gelu", bits=8,
              name="norm train 16n 24c 144x144 bf16 8 bits"),  # fmt: skip
        # GELU of the first stage's MLP at the benchmark's batch: the network's largest activation
        _flat("act_train", 128, 384, 56, 56, name="act train 128n 384c 56x56"),
        # SiLU in the third stage's MLP at a small batch
        _flat("act_train", 32, 1536, 14, 14, "bfloat16", "silu", name="act train 32n 1536c 14x14 bf16"),
        # an odd number of values: no dimension is a multiple of a block
        _flat("act_infer", 3, 197, 17, 5, "float32", name="act infer 3n 197c 17x5 float32"),
        # a convolution's input between its two passes: the benchmark's size, and a small ragged one
        _flat("pack", 128, 64, 56, 56, act="none", name="pack 128n 64c 56x56"),
        _flat("pack", 7, 40, 33, 29, "bfloat16", act="none", name="pack 7n 40c 33x29 bf16"),
    ]


def _log_uniform(rng, low, high):
    return math.exp(rng.uniform(math.log(low), math.log(high)))


def draw(rng):
    sizes = [work(c)["bytes"] for c in listed()]
    while True:
        op = rng.choices(("norm_infer", "norm_train", "act_infer", "act_train", "pack"), weights=(4, 6, 1, 3, 2))[0]
        dtype = rng.choices(("float16", "bfloat16", "float32"), weights=(4, 3, 2))[0]
        n = round(_log_uniform(rng, 1, 128))
        h = round(_log_uniform(rng, 5, 224))
        w = h if rng.random() < 0.5 else round(min(256, max(5, h * _log_uniform(rng, 0.5, 2))))
        if op.startswith("norm"):
            c = 8 * round(_log_uniform(rng, 3, 160))
            groups = rng.choice([g for g in range(1, 65) if c % g == 0])
            case = _norm(op, n, c, groups, h, w, dtype, rng.choice(("none", "silu", "gelu")),
                         8 if op == "norm_train" and rng.random() < 0.5 else 16, rng.random() < 0.85)  # fmt: skip
        else:
            c = round(_log_uniform(rng, 20, 2000))
            c = 8 * -(-c // 8) if rng.random() < 0.7 else c
            act = "none" if op == "pack" else rng.choice(("silu", "gelu"))
            case = _flat(op, n, c, h, w, dtype, act)
        if min(sizes) <= work(case)["bytes"] <= max(sizes):
            return case


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    n, c, h, w = (case[f] for f in "nchw")
    norm = case["op"].startswith("norm")

    def uniform(shape, low, high):
        return torch.empty(shape, device="cuda").uniform_(low, high, generator=gen)

    # activations are stored pixel by pixel; those between a network's linear layers have that as their shape
    shape, vector = ((n, c, h, w), (1, c, 1, 1)) if norm or case["op"] == "pack" else ((n, h, w, c), (c,))

    def normal():
        t = torch.empty((n, h, w, c), device="cuda", dtype=dtype).normal_(generator=gen)
        return t.permute(0, 3, 1, 2) if len(vector) == 4 else t

    # channels differ in scale and offset, as behind a convolution or linear layer with a bias
    x = normal().mul_(uniform(vector, 0.5, 2.0).to(dtype)).add_(uniform(vector, -1.0, 1.0).to(dtype))
    assert x.shape == shape
    state = {"case": case, "x": x, "weight": None, "bias": None}
    if norm and case["affine"]:
        state["weight"], state["bias"] = uniform((c,), 0.5, 1.5), uniform((c,), -0.5, 0.5)
    if case["op"].endswith("train"):
        state["dy"] = normal()
        for key in ("x", "weight", "bias"):
            if state[key] is not None:
                state[key].requires_grad_()
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from spio_amd.functional import activation_8bit, group_norm_2d, pack_8bit, unpack_8bit

    case, x = state["case"], state["x"]
    if case["op"] == "pack":
        return unpack_8bit(pack_8bit(x))
    if case["op"].startswith("norm"):
        y = group_norm_2d(x, case["groups"], state["weight"], state["bias"], eps=EPS, activation=case["act"],
                          checkpoint_8bit=case["bits"] == 8)  # fmt: skip
    else:
        y = activation_8bit(x, case["act"])
    if case["op"].endswith("infer"):
        return y
    wanted = [t for t in (x, state["weight"], state["bias"]) if t is not None]
    return [y.detach(), *torch.autograd.grad(y, wanted, state["dy"])]


# ---- plain form: elementary operations in 32 bits, rounded once at the end ----


def _rounded_blocks(blocks):
    """Blocks of values [..., 32] in 32 bits as their 8-bit codes and power-of-two steps stand for them."""
    largest = blocks.abs().amax(-1, keepdim=True)
    # exponent of the largest value, one more where it would round to 128 steps
    exponent = ((largest.view(torch.int32) + 0x10000) >> 23).clamp(7, 254)
    step = ((exponent - 6) << 23).view(torch.float32)
    inverse = ((260 - exponent) << 23).view(torch.float32)
    return torch.round(blocks * inverse).clamp(-127, 127) * step


def _rounded_rows(rows):
    """The last dimension in blocks of 32, the last block of a row with what is left."""
    length = rows.shape[-1]
    padded = torch.nn.functional.pad(rows, (0, -length % 32))
    blocks = padded.reshape(*padded.shape[:-1], -1, 32)
    return _rounded_blocks(blocks).reshape(padded.shape)[..., :length]


def _activate(z, act):
    """(value, derivative)"""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    cdf = 0.5 * torch.erfc(z * -math.sqrt(0.5))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _run_plain(state):
    with torch.no_grad():
        case = state["case"]
        op, x = case["op"], state["x"]
        dtype = x.dtype
        if op == "pack":
            flat = x.permute(0, 2, 3, 1).float()
            back = _rounded_rows(flat.reshape(-1)).reshape(flat.shape)
            return back.to(dtype).permute(0, 3, 1, 2)
        if op.startswith("act"):
            xf = x.float()
            y = _activate(xf, case["act"])[0].to(dtype)
            if op == "act_infer":
                return y
            kept = _rounded_rows(xf.reshape(-1)).reshape(xf.shape)
            return [y, (state["dy"].float() * _activate(kept, case["act"])[1]).to(dtype)]
        n, c, h, w = x.shape
        groups = case["groups"]
        split = (n, h * w, groups, c // groups)
        xf = x.permute(0, 2, 3, 1).float().reshape(split)
        weight = torch.ones(c, device=x.device) if state["weight"] is None else state["weight"]
        bias = torch.zeros(c, device=x.device) if state["bias"] is None else state["bias"]
        weight, bias = weight.reshape(groups, -1), bias.reshape(groups, -1)
        mean = xf.mean((1, 3), keepdim=True)
        centred = xf - mean
        rstd = torch.rsqrt((centred * centred).mean((1, 3), keepdim=True) + EPS)
        y = _activate(centred * rstd * weight + bias, case["act"])[0]

        def image(t):
            return t.reshape(n, h, w, c).to(dtype).permute(0, 3, 1, 2)

        if op == "norm_infer":
            return image(y)
        if case["bits"] == 8:
            xf = _rounded_rows(xf.reshape(n, h * w, c)).reshape(split)
        xhat = (xf - mean) * rstd
        dz = state["dy"].permute(0, 2, 3, 1).float().reshape(split) * _activate(xhat * weight + bias, case["act"])[1]
        g = dz * weight
        dx = rstd * (g - g.mean((1, 3), keepdim=True) - xhat * (g * xhat).mean((1, 3), keepdim=True))
        out = [image(y), image(dx)]
        if state["weight"] is not None:
            # image by image first: sums over all pixels at once are long for 32 bits
            out += [(dz * xhat).sum(1).sum(0).reshape(c), dz.sum(1).sum(0).reshape(c)]
        return out


# ---- the definition in 64 bits ----


def _exact_kept(x):
    """x [..., blocks of a row] by the definition of the 8-bit form: a block's step is the smallest power of two
    of which its largest magnitude is less than 127.5, and every value the nearest number of steps, ties to even."""
    *lead, length = x.shape
    out = torch.empty_like(x)
    whole = length // 32 * 32
    for part, size in ((slice(0, whole), 32), (slice(whole, length), length - whole)):
        if size == 0 or part.start == part.stop:
            continue
        b = x[..., part].unflatten(-1, (-1, size))
        top = b.abs().amax(-1, keepdim=True)
        _, e = torch.frexp(top / 127.5)  # 127.5 steps are exact in 64 bits, their quotient is not: look again below
        step = ((e.long() + 1023) << 52).view(torch.float64)  # 2**e to the last bit
        step = torch.where(top < 63.75 * step, step / 2, step)
        step = torch.where(top >= 127.5 * step, step * 2, step)
        step = step.clamp_min(2.0**-126)
        out[..., part] = (torch.round(b / step) * step).flatten(-2)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        x = state["x"].double()
        if op == "pack":
            return _exact_kept(x.permute(0, 2, 3, 1).reshape(-1)).reshape(
                case["n"], case["h"], case["w"], case["c"]).permute(0, 3, 1, 2)  # fmt: skip

        def act(z):
            if case["act"] == "silu":
                return z * torch.sigmoid(z)
            if case["act"] == "gelu":
                return z * torch.special.ndtr(z)
            return z

        def slope(z):  # derivative of act
            if case["act"] == "silu":
                s = torch.sigmoid(z)
                return s + z * s * torch.sigmoid(-z)
            if case["act"] == "gelu":
                return torch.special.ndtr(z) + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
            return torch.ones_like(z)

        if op.startswith("act"):
            y = act(x)
            if op == "act_infer":
                return y
            return [y, slope(_exact_kept(x.reshape(-1)).reshape(x.shape)) * state["dy"].double()]
        n, c, groups = case["n"], case["c"], case["groups"]
        grouped = x.unflatten(1, (groups, -1)).flatten(2)  # [n, g, values of the group]
        var, mean = torch.var_mean(grouped, 2, correction=0)
        spread = (var + EPS).sqrt().repeat_interleave(c // groups, 1)[:, :, None, None]
        mean = mean.repeat_interleave(c // groups, 1)[:, :, None, None]
        scale = torch.ones(c, device="cuda") if state["weight"] is None else state["weight"]
        shift = torch.zeros(c, device="cuda") if state["bias"] is None else state["bias"]
        scale, shift = scale.double()[:, None, None], shift.double()[:, None, None]
        y = act((x - mean) / spread * scale + shift)
        if op == "norm_infer":
            return y
        if case["bits"] == 8:
            x = _exact_kept(x.permute(0, 2, 3, 1).contiguous()).permute(0, 3, 1, 2)
        hat = (x - mean) / spread
        dz = state["dy"].double() * slope(hat * scale + shift)

        def share(t):  # of a group's sum that each of its values bears
            s = t.unflatten(1, (groups, -1)).mean((2, 3, 4))
            return s.repeat_interleave(c // groups, 1)[:, :, None, None]

        dx = (dz * scale - share(dz * scale) - hat * share(dz * scale * hat)) / spread
        out = [y, dx]
        if state["weight"] is not None:
            out += [(dz * hat).sum((0, 2, 3)), dz.sum((0, 2, 3))]
        return out


def work(case):
    count = case["n"] * case["c"] * case["h"] * case["w"]
    size = 4 if case["dtype"] == "float32" else 2
    kept = count + -(-count // 32)  # codes and the blocks' exponents
    vectors = 8 * case["c"] if case.get("affine") else 0
    per = {"none": 0, "silu": 6, "gelu": 20}[case["act"]]  # operations of an activation
    if case["op"] == "pack":
        return {"bytes": 2 * size * count + 2 * kept, "flops": 5 * count}
    norm = case["op"].startswith("norm")
    moved, flops = 2 * size * count + vectors, ((8 if norm else 0) + per) * count
    if case["op"].endswith("train"):
        # the backward pass: the input again (or its checkpoint, which was written) and the output's gradient in,
        # the input's and the vectors' gradients out
        packed = case.get("bits", 8) == 8
        moved += 2 * size * count + (2 * kept if packed else size * count) + 2 * vectors
        flops += ((16 if norm else 1) + per + (6 if packed else 0)) * count
    return {"bytes": moved, "flops": flops}
