"""Operators measured on their own: the root-mean-square norm of the head's rows (with the residual's addition, its gradients and
its 8-bit output), and the AdamW update of many tensors at once (states in 32 or in 8 bits) with the global gradient norm it clips by.

`run` computes one pass: in plain torch operations (`own = False`) or through this package (`own = True`).

    norm    h = round(x + residual);  y = h / sqrt(mean(h^2) + eps) * weight, over the last axis
    norm8   y as above, y ~ q * scale: one scale a row, max |y| / 448, q in float8_e4m3fn, rounded to nearest even
    clip    norm = sqrt(sum over all tensors of g^2);  g *= min(1, max_norm / (norm + 1e-6))
    adamw   m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;
            p -= lr (m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps) + weight_decay p)
    adamw8  the same with m and v held between steps as 8-bit floats (float8_e4m3fn and float8_e5m2), one power-of-two scale each
            for 256 consecutive elements of a tensor, rounded stochastically: a value between two neighbours of the format goes to
            the upper one with the probability of its distance from the lower one.  Random bits: 16 a value from the package's
            counter-based stream, element counter = position in the concatenation of the tensors.

The scale of a block with largest magnitude a: 2^(floor(log2 a) - k), twice that where a's mantissa is over 1.75 (k = 8 for m, 15 for
v: the formats' largest values are 1.75 * 2^8 and 1.75 * 2^15); held as its exponent + 127, between 1 and 254.
"""
import math

import torch

own = False

BETA1, BETA2, ADAM_EPS, LR, DECAY = 0.9, 0.999, 1e-8, 1e-4, 1e-2
NORM_EPS = 1e-6
BLOCK = 256
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def vgg16_sizes(classes):
    """Element counts of the trainable tensors of the VGG16 detector (convolutions from conv3_1 on, fc6, fc7, the eight predictor
    heads, the similarity head), weights first and biases behind them."""
    convs = [(256, 128), (256, 256), (256, 256), (512, 256)] + 5 * [(512, 512)]
    linears = [(4096, 25088), (4096, 4096), (4096, 4096), (128, 4096)]
    linears += [(n, 4096) for n in (classes, classes, classes, 4 * classes, classes, 4 * classes, classes, 4 * classes)]
    return [n * k for n, k in linears] + [n * k * 9 for n, k in convs] + [n for n, _ in convs + linears]


def head_sizes(classes):
    """The predictor heads alone: eight weights of `classes` or 4 * `classes` rows of 4096, and their biases."""
    rows = [classes, classes, classes, 4 * classes, classes, 4 * classes, classes, 4 * classes]
    return [n * 4096 for n in rows] + rows


def ragged_sizes(count, total, seed):
    """`count` sizes from one element on, spread over their logarithm, about `total` in all, odd ones among them."""
    import random
    r = random.Random(seed)
    raw = [math.exp(r.uniform(0.0, math.log(max(2.0, 4.0 * total / count)))) for _ in range(count)]
    f = total / sum(raw)
    return [max(1, int(x * f)) for x in raw]


def sizes_of(case):
    if case["tensors"] == "vgg16":
        return vgg16_sizes(case["classes"])
    if case["tensors"] == "head":
        return head_sizes(case["classes"])
    return ragged_sizes(case["count"], case["total"], case["layout"])


def listed():
    return [
        # one row behind its Linear at inference: nothing but latency
        {"name": "norm_one_row", "op": "norm", "rows": 1, "dim": 4096, "dtype": "bf16", "residual": True, "grad": False},
        # the 2000 proposals of one image in fp32 activations, forward and backward of a training step
        {"name": "norm_train_f32", "op": "norm", "rows": 2000, "dim": 4096, "dtype": "f32", "residual": True, "grad": True},
        # eight images' proposals in bf16, forward and backward
        {"name": "norm_train_bf16", "op": "norm", "rows": 16000, "dim": 4096, "dtype": "bf16", "residual": True, "grad": True},
        # an odd number of sampled rows of an odd width: no vector fits the row pitch
        {"name": "norm_train_odd", "op": "norm", "rows": 447, "dim": 1373, "dtype": "f32", "residual": False, "grad": True},
        # the pooled rows (512 x 7 x 7) of one image, stored in 8 bits
        {"name": "norm8_pooled_f32", "op": "norm8", "rows": 2000, "dim": 25088, "dtype": "f32", "residual": False},
        # a handful of head rows in 8 bits behind a residual
        {"name": "norm8_few_bf16", "op": "norm8", "rows": 37, "dim": 4100, "dtype": "bf16", "residual": True},
        # clipping all gradients of the VGG16 detector in place
        {"name": "clip_vgg16", "op": "clip", "tensors": "vgg16", "classes": 21, "grads": "f32"},
        # clipping those of the predictor heads alone
        {"name": "clip_head", "op": "clip", "tensors": "head", "classes": 21, "grads": "f32"},
        # a step over the VGG16 detector in 32-bit states, gradients clipped on the way, bf16 copies kept for the matrix cores
        {"name": "adamw_vgg16", "op": "adamw", "tensors": "vgg16", "classes": 21, "grads": "f32", "clip": True, "copies": True},
        # fine-tuning the predictor heads alone: few small tensors
        {"name": "adamw_head", "op": "adamw", "tensors": "head", "classes": 81, "grads": "bf16", "clip": False, "copies": False},
        # the detector's step with 8-bit states
        {"name": "adamw8_vgg16", "op": "adamw8", "tensors": "vgg16", "classes": 21, "grads": "f32", "clip": False, "copies": True},
        # many tensors of odd sizes packed back to back: no alignment, most of them smaller than a workgroup
        {"name": "adamw8_ragged", "op": "adamw8", "tensors": "ragged", "count": 120, "total": 3000001, "layout": 7, "grads": "bf16",
         "clip": False, "copies": False},
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm", "norm", "norm8", "clip", "adamw", "adamw", "adamw8", "adamw8"])
    if op in ("norm", "norm8"):
        dim = log_int(16, 25088)
        if rng.random() < 0.6:
            dim = max(16, dim // 16 * 16)
        rows = log_int(1, min(16000, 50000000 // dim))
        case = {"op": op, "rows": rows, "dim": dim, "dtype": rng.choice(["f32", "bf16"]), "residual": rng.random() < 0.5}
        if op == "norm":
            case["grad"] = rng.random() < 0.7
        return case
    total = log_int(3000, 100000000)
    case = {"op": op, "tensors": "ragged", "count": log_int(1, min(150, total // 1000)), "total": total, "layout": rng.randrange(1 << 20),
            "grads": rng.choice(["f32", "bf16"])}
    if op != "clip":
        case["clip"] = op == "adamw" and rng.random() < 0.5
        case["copies"] = rng.random() < 0.5
    return case


# ---- inputs ----------------------------------------------------------------------------------------------------------------------


def offsets_of(sizes):
    """Tensors lie in flat buffers as the engine keeps them: those of 1024 elements or more at multiples of 4, small ones (biases)
    back to back."""
    at, pos = [], 0
    for n in sizes:
        if n >= 1024:
            pos = (pos + 3) // 4 * 4
        at.append(pos)
        pos += n
    return at, pos


def views(flat, sizes, at):
    return [flat[o:o + n] for o, n in zip(at, sizes)]


def block_exponents(a, k):
    """Exponent + 127 of the scales of blocks with largest magnitudes a (fp32)."""
    bits = a.view(torch.int32)
    return ((bits >> 23) - k + ((bits & 0x7FFFFF) > 0x600000)).clamp(1, 254)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    if case["op"] in ("norm", "norm8"):
        R, D, dt = case["rows"], case["dim"], DTYPES[case["dtype"]]
        # head activations: rows of different size, some far larger columns
        x = normal(R, D)
        x *= torch.exp(normal(R, 1))
        x *= 1 + 8 * (torch.rand(1, D, generator=g, device="cuda") > 0.995)
        s = {"case": case, "x": x.to(dt), "weight": 1 + 0.1 * normal(D)}
        if case["residual"]:
            s["residual"] = normal(R, D, dtype=dt)
        if case.get("grad"):
            s["dy"] = normal(R, D, dtype=dt, scale=1e-2)
            if case["residual"]:
                s["dh"] = normal(R, D, dtype=dt, scale=1e-2)
                s["residual"].requires_grad_(True)
            s["x"].requires_grad_(True)
            s["weight"].requires_grad_(True)
        return s
    sizes = sizes_of(case)
    at, total = offsets_of(sizes)
    # gradients: each tensor has a size of its own, the values within it vary
    grads = torch.randn(total, generator=g, device="cuda")
    level = torch.exp(2 * torch.randn(len(sizes), generator=g, device="cuda") - 8)
    reach = torch.tensor(at[1:] + [total], device="cuda") - torch.tensor(at, device="cuda")
    grads *= torch.repeat_interleave(level, reach, output_size=total)
    if case["op"] == "clip":
        grads = grads.to(DTYPES[case["grads"]])
        return {"case": case, "flat_g": grads, "grads": views(grads, sizes, at), "max_norm": 0.5 * float(grads.double().norm())}
    noise = torch.randn(total, generator=g, device="cuda")
    m = 0.3 * (noise * grads.abs() + grads)
    v = grads.square() * torch.exp(0.5 * noise)
    del noise
    params = torch.randn(total, generator=g, device="cuda") * 0.02
    s = {"case": case, "sizes": sizes, "at": at, "step": 1000, "seed": seed, "flat_p": params, "p": views(params, sizes, at)}
    grads = grads.to(DTYPES[case["grads"]])
    s["flat_g"], s["g"] = grads, views(grads, sizes, at)
    if case["clip"]:
        s["max_norm"] = 0.5 * float(grads.double().norm())
    if case["op"] == "adamw8":
        starts, blocks = [], 0
        for n in sizes:
            starts.append(blocks)
            blocks += -(-n // BLOCK)
        s["scales"] = torch.empty(blocks, 2, dtype=torch.uint8, device="cuda")
        s["e"] = [s["scales"][b:b - (-n // BLOCK)] for b, n in zip(starts, sizes)]
        s["flat_m"] = torch.empty(total, dtype=torch.float8_e4m3fn, device="cuda")
        s["flat_v"] = torch.empty(total, dtype=torch.float8_e5m2, device="cuda")
        for o, n, e in zip(at, sizes, s["e"]):
            for flat, out, col, k in ((m, s["flat_m"], 0, 8), (v, s["flat_v"], 1, 15)):
                x = torch.nn.functional.pad(flat[o:o + n], (0, -n % BLOCK)).view(-1, BLOCK)
                b = block_exponents(x.abs().amax(1), k)
                e[:, col] = b.to(torch.uint8)
                q = torch.ldexp(x, 127 - b.view(-1, 1)).view(-1)[:n].to(out.dtype)
                out.view(torch.uint8)[o:o + n] = q.view(torch.uint8)
        s["m"] = [s["flat_m"].view(torch.uint8)[o:o + n].view(torch.float8_e4m3fn) for o, n in zip(at, sizes)]
        s["v"] = [s["flat_v"].view(torch.uint8)[o:o + n].view(torch.float8_e5m2) for o, n in zip(at, sizes)]
    else:
        s["flat_m"], s["m"] = m, views(m, sizes, at)
        s["flat_v"], s["v"] = v, views(v, sizes, at)
    if case["copies"]:
        s["flat_copy"] = params.to(torch.bfloat16)
        s["copy"] = views(s["flat_copy"], sizes, at)
    return s


def key_of(seed, step):
    """The two 32-bit keys of a step's random bits."""
    return (seed * 2654435761 + step * 40503) & 0xFFFFFFFF, (seed * 2246822519 + step * 3266489917 + 1) & 0xFFFFFFFF


# ---- the plain forms -------------------------------------------------------------------------------------------------------------


def plain_rows(x, weight, residual):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    f = h.float()
    return h, f * torch.rsqrt(f.square().mean(-1, keepdim=True) + NORM_EPS) * weight


def plain_norm8(x, weight, residual):
    h, y = plain_rows(x, weight, residual)
    scale = (y.abs().amax(-1) / 448).clamp_min(2.0 ** -126)
    return h, (y / scale.unsqueeze(-1)).clamp(-448, 448).to(torch.float8_e4m3fn), scale


def plain_norm_of(grads):
    return torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()


def plain_update(p, m, v, c1, c2):
    """p after the step with new averages m, v and bias corrections c1, c2."""
    return p - LR * (m / c1 / (torch.sqrt(v / c2) + ADAM_EPS) + DECAY * p)


def plain_averages(g, m, v):
    return m * BETA1 + g * (1 - BETA1), v * BETA2 + g * g * (1 - BETA2)


def plain_mix(x):
    x = x ^ (x >> 16)
    x = x * 0x7FEB352D & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = x * 0x846CA68B & 0xFFFFFFFF
    return x ^ (x >> 16)


def plain_bits(first, n, key):
    i = torch.arange(first, first + n, device="cuda")
    h = plain_mix((i & 0xFFFFFFFF) ^ key[0])
    return plain_mix((h + key[1] + (i >> 32)) & 0xFFFFFFFF)


def plain_encode(x, rand, k, bias, mantissa):
    """fp32 values and 16 random bits each -> (codes as uint8, the blocks' exponents): the bits below the format's last mantissa bit
    take a random number's addition and are cut; below the smallest normal number the values are moved up by it first, where the
    format's steps are the same."""
    n = x.numel()
    blocks = torch.nn.functional.pad(x.abs(), (0, -n % BLOCK)).view(-1, BLOCK)
    e = block_exponents(blocks.amax(1), k)
    y = (blocks * ((254 - e) << 23).view(torch.float32).view(-1, 1)).view(-1)[:n]
    low = y < 2.0 ** (1 - bias)
    drop = 23 - mantissa
    z = torch.where(low, y + 2.0 ** (1 - bias), y).view(torch.int32) + ((rand << (drop - 16)) + (1 << (drop - 17))).to(torch.int32)
    code = (z >> drop) - ((127 - bias) << mantissa) - (low.to(torch.int32) << mantissa)
    return (code | (torch.signbit(x).to(torch.int32) << 7)).to(torch.uint8), e.to(torch.uint8)


def plain_decode(q, e):
    scale = (e.to(torch.int32) << 23).view(torch.float32)
    return q.float() * torch.repeat_interleave(scale, BLOCK)[:q.numel()]


def plain_adamw8(p, g, mq, vq, e, first, key, c1, c2):
    m, v = plain_averages(g.float(), plain_decode(mq, e[:, 0]), plain_decode(vq, e[:, 1]))
    p.copy_(plain_update(p, m, v, c1, c2))
    bits = plain_bits(first, p.numel(), key)
    code, em = plain_encode(m, bits & 0xFFFF, 8, 7, 3)
    mq.view(torch.uint8).copy_(code)
    code, ev = plain_encode(v, bits >> 16, 15, 15, 2)
    vq.view(torch.uint8).copy_(code)
    e.copy_(torch.stack([em, ev], 1))


def plain_adamw(p, g, m, v, coef, c1, c2):
    m2, v2 = plain_averages(g.float() if coef is None else g.float() * coef, m, v)
    m.copy_(m2)
    v.copy_(v2)
    p.copy_(plain_update(p, m2, v2, c1, c2))


def run_plain(s):
    case = s["case"]
    if case["op"] == "norm":
        h, y = plain_rows(s["x"], s["weight"], s.get("residual"))
        return with_gradients(s, h, y.to(s["x"].dtype))
    if case["op"] == "norm8":
        h, q, scale = plain_norm8(s["x"], s["weight"], s.get("residual"))
        return {"q": q, "scale": scale, "h": h} if case["residual"] else {"q": q, "scale": scale}
    if case["op"] == "clip":
        norm = plain_norm_of(s["grads"])
        coef = (s["max_norm"] / (norm + 1e-6)).clamp_max(1.0)
        [g.copy_(g.float() * coef.float()) for g in s["grads"]]
        return {"norm": norm.float(), "grads": s["flat_g"]}
    s["step"] += 1
    c1, c2 = 1 - BETA1 ** s["step"], 1 - BETA2 ** s["step"]
    coef = (s["max_norm"] / (plain_norm_of(s["g"]) + 1e-6)).clamp_max(1.0).float() if case["clip"] else None
    if case["op"] == "adamw":
        [plain_adamw(p, g, m, v, coef, c1, c2) for p, g, m, v in zip(s["p"], s["g"], s["m"], s["v"])]
    else:
        firsts = [sum(s["sizes"][:i]) for i in range(len(s["sizes"]))]
        [plain_adamw8(p, g, m, v, e, first, key_of(s["seed"], s["step"]), c1, c2)
         for p, g, m, v, e, first in zip(s["p"], s["g"], s["m"], s["v"], s["e"], firsts)]
    if case["copies"]:
        [c.copy_(p) for c, p in zip(s["copy"], s["p"])]
    return step_outputs(s)


# ---- what both return ------------------------------------------------------------------------------------------------------------


def with_gradients(s, h, y):
    out = {"y": y.detach()}
    if s["case"]["residual"]:
        out["h"] = h.detach()
    if not s["case"]["grad"]:
        return out
    if s["case"]["residual"]:
        out["dx"], out["dresidual"], out["dweight"] = torch.autograd.grad((y, h), (s["x"], s["residual"], s["weight"]), (s["dy"], s["dh"]))
    else:
        out["dx"], out["dweight"] = torch.autograd.grad(y, (s["x"], s["weight"]), s["dy"])
    return out


def step_outputs(s):
    out = {"p": s["flat_p"], "m": s["flat_m"], "v": s["flat_v"]}
    if "scales" in s:
        out["scales"] = s["scales"]
    if "copy" in s:
        out["copy"] = s["flat_copy"]
    return out


# ---- one pass --------------------------------------------------------------------------------------------------------------------


def run_own(s):
    from od_wscl_amd import layers, optim
    case = s["case"]
    if case["op"] == "norm":
        if case["residual"]:
            y, h = layers.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=NORM_EPS)
        else:
            y, h = layers.rms_norm(s["x"], s["weight"], eps=NORM_EPS), None
        return with_gradients(s, h, y)
    if case["op"] == "norm8":
        if case["residual"]:
            q, scale, h = layers.rms_norm_fp8(s["x"], s["weight"], residual=s["residual"], eps=NORM_EPS)
            return {"q": q, "scale": scale, "h": h}
        q, scale = layers.rms_norm_fp8(s["x"], s["weight"], eps=NORM_EPS)
        return {"q": q, "scale": scale}
    if case["op"] == "clip":
        norm = optim.clip_grad_norm_(s["grads"], s["max_norm"])
        return {"norm": norm, "grads": s["flat_g"]}
    s["step"] += 1
    coef = optim.grad_norm(s["g"], max_norm=s["max_norm"])[1] if case["clip"] else None
    more = dict(lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY, grad_scale=coef, copies=s.get("copy"))
    if case["op"] == "adamw":
        optim.adamw_step(s["p"], s["g"], s["m"], s["v"], s["step"], **more)
    else:
        k0, k1 = key_of(s["seed"], s["step"])         # the stream's words; adamw8_step adds 0x9E3779B9 key[0] to the second one
        optim.adamw8_step(s["p"], s["g"], s["m"], s["v"], s["e"], s["step"], (k0, (k1 - 0x9E3779B9 * k0) & 0xFFFFFFFF), hold_v=False, **more)
    return step_outputs(s)


def run(state):
    with torch.set_grad_enabled(bool(state["case"].get("grad"))):
        return run_own(state) if own else run_plain(state)


def work(case):
    """Bytes: each input read once, each output written once.  Operations: a few an element, far below what the bytes cost."""
    if case["op"] in ("norm", "norm8"):
        e = DTYPES[case["dtype"]].itemsize
        n, R, D = case["rows"] * case["dim"], case["rows"], case["dim"]
        res = case["residual"]
        if case["op"] == "norm8":
            return {"bytes": n * (e + (2 * e if res else 0) + 1) + 4 * (R + D), "flops": 6 * n}
        b = n * (2 * e + (2 * e if res else 0)) + 4 * D
        f = 5 * n
        if case["grad"]:                      # reads dy (and dh), writes dx (and dresidual), the weight's gradient
            b += n * (2 * e + (2 * e if res else 0)) + 4 * D
            f += 10 * n
        return {"bytes": b, "flops": f}
    n, e = sum(sizes_of(case)), DTYPES[case["grads"]].itemsize
    if case["op"] == "clip":
        return {"bytes": 2 * n * e, "flops": 3 * n}
    state = 16 if case["op"] == "adamw" else 4 + 4 / BLOCK
    return {"bytes": n * (8 + e + state + (2 if case["copies"] else 0)), "flops": (18 if case["op"] == "adamw" else 50) * n}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------


def exact_round8(x, scale_exp, frac, digits, lowest):
    """x (64 bits) on the grid of an 8-bit float: steps of 2^(e - digits) for x in [2^e, 2^(e+1)), e not under `lowest`; up where
    the distance from the lower neighbour, in steps, is more than 1 - frac."""
    y = torch.ldexp(x.abs(), -scale_exp)
    e = (torch.frexp(y)[1] - 1).clamp_min(lowest)
    steps = torch.ldexp(y, digits - e)
    return torch.copysign(torch.ldexp(torch.floor(steps + frac), e - digits), x)


def exact_scale(x, k):
    """log2 of the block scale of every element."""
    n = x.numel()
    blocks = torch.nn.functional.pad(x.abs(), (0, -n % BLOCK)).view(-1, BLOCK)
    mant, e = torch.frexp(blocks.amax(1))                       # mant in [0.5, 1)
    return (e - 1 - k + (mant > 0.875)).clamp(-126, 127).repeat_interleave(BLOCK)[:n]


def exact_random(first, n, key):
    """The two 16-bit numbers of each element, as fractions of one step at the middle of their interval."""
    u = (torch.arange(n, dtype=torch.int64, device="cuda") + first)
    low, high = u % (1 << 32), u // (1 << 32)

    def scramble(w):
        for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B), (16, 1)):
            w = torch.bitwise_xor(w, w // (1 << shift))
            a, b = w // 65536, w % 65536                        # 32-bit product in two halves
            w = ((a * factor % 65536) * 65536 + b * factor) % (1 << 32)
        return w
    w = scramble((scramble(torch.bitwise_xor(low, torch.full_like(low, key[0]))) + key[1] + high) % (1 << 32))
    return (w % 65536 + 0.5).double() / 65536, (w // 65536 + 0.5).double() / 65536


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("norm", "norm8"):
            x, w = s["x"].double(), s["weight"].double()
            if case["residual"]:
                x = (x + s["residual"].double()).to(s["x"].dtype).double()     # h is an output of x's type
            D = case["dim"]
            r = 1 / torch.sqrt((x * x).sum(1, keepdim=True) / D + NORM_EPS)
            y = x * r * w
            if case["op"] == "norm8":
                scale = y.abs().max(1).values / 448
                z = y / scale[:, None]
                e = (torch.frexp(z)[1] - 1).clamp_min(-6)
                out = {"q": torch.ldexp(torch.round(torch.ldexp(z, 3 - e)), e - 3), "scale": scale}
                return {**out, "h": x} if case["residual"] else out
            out = {"y": y}
            if case["residual"]:
                out["h"] = x
            if case["grad"]:
                dy = s["dy"].double()
                out["dweight"] = (dy * x * r).sum(0)
                wd = dy * w
                out["dx"] = r * (wd - x * r * r * (wd * x).sum(1, keepdim=True) / D)
                if case["residual"]:
                    out["dx"] = out["dx"] + s["dh"].double()
                    out["dresidual"] = out["dx"]
            return out
        if case["op"] == "clip":
            g = s["flat_g"].double()
            sizes = sizes_of(case)
            at, total = offsets_of(sizes)
            norm = torch.sqrt(sum((g[o:o + n] ** 2).sum() for o, n in zip(at, sizes)))
            keep = torch.zeros(total, dtype=torch.bool, device="cuda")
            for o, n in zip(at, sizes):
                keep[o:o + n] = True
            return {"norm": norm, "grads": torch.where(keep, g * torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0), g)}
        t = s["step"] + 1
        coef = 1.0
        if case["clip"]:
            norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in s["g"]))
            coef = min(1.0, s["max_norm"] / (norm + 1e-6))
        out = {"p": s["flat_p"].double(), "m": s["flat_m"].double(), "v": s["flat_v"].double()}
        if "scales" in s:
            out["scales"] = None                               # exponents: whole numbers
        if case["copies"]:
            out["copy"] = s["flat_copy"].double()
        first = 0
        for i, (o, n) in enumerate(zip(s["at"], s["sizes"])):
            p, g = out["p"][o:o + n], s["g"][i].double() * coef
            m, v = out["m"][o:o + n], out["v"][o:o + n]
            if case["op"] == "adamw8":
                e = s["e"][i].long() - 127
                m *= torch.ldexp(torch.ones_like(e[:, 0], dtype=torch.float64), e[:, 0]).repeat_interleave(BLOCK)[:n]
                v *= torch.ldexp(torch.ones_like(e[:, 1], dtype=torch.float64), e[:, 1]).repeat_interleave(BLOCK)[:n]
            m += (g - m) * (1 - BETA1)
            v += (g * g - v) * (1 - BETA2)
            p -= LR * (DECAY * p + (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + ADAM_EPS))
            if case["copies"]:
                out["copy"][o:o + n] = p
            if case["op"] == "adamw8":
                rm, rv = exact_random(first, n, key_of(s["seed"], t))
                m.copy_(exact_round8(m, exact_scale(m, 8), rm, 3, -6))
                v.copy_(exact_round8(v, exact_scale(v, 15), rv, 2, -14))
            first += n
        return out
