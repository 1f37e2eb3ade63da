"""csrc/adamw.hip through optim.adamw_step / adamw8_step / grad_norm / clip_grad_norm_ / AdamW: the update against its formula in 64 bits,
the 8-bit codes bit for bit against their definition."""
import copy
import math

import numpy as np
import pytest
import torch

from oracle import rng_ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
SIZES = [1, 0, 3, 21, 84, 255, 256, 257, 4096, 4097, 12289, 100003]


def _lists(sizes, seed, pt=F32, gt=F32, packed=False, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    off = 0 if not packed else 1
    pos = []
    for n in sizes:
        pos.append(off)
        off += n if packed else (n + 7) // 8 * 8
    out = []
    for dt, s in ((pt, 0.05), (gt, scale)):
        flat = (torch.randn(off + 8, generator=g) * s).to(dt).cuda()
        out.append([flat[o:o + n] for o, n in zip(pos, sizes)])
    return out


def _formula(p, g, m, v, t, lr, wd, b1=0.9, b2=0.999, eps=1e-8):
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p - lr * (m / (1 - b1 ** t) / (np.sqrt(v / (1 - b2 ** t)) + eps) + wd * p), m, v


def _np(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("pt,gt,packed", [(F32, F32, False), (F32, F32, True), (F32, BF16, True), (BF16, BF16, False), (BF16, F32, True)])
def test_steps_against_the_formula(pt, gt, packed):
    """Three steps.  m, v: fp32 factors, two products and a sum: 4 u of their terms a step.  p: lr times a ratio that is off by ~12 u (m, v / 2,
    the root, the division, the bias corrections), and its own rounding (half a step of its type) a step."""
    from od_wscl_amd import optim
    p, g = _lists(SIZES, 1, pt, gt, packed)
    m, v = [torch.zeros(n, device="cuda") for n in SIZES], [torch.zeros(n, device="cuda") for n in SIZES]
    copies = [torch.zeros(n, dtype=BF16, device="cuda") if i % 3 else None for i, n in enumerate(SIZES)]
    lr, wd = [1e-3 * (i + 1) for i in range(len(SIZES))], [0.1 * (i % 3) for i in range(len(SIZES))]
    want = [(_np(a), np.zeros(n), np.zeros(n)) for a, n in zip(p, SIZES)]
    half = U if pt == F32 else 2.0 ** -8
    for t in (1, 2, 3):
        optim.adamw_step(p, g, m, v, t, lr=lr, weight_decay=wd, copies=copies)
        for i, n in enumerate(SIZES):
            want[i] = _formula(want[i][0], _np(g[i]), want[i][1], want[i][2], t, lr[i], wd[i])
            rp, rm, rv = want[i]
            gn = np.abs(_np(g[i]))
            assert (np.abs(_np(m[i]) - rm) <= t * 4 * U * gn + 1e-40).all()
            assert (np.abs(_np(v[i]) - rv) <= t * 4 * U * gn * gn + 1e-40).all()
            # (|update| is at most lr (1 + wd |p|) and a little for gradients of one sign)
            assert (np.abs(_np(p[i]) - rp) <= t * ((half + U) * (np.abs(rp) + 2 * lr[i]) + 16 * U * 2 * lr[i])).all(), (i, n, t)
            if copies[i] is not None:
                assert torch.equal(copies[i], p[i].to(BF16))


def test_nothing_outside_the_tensors_is_written():
    from od_wscl_amd import optim
    n, pad = 1001, 9
    for bits in (32, 8):
        bufs = [torch.full((n + 2 * pad,), 7, dtype=d, device="cuda") for d in
                ((F32, F32, F32, F32, BF16) if bits == 32 else (F32, F32, torch.uint8, torch.uint8, BF16))]
        e = torch.full((4 + 2, 2), 7, dtype=torch.uint8, device="cuda")
        views = [b[pad:pad + n] for b in bufs]
        if bits == 32:
            optim.adamw_step([views[0]], [views[1]], [views[2]], [views[3]], 1, copies=[views[4]])
        else:
            optim.adamw8_step([views[0]], [views[1]], [views[2].view(torch.float8_e4m3fn)], [views[3].view(torch.float8_e5m2)], [e[1:5]], 1, (1, 2),
                              copies=[views[4]])
            assert (e[0] == 7).all() and (e[5] == 7).all() and (e[1:5] != 7).all()
        for b in bufs:
            assert (b[:pad].float() == 7).all() and (b[pad + n:].float() == 7).all()


def test_more_tensors_than_a_launch_takes_and_a_narrow_grid():
    from od_wscl_amd import optim
    sizes = [int(x) for x in np.random.RandomState(0).randint(1, 9000, 101)]
    p, g = _lists(sizes, 2)
    q = [x.clone() for x in p]
    s = [[torch.zeros_like(x) for x in p] for _ in range(4)]
    optim.adamw_step(p, g, s[0], s[1], 1)
    optim.adamw_step(q, g, s[2], s[3], 1, max_workgroups=5)
    for i in range(len(sizes)):
        a = [torch.zeros_like(p[i]) for _ in range(2)]
        one = _lists(sizes, 2)[0][i].clone()
        optim.adamw_step([one], [g[i]], [a[0]], [a[1]], 1)
        assert torch.equal(one, p[i]) and torch.equal(q[i], p[i]) and torch.equal(a[1], s[1][i]) and torch.equal(s[3][i], s[1][i])


# ---- 8-bit states: the definition -------------------------------------------------------------------------------------------------


def _grid(code, bits_mant, bias):
    """Value of an 8-bit float's magnitude code."""
    e, m = code >> bits_mant, code & ((1 << bits_mant) - 1)
    return np.where(e == 0, m * 2.0 ** (1 - bias - bits_mant), (1 + m / 2.0 ** bits_mant) * 2.0 ** (e.astype(float) - bias))


def _oracle8(x, rand16, top, mant, bias, least):
    """fp32 values -> (signed values of the codes, block exponents): exact in float64."""
    n = x.size
    codes = np.arange(1 << 7)
    grid = _grid(codes, mant, bias)
    grid = grid[grid <= 1.75 * 2.0 ** top]
    out, es = np.zeros(n), []
    for b in range(0, n, 256):
        y = np.abs(x[b:b + 256].astype(np.float64))
        a = y.max()
        e = 1
        if a > 0:
            k = math.floor(math.log2(a)) if a >= 2.0 ** -126 else -127
            e = max(1, k + 127 - top + (1 if a > 1.75 * 2.0 ** k else 0))
        es.append(e)
        y = y * 2.0 ** (127 - e)
        lo = np.searchsorted(grid, y, side="right") - 1
        hi = np.minimum(lo + 1, grid.size - 1)
        step = np.where(hi > lo, grid[hi] - grid[lo], 1.0)
        frac = (y - grid[lo]) / step
        up = np.floor(frac + (rand16[b:b + 256] + 0.5) / 65536) >= 1
        near = np.where(up, grid[hi], grid[lo])
        if least:                                    # (v: what is not zero does not become zero)
            near = np.where((x[b:b + 256] != 0) & (near == 0), grid[1], near)
        out[b:b + 256] = np.copysign(near, x[b:b + 256])
    return out, np.array(es)


def _bits(first, n, key):
    i = np.arange(n, dtype=np.uint64) + np.uint64(first)
    h = rng_ref._mix32((i & np.uint64(0xFFFFFFFF)) ^ np.uint64(key[0]))
    return rng_ref._mix32((h + np.uint64((key[1] + 0x9E3779B9 * key[0]) & 0xFFFFFFFF) + (i >> np.uint64(32))) & np.uint64(0xFFFFFFFF)).astype(np.int64)


@pytest.mark.parametrize("gt,packed", [(F32, False), (F32, True), (BF16, True)])
def test_8_bit_codes_are_the_definitions_bit_for_bit(gt, packed):
    from od_wscl_amd import optim
    p, g = _lists(SIZES, 3, F32, gt, packed, scale=1e-3)
    for i, x in enumerate(g):
        x *= torch.exp(3 * torch.randn(x.shape, generator=torch.Generator().manual_seed(i))).to(x)      # a wide range within a block
    g[4].zero_()
    st = [optim.state8_zeros(x) for x in p]
    m, v, e = ([s[k] for s in st] for k in range(3))
    if packed:      # codes that start at odd bytes
        m = [torch.zeros(x.numel() + 3, dtype=torch.uint8, device="cuda")[3:].view(torch.float8_e4m3fn) for x in p]
        v = [torch.zeros(x.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(torch.float8_e5m2) for x in p]
    b1, o1, b2, o2 = (np.float32(x) for x in (0.9, 1 - 0.9, 0.999, 1 - 0.999))
    for t in (1, 2, 3):
        key = (12345 * t, (1 << 32) - 7 * t)
        before = [[_np(x) for x in optim.state8_read(*s)] for s in zip(m, v, e)]
        pw = [_np(x) for x in p]
        optim.adamw8_step(p, g, m, v, e, t, key, lr=1e-2)
        first = 0
        for i, n in enumerate(SIZES):
            if n == 0:
                continue
            gf = g[i].float().cpu().numpy()
            mm = before[i][0].astype(np.float32) * b1 + gf * o1
            vv = before[i][1].astype(np.float32) * b2 + gf * gf * o2
            r = _bits(first, n, key)
            for x, q, col, top, mant, bias, rand in ((mm, m[i], 0, 8, 3, 7, r & 0xFFFF), (vv, v[i], 1, 15, 2, 15, r >> 16)):
                want, es = _oracle8(x, rand, top, mant, bias, col == 1)
                assert np.array_equal(e[i][:, col].cpu().numpy(), es), (t, n, col)
                assert np.array_equal(_np(q.float()), want), (t, n, col)
            rp = _formula(pw[i], gf.astype(np.float64), before[i][0], before[i][1], t, 1e-2, 1e-2)[0]
            assert (np.abs(_np(p[i]) - rp) <= 2 * U * np.abs(rp) + 24 * U * 10 * 1e-2).all()
            first += n


def test_8_bit_extremes():
    """Zero, subnormal and huge averages; non-finite gradients make NaN of their own element and leave the block's others alone."""
    from od_wscl_amd import optim

    def one(gr, n_steps=1):
        p = torch.zeros(gr.numel(), device="cuda")
        s = optim.state8_zeros(p)
        for t in range(n_steps):
            optim.adamw8_step([p], [gr], [s[0]], [s[1]], [s[2]], t + 1, (5, t), lr=1e-3, weight_decay=0.0)
        return p, optim.state8_read(*s), s
    p, (m, v), s = one(torch.zeros(300, device="cuda"))
    assert not p.any() and not m.any() and not v.any() and (s[2] == 1).all()
    gr = torch.full((300,), 1e-19, device="cuda")           # g^2 (1 - b2) = 1e-41: below fp32's normal numbers
    p, (m, v), s = one(gr, 3)
    assert torch.isfinite(p).all() and (m > 0).all()
    gr = torch.full((300,), 1e18, device="cuda")
    p, (m, v), s = one(gr)
    assert torch.isfinite(p).all() and torch.allclose(p, torch.full_like(p, -1e-3), rtol=1e-5)
    assert ((m / 1e17 - 1).abs() < 0.13).all() and ((v / 1e33 - 1).abs() < 0.26).all()
    gr = torch.linspace(0.5, 1.0, 512, device="cuda")
    good = one(gr)[2]
    gr = gr.clone()
    gr[10], gr[300] = float("nan"), float("inf")
    p, (m, v), s = one(gr)
    bad = torch.zeros(512, dtype=torch.bool, device="cuda")
    bad[10] = bad[300] = True
    assert m[bad].isnan().all() and v[bad].isnan().all() and p[10].isnan()
    assert torch.equal(s[0].float()[~bad], good[0].float()[~bad]) and torch.equal(s[1].float()[~bad], good[1].float()[~bad])
    assert torch.equal(s[2], good[2])


def test_state8_read_and_write_give_back_every_code():
    from od_wscl_amd import optim
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    for scale in (1, 100, 127, 200, 240):
        s = torch.full((1, 2), scale, dtype=torch.uint8, device="cuda")
        q = (codes.view(torch.float8_e4m3fn), codes.view(torch.float8_e5m2))
        m, v = optim.state8_read(*q, s)
        back = optim.state8_read(*optim.state8_write(m, v))
        assert torch.equal(torch.nan_to_num(back[0], nan=-1.0), torch.nan_to_num(m, nan=-1.0))
        fin = torch.isfinite(v)
        assert torch.equal(back[1][fin], v[fin]) and back[1][~fin].isnan().all()
        # the step decodes as state8_read does: beta = 0.5 of the held value, gradient 0, exact in fp32; then held again
        p = torch.zeros(256, device="cuda")
        st = [x.clone() for x in optim.state8_write(*(torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0) for x in (m, v.abs())))]
        old = optim.state8_read(*st)
        optim.adamw8_step([p], [torch.zeros_like(p)], [st[0]], [st[1]], [st[2]], 1, (1, 1), betas=(0.5, 0.5), weight_decay=0.0)
        new = optim.state8_read(*st)
        if scale > 100:     # (a power of two keeps the grid: nothing is rounded)
            assert torch.equal(new[0], old[0] / 2) and torch.equal(new[1], old[1] / 2)


def test_small_elements_beside_large_ones_take_bounded_steps():
    """A block whose gradients span 2^-60 .. 1: an element's first average, rounded up to the smallest number now and then, must not meet
    a second average held as zero.  The ratio is at most 3.2 where m is right, and 2^-17 * 3.2 / 2^-16 = 1.6 (in sqrt(v)'s lowest binade; sqrt of
    2 for the scale's) where it was rounded up; bias corrections at most 1 / sqrt(1 - b2^t) > 1 divide it."""
    from od_wscl_amd import optim
    n = 1 << 16
    size = 2.0 ** -(60 * (torch.arange(n, device="cuda") % 256) / 255)
    gen = torch.Generator(device="cuda").manual_seed(4)
    p = torch.zeros(n, device="cuda")
    s = optim.state8_zeros(p)
    for t in range(1, 60):
        old = p.clone()
        optim.adamw8_step([p], [torch.randn(n, generator=gen, device="cuda") * size], [s[0]], [s[1]], [s[2]], t, (t, 1), lr=1.0, weight_decay=0.0, eps=1e-15)
        assert (p - old).abs().max().item() <= 4.0, t


def test_rounding_is_unbiased_and_keys_matter():
    """One value in every element, many random numbers: the mean of the held values is the value, within 6 standard deviations of a
    coin's mean (at most half a grid step each) and the 2^-17 of a step that 16 random bits leave."""
    from od_wscl_amd import optim
    n = 1 << 20
    p = torch.zeros(n, device="cuda")
    for gv in (1.0, 1.03, 0.77, 0.0371):
        gr = torch.full((n,), gv, device="cuda")
        gr[::256] = 1.75                                       # the blocks' scale: all the same
        held = []
        for key in ((1, 2), (1, 2), (3, 4)):
            s = optim.state8_zeros(p)
            optim.adamw8_step([p], [gr], [s[0]], [s[1]], [s[2]], 1, key)
            held.append(optim.state8_read(*s))
        assert torch.equal(held[0][0], held[1][0]) and torch.equal(held[0][1], held[1][1])
        pick = torch.arange(n, device="cuda") % 256 != 0
        for k, (f, rel) in enumerate(((np.float32(1 - 0.9) * np.float32(gv), 0.125), (np.float32(gv) * np.float32(gv) * np.float32(1 - 0.999), 0.25))):
            a, b = (x[k][pick].double() for x in (held[0], held[2]))
            step = rel * float(f)
            assert abs(a.mean().item() / float(f) - 1) <= (6 * 0.5 / math.sqrt(n) + 2.0 ** -16) * rel + 1e-7
            assert (a - float(f)).abs().max().item() <= step
            if a.std().item() > 0:
                assert not torch.equal(a, b)


def test_8_bit_averages_follow_the_32_bit_ones():
    """v moves by a tenth of a percent a step, far below the format's steps: over 3000 steps its mean over the elements stays the
    32-bit one's.  sd of a held v about 0.35 of it (0.5 grid steps of at most 1/4, in all): the mean of 2^16 is good to 6 * 0.35 / 256 = 0.8 %."""
    from od_wscl_amd import optim
    n = 1 << 16
    gen = torch.Generator(device="cuda").manual_seed(3)
    level = torch.exp(torch.randn(n, generator=gen, device="cuda"))
    p8, p32 = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    s8, m, v = optim.state8_zeros(p8), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    for t in range(1, 3001):
        gr = torch.randn(n, generator=gen, device="cuda") * level * (2.0 if t < 800 else 1.0)     # up, then down
        optim.adamw8_step([p8], [gr], [s8[0]], [s8[1]], [s8[2]], t, (t, 17), lr=1e-3)
        optim.adamw_step([p32], [gr], [m], [v], t, lr=1e-3)
    held = optim.state8_read(*s8)[1].double()
    ratio = (held / v.double())
    assert abs(ratio.mean().item() - 1) <= 0.01, ratio.mean().item()
    assert ratio.std().item() <= 0.5
    # the parameters: random walks of the same gradients, with rates that differ by ~15 % an element
    c = torch.corrcoef(torch.stack([p8, p32]))[0, 1].item()
    assert c > 0.95, c


# ---- steps on the device, graphs, streams ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("bits", [32, 8])
def test_device_steps_and_replays(bits):
    from od_wscl_amd import optim
    p0, g = _lists([1000, 37, 5000], 5)

    def fresh():
        p = [x.clone() for x in p0]
        if bits == 8:
            st = [optim.state8_zeros(x) for x in p]
            return p, [[s[k] for s in st] for k in range(3)]
        return p, [[torch.zeros_like(x) for x in p] for _ in range(2)]

    def call(p, st, step, coef, key=(9, 10)):
        if bits == 8:
            optim.adamw8_step(p, g, st[0], st[1], st[2], step, key, grad_scale=coef)
        else:
            optim.adamw_step(p, g, st[0], st[1], step, grad_scale=coef)
    pa, sa = fresh()
    pb, sb = fresh()
    count = torch.zeros(1, dtype=torch.int64, device="cuda")
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        call(*fresh(), torch.zeros(1, dtype=torch.int64, device="cuda"), optim.grad_norm(g, 0.5)[1])
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(pb, sb, count, optim.grad_norm(g, 0.5)[1])
    for t in range(1, 6):
        for x in g:
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(100 * t + x.numel())))
        call(pa, sa, t, optim.grad_norm(g, 0.5)[1], key=(9, 10 + t))        # (the device's step is added to the key)
        graph.replay()
        torch.cuda.synchronize()
        assert int(count) == t
        for a, b in zip(pa, pb):
            # the bias corrections: pow() of the host and of the device, each rounded to fp32
            assert torch.allclose(a, b, rtol=1e-6, atol=1e-8)
        for a, b in zip(sum(sa, []), sum(sb, [])):
            assert torch.equal(a.float(), b.float())


def test_another_stream_and_versions():
    from od_wscl_amd import optim
    p, g = _lists([70001], 6)
    q = [p[0].clone()]
    s = [[torch.zeros_like(p[0])] for _ in range(4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        optim.adamw_step(q, g, s[2], s[3], 1)
    torch.cuda.current_stream().wait_stream(side)
    optim.adamw_step(p, g, s[0], s[1], 1)
    assert torch.equal(p[0], q[0])
    w = torch.ones(8, device="cuda", requires_grad=True)
    y = (w * w).sum()
    optim.adamw_step([w.detach()], [torch.ones(8, device="cuda")], [torch.zeros(8, device="cuda")], [torch.zeros(8, device="cuda")], 1)
    with pytest.raises(RuntimeError):                      # autograd sees that a saved tensor was changed
        y.backward()


# ---- norm and clipping -----------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("gt,packed", [(F32, False), (F32, True), (BF16, True)])
def test_norm_and_clip(gt, packed):
    from od_wscl_amd import optim
    sizes = SIZES + [5] * 60
    g = _lists(sizes, 8, F32, gt, packed)[1]
    want = math.sqrt(sum(float((x.double() ** 2).sum()) for x in g))
    norm = optim.grad_norm(g)
    assert norm.shape == () and norm.dtype == F32 and abs(norm.item() - want) <= 2 * U * want
    norm2, coef = optim.grad_norm(g, max_norm=want / 3)
    assert torch.equal(norm, norm2) and abs(coef.item() - (want / 3) / (want + 1e-6)) <= 2 * U
    assert optim.grad_norm(g, max_norm=2 * want)[1].item() == 1.0
    ref = [x.clone() for x in g]
    assert torch.equal(optim.clip_grad_norm_(g, 2 * want), norm) and all(torch.equal(a, b) for a, b in zip(g, ref))
    assert torch.equal(optim.clip_grad_norm_(g, want / 3), norm)
    for a, b in zip(g, ref):
        assert torch.equal(a, (b.float() * coef).to(gt))
    params = [torch.zeros(4, device="cuda", requires_grad=True) for _ in range(3)]
    params[0].grad, params[2].grad = torch.full((4,), 3.0, device="cuda"), torch.full((4,), 4.0, device="cuda")
    assert optim.clip_grad_norm_(params, 1.0).item() == 10.0 and abs(params[2].grad[0].item() - 0.4) < 1e-6


def test_norm_of_nothing_zeros_and_bad_values():
    from od_wscl_amd import optim
    z = torch.zeros(1000, device="cuda")
    n, c = optim.grad_norm([z, z[:0]], max_norm=1.0)
    assert n.item() == 0.0 and c.item() == 1.0
    assert optim.grad_norm([z[:0]]).item() == 0.0
    z[999] = float("nan")
    n, c = optim.grad_norm([z], max_norm=1.0)
    assert n.isnan() and c.isnan()
    z[999] = float("inf")
    n, c = optim.grad_norm([z], max_norm=1.0)
    assert n.isinf() and c.item() == 0.0
    big = torch.full((4,), 1e30, device="cuda")            # squares past fp32, not past fp64
    assert optim.grad_norm([big]).item() == pytest.approx(2e30, rel=1e-6)
    many = torch.full((1 << 24,), 1e-3, device="cuda")
    assert abs(optim.grad_norm([many]).item() / (float(np.float32(1e-3)) * 4096) - 1) <= 2 * U
    t = torch.randn(64, 48, device="cuda").t()             # a gradient with another order of its elements
    assert abs(optim.grad_norm([t]).item() / t.double().norm().item() - 1) <= 2 * U


# ---- the optimiser object -----------------------------------------------------------------------------------------------------------------


def _params(seed=11):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=g).cuda()) for s in ((30, 40), (40,), (7, 3, 3, 3), ())]


def _loss(ps, x):
    return ((x @ ps[0] + ps[1]).tanh() * ps[3]).square().sum() + ps[2].square().sum()


@pytest.mark.parametrize("clip,capturable", [(None, False), (0.3, False), (0.3, True)])
def test_adamw_object_against_torch(clip, capturable):
    """Twelve steps, gradients taken at the same points: the products' parameters are set to torch's before each backward, so that only
    one step's rounding is compared."""
    from od_wscl_amd import optim
    a, b = _params(), _params()
    groups = lambda ps: [{"params": ps[:2], "lr": 3e-3}, {"params": ps[2:], "weight_decay": 0.1}]     # noqa: E731
    ours, ref = optim.AdamW(groups(a), lr=1e-3, max_grad_norm=clip, capturable=capturable), torch.optim.AdamW(groups(b), lr=1e-3)
    sched = torch.optim.lr_scheduler.StepLR(ours, 5), torch.optim.lr_scheduler.StepLR(ref, 5)
    for it in range(12):
        x = torch.randn(16, 30, device="cuda")
        with torch.no_grad():
            for u, w in zip(a, b):
                u.copy_(w)
        for ps, o in ((a, ours), (b, ref)):
            o.zero_grad()
            _loss(ps, x).backward()
        if it == 4 and not capturable:                       # a parameter without a gradient is passed over
            a[2].grad = b[2].grad = None
        if clip is not None:
            n = torch.nn.utils.clip_grad_norm_([p for p in b if p.grad is not None], clip)
        ours.step()
        ref.step()
        if clip is not None:
            assert abs(ours.grad_norm.item() / n.item() - 1) < 1e-5
        for s in sched:
            s.step()
        for u, w in zip(a, b):
            assert torch.allclose(u, w, rtol=1e-6, atol=2e-8), it
    sd = ours.state_dict()
    assert set(sd["state"][0]) == {"step", "exp_avg", "exp_avg_sq"} and float(sd["state"][0]["step"]) == 12
    assert float(sd["state"][2]["step"]) == (12 if capturable else 11)
    ref.load_state_dict(sd)                                  # torch's reads ours
    again = optim.AdamW(groups(a), lr=1e-3, capturable=capturable)
    again.load_state_dict(ref.state_dict())                  # and ours torch's
    for u, w in zip(a, b):
        u.grad = torch.ones_like(u)
        w.grad = torch.ones_like(w)
        with torch.no_grad():
            u.copy_(w)
    again.step()
    ref.step()
    for u, w in zip(a, b):
        assert torch.allclose(u, w, rtol=1e-6, atol=2e-8)


def test_adamw_object_in_8_bits():
    from od_wscl_amd import optim
    a = _params()
    o = optim.AdamW(a, lr=1e-2, state_bits=8, max_grad_norm=1.0, seed=3)
    for it in range(5):
        o.zero_grad()
        _loss(a, torch.randn(16, 30, device="cuda")).backward()
        o.step()
    st = o.state[a[0]]
    assert st["exp_avg"].dtype == torch.float8_e4m3fn and st["exp_avg_sq"].dtype == torch.float8_e5m2 and st["step"] == 5
    sd = o.state_dict()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    o2 = optim.AdamW(b, lr=1e-2, state_bits=8, max_grad_norm=1.0, seed=3)
    o2.load_state_dict(sd)
    for ps, oo in ((a, o), (b, o2)):
        for it in range(2):
            for k, p in enumerate(ps):
                p.grad = torch.full_like(p, 0.1 * (k + 1 + it))
            oo.step()
    for p, q in zip(a, b):                                   # a resumed run continues bit for bit
        assert torch.equal(p, q)
    o3 = optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in a], state_bits=32)
    o3.load_state_dict(o.state_dict())
    ref = o.state_dict()["state"]
    assert all(torch.equal(o3.state_dict()["state"][i][k], ref[i][k]) for i in ref for k in ("exp_avg", "exp_avg_sq"))


def test_refusals():
    from od_wscl_amd import optim
    p, g = [torch.zeros(8, device="cuda")], [torch.zeros(8, device="cuda")]
    m, v = [torch.zeros(8, device="cuda")], [torch.zeros(8, device="cuda")]
    s = optim.state8_zeros(p[0])
    step8 = lambda **k: optim.adamw8_step(**{**dict(params=p, grads=g, exp_avgs=[s[0]], exp_avg_sqs=[s[1]], scales=[s[2]], step=1, key=(1, 2)), **k})  # noqa: E731
    step = lambda **k: optim.adamw_step(**{**dict(params=p, grads=g, exp_avgs=m, exp_avg_sqs=v, step=1), **k})     # noqa: E731
    wide = torch.zeros(8, 2, device="cuda")
    for bad, error in ((lambda: step(grads=[]), ValueError), (lambda: step(grads=[g[0].half()]), TypeError), (lambda: step(grads=[g[0][:7]]), ValueError),
                       (lambda: step(params=[wide[:, 0]]), ValueError), (lambda: step(exp_avgs=[m[0].bfloat16()]), TypeError),
                       (lambda: step(grads=[g[0].cpu()]), RuntimeError), (lambda: step(step=0), ValueError), (lambda: step(step=1.5), ValueError),
                       (lambda: step(step=torch.zeros(1, device="cuda")), ValueError), (lambda: step(lr=float("nan")), ValueError),
                       (lambda: step(lr=[1e-3, 1e-3]), ValueError), (lambda: step(weight_decay=-1.0), ValueError), (lambda: step(betas=(1.0, 0.9)), ValueError),
                       (lambda: step(eps=0.0), ValueError), (lambda: step(eps=1e-30), ValueError), (lambda: step(copies=[torch.zeros(8, device="cuda")]), TypeError),
                       (lambda: step(copies=[]), ValueError), (lambda: step(grad_scale=torch.ones(2, device="cuda")), ValueError),
                       (lambda: step(max_workgroups=-1), RuntimeError), (lambda: step(grad_mult=float("inf")), ValueError),
                       (lambda: optim.adamw_step(p * 2, g * 2, m * 2, v * 2, 1), ValueError),
                       (lambda: step8(scales=[s[2][:0]]), ValueError), (lambda: step8(exp_avgs=[m[0]]), TypeError), (lambda: step8(key=(1, -1)), ValueError),
                       (lambda: step8(key=(1,)), ValueError), (lambda: optim.grad_norm([]), ValueError), (lambda: optim.grad_norm(g, max_norm=0.0), ValueError),
                       (lambda: optim.clip_grad_norm_(g * 2, 1.0), ValueError), (lambda: optim.clip_grad_norm_([wide[:, 0]], 1.0), ValueError),
                       (lambda: optim.clip_grad_norm_([g[0].half()], 1.0), TypeError), (lambda: optim.AdamW(p, state_bits=4), ValueError),
                       (lambda: optim.AdamW(p, max_grad_norm=0.0), ValueError)):
        with pytest.raises(error):
            bad()
    optim.adamw_step([], [], [], [], 1)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="captured"):
                step()
            m[0].add_(1.0)
        finally:
            graph.capture_end()


def test_a_first_step_is_not_captured_and_later_ones_are():
    from od_wscl_amd import optim
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.ones(1000, device="cuda"))
        ref = torch.nn.Parameter(torch.ones(1000, device="cuda"))
        p.grad, ref.grad = (torch.linspace(-1, 1, 1000, device="cuda") for _ in range(2))
        o, r = (optim.AdamW([x], lr=1e-2, state_bits=bits, max_grad_norm=1.0, capturable=True) for x in (p, ref))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph = torch.cuda.CUDAGraph()
            graph.capture_begin()
            try:
                with pytest.raises(RuntimeError, match="first step"):
                    o.step()
                p.grad.mul_(1.0)
            finally:
                graph.capture_end()
        torch.cuda.current_stream().wait_stream(side)
        assert not o.state_dict()["state"]
        o.step()
        r.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o.step()
        for t in range(4):
            for x in (p, ref):
                x.grad.copy_(torch.randn(1000, generator=torch.Generator().manual_seed(t)))
            graph.replay()
            r.step()
            torch.cuda.synchronize()
            assert torch.equal(p, ref) and float(o.state_dict()["state"][0]["step"]) == t + 2


def test_norm_of_more_tensors_than_a_launch_takes():
    from od_wscl_amd import optim
    sizes = [int(x) for x in np.random.RandomState(1).randint(0, 3000, 401)] + [70000]
    g = _lists(sizes, 12, gt=BF16, packed=True)[1]
    want = math.sqrt(sum(float((x.double() ** 2).sum()) for x in g))
    ref = [x.clone() for x in g]
    norm, coef = optim.grad_norm(g, max_norm=1.0)
    assert abs(norm.item() / want - 1) <= 2 * U
    assert torch.equal(optim.clip_grad_norm_(g, 1.0), norm)
    assert all(torch.equal(a, (b.float() * coef).to(BF16)) for a, b in zip(g, ref))


def test_tensors_made_in_inference_mode():
    from od_wscl_amd import layers, optim
    with torch.inference_mode():
        p, g, m, v = (torch.ones(300, device="cuda") for _ in range(4))
        optim.adamw_step([p], [g], [m], [v], 1, lr=0.5)
        optim.clip_grad_norm_([g], 1.0)
        y, h = layers.rms_norm(p.view(3, 100), g[:100], residual=v.view(3, 100))
    assert (p < 1).all() and abs(g.norm().item() - 1) < 1e-5 and torch.isfinite(y).all()


def test_one_parameter_stands_for_its_gradient():
    from od_wscl_amd import optim
    p = torch.nn.Parameter(torch.full((6, 5), 3.0, device="cuda"))
    p.grad = torch.full((6, 5), 2.0, device="cuda")
    want = math.sqrt(30 * 4.0)                                     # (a sum of small integers: exact; its root rounded once)
    assert float(optim.grad_norm(p)) == torch.tensor(want).item() == float(optim.grad_norm([p]))
    assert float(optim.clip_grad_norm_(p, 1e3)) == torch.tensor(want).item()
    assert torch.equal(p.grad, torch.full_like(p, 2.0)) and torch.equal(p.detach(), torch.full_like(p, 3.0))


def test_numbers_past_fp32_are_refused():
    from od_wscl_amd import layers, optim
    t = [torch.ones(4, device="cuda") for _ in range(4)]
    args = [[x] for x in t]
    for more in (dict(lr=1e39), dict(lr=[1e39]), dict(weight_decay=1e39), dict(eps=1e39), dict(grad_mult=1e39), dict(grad_mult=-1e39)):
        with pytest.raises(ValueError):
            optim.adamw_step(*args, 1, **more)
    for x in t:
        assert torch.equal(x, torch.ones_like(x))
    with pytest.raises(ValueError, match="eps"):
        layers.rms_norm(torch.ones(2, 4, device="cuda"), eps=1e39)


@pytest.mark.parametrize("bits,capturable", [(32, False), (8, False), (8, True)])
def test_a_copied_optimiser_goes_on_alike(bits, capturable):
    from od_wscl_amd import optim
    torch.manual_seed(5)
    mod = torch.nn.Linear(37, 19).cuda()
    opt = optim.AdamW(mod.parameters(), state_bits=bits, capturable=capturable, max_grad_norm=0.5, seed=3)

    def step(m, o, k):
        for i, p in enumerate(m.parameters()):
            p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(10 * k + i)).cuda()
        o.step()
    step(mod, opt, 1)
    twin, topt = copy.deepcopy((mod, opt))
    for k in (2, 3):
        step(mod, opt, k)
        step(twin, topt, k)
    for a, b in zip(mod.parameters(), twin.parameters()):
        assert a is not b and torch.equal(a, b)
