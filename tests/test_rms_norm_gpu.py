"""csrc/rms_norm.hip through layers.rms_norm / rms_norm_fp8 / RMSNorm, against the definition in 64 bits.

Tolerances (u = 2^-24, one rounding of fp32; U = half a step of the output's type): a sum of D terms that W lanes share is off by at most
(D / W + 12) u of the sum of its terms' magnitudes (W = 256 at least), the factors behind it by a few u more."""
import time

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = 1e-6
U32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F32, BF16 = torch.float32, torch.bfloat16


def _sum_ulps(D):
    return (D / 256 + 16) * U32


def _rand(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def _reference(x, w, res):
    """h (in its type, as fp64), rs, y in fp64."""
    h = x.double()
    if res is not None:
        h = (x.double() + res.double()).to(res.dtype).double()
    D = x.shape[-1]
    rs = 1 / torch.sqrt((h * h).sum(-1, keepdim=True) / D + EPS)
    return h, rs, h * rs * (w.double() if w is not None else 1.0)


def _near(got, want, rel, floor=0.0):
    err = (got.double() - want).abs()
    bound = rel * want.abs() + floor + 1e-37
    assert (err <= bound).all(), "off by %.3e of the bound" % (err / bound).max().item()


def _case(R, D, xt, rt, wt, seed=0):
    x = _rand(seed, R, D, dtype=xt) * torch.exp(_rand(seed + 1, R, 1)).to(xt)
    res = _rand(seed + 2, R, D, dtype=rt) if rt is not None else None
    w = (1 + 0.2 * _rand(seed + 3, D)).to(wt) if wt is not None else None
    return x, res, w


SHAPES = [(1, 1), (3, 7), (1, 64), (5, 130), (64, 128), (17, 1373), (33, 512), (1, 4096), (300, 1024), (9, 4104), (4, 8200), (3, 12545),
          (2, 25088), (2, 40000), (2, 65537)]
TYPES = [(F32, None, F32), (F32, F32, F32), (BF16, BF16, F32), (BF16, F32, BF16), (BF16, None, None), (F32, F32, None)]


@pytest.mark.parametrize("R,D", SHAPES)
@pytest.mark.parametrize("xt,rt,wt", TYPES)
def test_forward_and_gradients(R, D, xt, rt, wt):
    from od_wscl_amd import layers
    x, res, w = _case(R, D, xt, rt, wt)
    leaves = [t.requires_grad_(True) for t in (x, res, w) if t is not None]
    out = layers.rms_norm(x, w, residual=res, eps=EPS)
    y, h = out if res is not None else (out, None)
    xd, rd, wd = (t.detach() if t is not None else None for t in (x, res, w))
    rh, rs, ry = _reference(xd, wd, rd)
    assert y.dtype == xt and y.shape == x.shape
    _near(y.detach(), ry, _sum_ulps(D) + HALF[xt])
    if res is not None:
        assert h.dtype == rt
        # the sum of two fp32 or bf16 numbers, rounded once: fp64 rounded to the type is the same number
        assert torch.equal(h.detach().double(), rh)
    dy, dh = _rand(7, R, D, dtype=xt), _rand(8, R, D, dtype=rt) if rt is not None else None
    grads = list(torch.autograd.grad((y, h) if res is not None else y, leaves, (dy, dh) if res is not None else dy))
    # the same without a gradient of h, and nothing but the outputs differs without gradients
    with torch.no_grad():
        out2 = layers.rms_norm(xd, wd, residual=rd, eps=EPS)
    assert torch.equal(out2[0] if res is not None else out2, y)
    g, wf = dy.double(), wd.double() if wd is not None else torch.ones(D, dtype=torch.float64, device="cuda")
    dot = (g * wf * rh).mean(-1, keepdim=True)
    dx = rs * (g * wf - rh * rs * rs * dot)
    size = rs * ((g * wf).abs() + rh.abs() * rs * rs * (g * wf * rh).abs().mean(-1, keepdim=True))
    if dh is not None:
        dx, size = dx + dh.double(), size + dh.double().abs()
    slack = 3 * _sum_ulps(D) * size
    _near(grads[0], dx, HALF[xt], slack)
    if res is not None:
        _near(grads[1], dx, HALF[rt], slack)
    if w is not None:
        dw, dsize = (g * rh * rs).sum(0), (g * rh * rs).abs().sum(0)
        _near(grads[-1], dw, HALF[wt], ((R + 16) * U32 + _sum_ulps(D)) * dsize)


@pytest.mark.parametrize("xt", [F32, BF16])
def test_row_pitch_order_and_batch_axes(xt):
    from od_wscl_amd import layers
    base, w = _rand(1, 40, 100, dtype=xt), 1 + _rand(2, 64)
    for x in (base[:, :64], base[:, 3:67], base[::3, 4:68], base.t()[:64].t()[:7], base[:1, :64].expand(9, 64), base[:, 36:].reshape(5, 8, 64),
              base.t()[:, :64]):
        out = layers.rms_norm(x, w[: x.shape[-1]], eps=EPS)
        assert out.shape == x.shape and torch.equal(out, layers.rms_norm(x.contiguous(), w[: x.shape[-1]], eps=EPS))
        _near(out, _reference(x, w[: x.shape[-1]], None)[2], _sum_ulps(64) + HALF[xt])
    x = base[:, 1:65].detach().requires_grad_(True)                     # rows that start off the vectors' alignment
    layers.rms_norm(x, w, eps=EPS).backward(base[:1, :64].expand(40, 64))       # a gradient whose rows are one row
    x2 = x.detach().clone().requires_grad_(True)
    layers.rms_norm(x2, w, eps=EPS).backward(base[:1, :64].expand(40, 64).contiguous())
    assert torch.equal(x.grad, x2.grad)


def test_no_rows_and_partial_use():
    from od_wscl_amd import layers
    x, w = torch.zeros(0, 37, device="cuda", requires_grad=True), torch.ones(37, device="cuda", requires_grad=True)
    y, h = layers.rms_norm(x, w, residual=x)
    (y.sum() + h.sum()).backward()
    assert y.shape == (0, 37) and torch.equal(w.grad, torch.zeros_like(w))
    q, s = layers.rms_norm_fp8(x.detach(), w.detach())
    assert q.shape == (0, 37) and s.shape == (0,)
    x, r = _rand(1, 6, 50).requires_grad_(True), _rand(2, 6, 50).requires_grad_(True)
    w = torch.ones(50, device="cuda", requires_grad=True)
    y, h = layers.rms_norm(x, w, residual=r)
    gx, gr, gw = torch.autograd.grad(h, (x, r, w), h.detach())          # y unused
    assert torch.equal(gx, h) and torch.equal(gr, h) and not gw.any()
    y, h = layers.rms_norm(x, w, residual=r)
    gx, = torch.autograd.grad(y, x, h.detach())                        # h unused, only x asked for
    y2, h2 = layers.rms_norm(x, w, residual=r)
    gr, gw = torch.autograd.grad(y2, (r, w), h.detach())
    assert torch.equal(gx, gr)
    s = _rand(3, 6, 50).requires_grad_(True)                           # one tensor in both places
    y, h = layers.rms_norm(s, w, residual=s)
    g, = torch.autograd.grad((y, h), s, (y.detach(), h.detach()))
    d = (2 * s.detach()).requires_grad_(True)
    g2, = torch.autograd.grad(layers.rms_norm(d, w), d, y.detach())
    assert torch.allclose(g, 2 * (g2 + h.detach()), rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("D", [64, 1373, 4096, 40000])
def test_bad_rows_stay_where_they_are(D):
    from od_wscl_amd import layers
    x = _rand(4, 8, D)
    good = layers.rms_norm(x, eps=EPS)
    qg, sg = layers.rms_norm_fp8(x, eps=EPS)
    x[2, D // 2], x[5, 0], x[6] = float("nan"), float("inf"), 0.0
    y = layers.rms_norm(x, eps=EPS)
    q, s = layers.rms_norm_fp8(x, eps=EPS)
    keep = [0, 1, 3, 4, 7]
    assert torch.equal(y[keep], good[keep]) and torch.equal(q[keep].float(), qg[keep].float()) and torch.equal(s[keep], sg[keep])
    assert y[2].isnan().all() and q[2].float().isnan().all() and s[2].isnan()
    assert y[5, 0].isnan() and not y[5, 1:].any()                      # inf * 0, and number * 0
    assert s[5].isnan() and q[5].float().isnan().all()
    assert not y[6].any() and not q[6].float().any() and s[6].item() == 2.0 ** -126


@pytest.mark.parametrize("R,D", SHAPES)
@pytest.mark.parametrize("xt,rt", [(F32, None), (F32, F32), (BF16, BF16), (BF16, F32)])
def test_8_bit_output(R, D, xt, rt):
    from od_wscl_amd import layers
    x, res, w = _case(R, D, xt, rt, F32, seed=20)
    out = layers.rms_norm_fp8(x, w, residual=res, eps=EPS)
    q, scale = out[0], out[1]
    rh, _, ry = _reference(x, w, res)
    if res is not None:
        assert torch.equal(out[2].double(), rh)
    top = ry.abs().amax(1)
    _near(scale, top / 448, _sum_ulps(D) + 4 * U32)
    z = ry / scale.double()[:, None]
    # half a step of the format: 2^-4 of the value, 2^-10 below the normal numbers; z itself is off by a few u
    _near(q.float(), z, 2.0 ** -4 + _sum_ulps(D) + 4 * U32, 2.0 ** -10)
    step = torch.ldexp(torch.ones_like(z), (torch.frexp(z)[1] - 1).clamp_min(-6) - 3)
    assert ((q.double() - z).abs() <= step * (0.5 + 16 * (_sum_ulps(D) + 4 * U32))).all()
    if D > 1:
        assert (q.float().abs().amax(1) == 448).all()


def test_gradients_against_differences():
    """Directional derivatives of the kernel's own forward in fp32: step t = 2^-6, error t^2 times the third derivative (inputs of size 1:
    below 20 on 8 x 96 values) over 6, and the forward's rounding, 96 * 8 * 2^-22, over 2 t."""
    from od_wscl_amd import layers
    x, r, w = _rand(31, 8, 96), _rand(32, 8, 96), 1 + 0.2 * _rand(33, 96)
    dy, dh = _rand(34, 8, 96), _rand(35, 8, 96)

    def f(a, b, c):
        y, h = layers.rms_norm(a, c, residual=b, eps=EPS)
        return ((y.double() * dy.double()).sum() + (h.double() * dh.double()).sum()).item()
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    y, h = layers.rms_norm(leaves[0], leaves[2], residual=leaves[1], eps=EPS)
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))
    t = 2.0 ** -6
    for k in range(3):
        for s in range(3):
            d = _rand(40 + 3 * k + s, *(x, r, w)[k].shape)
            d /= d.norm()
            plus, minus = [[u + sign * t * d if i == k else u for i, u in enumerate((x, r, w))] for sign in (1, -1)]
            want = (grads[k].double() * d.double()).sum().item()
            assert abs((f(*plus) - f(*minus)) / (2 * t) - want) <= 20 * t * t / 6 + 96 * 8 * 2.0 ** -22 / (2 * t)


def test_same_bits_every_time_and_on_another_stream():
    from od_wscl_amd import layers
    x, r, w = _case(3001, 640, F32, F32, F32, seed=50)
    dy = _rand(51, 3001, 640)

    def once():
        ls = [t.detach().clone().requires_grad_(True) for t in (x, r, w)]
        y, h = layers.rms_norm(ls[0], ls[2], residual=ls[1])
        return (y, h) + torch.autograd.grad((y, h), ls, (dy, dy)) + layers.rms_norm_fp8(x, w, residual=r)
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a.float(), b.float())


def test_captured_and_replayed():
    from od_wscl_amd import layers
    x, r, w = _case(130, 1000, BF16, BF16, F32, seed=60)
    dy = _rand(61, 130, 1000, dtype=BF16)

    def work(a, b):
        a, b, c = a.detach().requires_grad_(True), b.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y, h = layers.rms_norm(a, c, residual=b)
        return (y.detach(), h.detach()) + torch.autograd.grad((y, h), (a, b, c), (dy, dy)) + layers.rms_norm_fp8(a.detach(), w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(x, r)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                  # two graphs, each with workspaces of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work(x, r)
        graphs.append((graph, out))
    for k in range(4):
        x.copy_(_rand(70 + k, 130, 1000, dtype=BF16))
        want = work(x, r)
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a.float(), b.float())


def test_offsets_past_32_bits():
    from od_wscl_amd import layers
    R, D = 140001, 16384                                # 2.3e9 elements
    x = torch.zeros(R, D, dtype=BF16, device="cuda")
    x[-3:] = _rand(80, 3, D, dtype=BF16)
    y = layers.rms_norm(x, eps=EPS)
    _near(y[-3:], _reference(x[-3:], None, None)[2], _sum_ulps(D) + HALF[BF16])
    assert not y[:2].any() and not y[70000].any()
    q, s = layers.rms_norm_fp8(x, eps=EPS)
    assert (q[-3:].float().abs().amax(1) == 448).all() and not q[R // 2].float().any()
    dx = torch.autograd.grad(layers.rms_norm(x.requires_grad_(True), eps=EPS), x, y)[0]
    small = x[-3:].detach().requires_grad_(True)
    assert torch.equal(dx[-3:], torch.autograd.grad(layers.rms_norm(small, eps=EPS), small, y[-3:])[0])


def test_module_and_refusals():
    from od_wscl_amd import layers
    m = layers.RMSNorm(48).cuda()
    x = _rand(90, 5, 48)
    assert torch.equal(m(x), layers.rms_norm(x, m.weight)) and list(m.state_dict()) == ["weight"]
    y, h = m(x, x)
    assert torch.equal(h, x + x)
    assert layers.RMSNorm(48, elementwise_affine=False).weight is None
    w = torch.ones(48, device="cuda")
    for bad, error in ((lambda: m(x[:, :47]), ValueError), (lambda: layers.rms_norm(x, w[:47]), ValueError),
                       (lambda: layers.rms_norm(x.half(), w), TypeError), (lambda: layers.rms_norm(x, w.half()), TypeError),
                       (lambda: layers.rms_norm(x, w, residual=x[:4]), ValueError),
                       (lambda: layers.rms_norm(x, w, residual=x.bfloat16()), TypeError),
                       (lambda: layers.rms_norm(x, w, eps=-1.0), ValueError), (lambda: layers.rms_norm(x, w, eps=float("nan")), ValueError),
                       (lambda: layers.rms_norm(x[:, :0], w[:0]), ValueError), (lambda: layers.rms_norm(x, w.cpu()), RuntimeError),
                       (lambda: layers.rms_norm_fp8(x.double(), w), TypeError)):
        with pytest.raises(error):
            bad()


def test_a_second_derivative_is_refused():
    from od_wscl_amd import layers
    x, w = _rand(95, 6, 40).requires_grad_(True), torch.ones(40, device="cuda", requires_grad=True)
    y = layers.rms_norm(x, w)
    first, = torch.autograd.grad(y.square().sum(), x, retain_graph=True)
    gx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    assert torch.equal(gx, first)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), x)


def test_more_rows_than_a_launch_takes():
    from od_wscl_amd import layers
    R = (1 << 23) + 5                                   # (2^21 workgroups of four rows)
    x, r, w = _rand(96, R, 3), _rand(97, R, 3), 1 + _rand(98, 3)
    y, h = layers.rms_norm(x, w, residual=r, eps=EPS)
    q, s, h2 = layers.rms_norm_fp8(x, w, residual=r, eps=EPS)
    rh, _, ry = _reference(x, w, r)
    assert torch.equal(h.double(), rh) and torch.equal(h2, h)
    _near(y, ry, _sum_ulps(3) + HALF[F32])
    _near(s, ry.abs().amax(1) / 448, _sum_ulps(3) + 4 * U32)
    assert (q.float().abs().amax(1) == 448).all()
    xs, ws = x.requires_grad_(True), w.requires_grad_(True)
    dx, dw = torch.autograd.grad(layers.rms_norm(xs, ws, residual=r, eps=EPS)[0], (xs, ws), r)
    tail = x.detach()[-7:].requires_grad_(True)
    assert torch.equal(torch.autograd.grad(layers.rms_norm(tail, w, residual=r[-7:], eps=EPS)[0], tail, r[-7:])[0], dx[-7:])
    rs = 1 / torch.sqrt((rh * rh).mean(-1, keepdim=True) + EPS)
    # (2048 groups of 4097 rows each and 2048 partial sums: all in fp32)
    assert ((dw.double() - (r.double() * rh * rs).sum(0)).abs() <= (4097 + 2048 + 16) * U32 * (r.double() * rh * rs).abs().sum(0)).all()


@pytest.mark.parametrize("R,D", [s for s in SHAPES if s[1] <= 32768] + [(2000, 4100), (300, 25088)])
@pytest.mark.parametrize("xt,wt", [(F32, F32), (BF16, F32), (F32, None), (BF16, BF16)])
def test_8_bit_codes_are_the_correctly_rounded_ones(R, D, xt, wt):
    """rne(448 t / max |t|), t = h w: the products and their quotient in fp64 (off by 2^-52: an element would have to lie that near to the
    middle of two codes, and one that lies on it goes to the even code on both sides)."""
    from od_wscl_amd import layers
    x, res, w = _case(R, D, xt, xt, wt, seed=120)
    q, _, h = layers.rms_norm_fp8(x, w, residual=res, eps=EPS)
    t = h.double().cpu().numpy() * (w.double().cpu().numpy() if w is not None else 1.0)
    z = 448 * t / np.abs(t).max(1, keepdims=True)
    e = np.maximum(np.frexp(z)[1] - 1, -6)
    want = np.ldexp(np.rint(np.ldexp(z, 3 - e)), e - 3)          # (torch.ldexp and ** go through pow on the GPU: off by an ulp)
    assert np.array_equal(q.float().cpu().numpy(), want)


def test_8_bit_rows_of_any_size():
    """Rows scaled by powers of two from 2^-140 to 2^50 hold the same codes wherever fp32 can form them: the scale takes the factor (eps is in
    its way below 2^-10, so the row's factor there is 1 / sqrt(eps), and 2^-126 is the smallest scale)."""
    from od_wscl_amd import layers
    base = _rand(130, 1, 1000)
    q0, s0 = layers.rms_norm_fp8(base, eps=EPS)
    for k in (-140, -120, -100, -60, -20, -8, 8, 30, 50):
        x = base * 2.0 ** k if k > -100 else base * 2.0 ** -100 * 2.0 ** (k + 100)
        q, s = layers.rms_norm_fp8(x, eps=EPS)
        y = _reference(x, None, None)[2]
        assert s.item() >= 2.0 ** -126 and torch.isfinite(q.float()).all()
        assert ((q.double() * s.double() - y).abs() <= y.abs() * (2.0 ** -4 + 2.0 ** -20) + s.double() * 2.0 ** -10 + 2.0 ** -149).all(), k
        if -100 <= k:
            assert torch.equal(q.float(), q0.float()), k


def test_nothing_is_held_once_its_graph_is_gone():
    from od_wscl_amd import layers
    x, r, w = _rand(140, 64, 1000).requires_grad_(True), _rand(141, 64, 1000).requires_grad_(True), torch.ones(1000, device="cuda", requires_grad=True)

    def once(back):
        y, h = layers.rms_norm(x, w, residual=r)
        if back:
            torch.autograd.grad((y, h), (x, r, w), (y.detach(), h.detach()))
    once(True)
    torch.cuda.synchronize()
    time.sleep(0.1)
    before = torch.cuda.memory_allocated()
    for k in range(20):
        once(k % 2 == 0)
    # autograd's own thread lets go of the last gradients (260096 bytes: dx and dw) a moment after grad() has returned them
    for _ in range(100):
        if torch.cuda.memory_allocated() == before:
            break
        time.sleep(0.01)
    assert torch.cuda.memory_allocated() == before
    y, h = layers.rms_norm(x, w, residual=r)
    h.data.add_(0.0)                                     # (behind autograd's back)
    with torch.no_grad():
        h.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
