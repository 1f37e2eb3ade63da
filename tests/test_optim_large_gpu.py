"""The update and the norm where element numbers, byte offsets and the random counter pass 32 bits."""
import numpy as np
import pytest
import torch

from test_optim_gpu import BF16, F32, U, _bits, _formula, _np, _oracle8

pytestmark = pytest.mark.gpu


def _tail(n, k, dtype, seed, scale=1.0):
    x = torch.zeros(n, dtype=dtype, device="cuda")
    x[-k:] = (torch.randn(k, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)
    return x


def test_states_in_32_bits():
    from od_wscl_amd import optim
    n, k = (1 << 31) + 777, 1000
    p, g = _tail(n, k, F32, 1, 0.05), _tail(n, k, BF16, 2)
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    p0, g0 = p[-k:].clone(), g[-k:].clone()
    norm, coef = optim.grad_norm([g], 1.0)
    want = g0.double().norm().item()
    assert abs(norm.item() / want - 1) <= 2 * U
    optim.adamw_step([p], [g], [m], [v], 1, lr=1e-3, grad_scale=coef)
    rp, rm, rv = _formula(_np(p0), _np(g0) * coef.double().item(), 0.0, 0.0, 1, 1e-3, 1e-2)
    assert (np.abs(_np(p[-k:]) - rp) <= 2 * U * (np.abs(rp) + 1e-3) + 24 * U * 2e-3).all()
    assert (np.abs(_np(m[-k:]) - rm) <= 6 * U * np.abs(rm) + 1e-40).all() and (np.abs(_np(v[-k:]) - rv) <= 8 * U * rv + 1e-40).all()
    for x in (p, m, v):
        assert not x[:-k].any()
    assert torch.equal(optim.clip_grad_norm_([g], 1.0), norm) and torch.equal(g[-k:], (g0.float() * coef).to(BF16)) and not g[:-k].any()


def test_states_in_8_bits():
    from od_wscl_amd import optim
    n, k = (1 << 32) + 777, 777 + 256                     # the last 777 elements' counters have a high word
    p, g = _tail(n, k, BF16, 3, 0.05), _tail(n, k, BF16, 4)
    m, v, e = optim.state8_zeros(p)
    key = (77, 1 << 31)
    p0, gf = _np(p[-k:]), g[-k:].float().cpu().numpy()
    optim.adamw8_step([p], [g], [m], [v], [e], 1, key, lr=1e-3)
    r = _bits(n - k, k, key)
    o1, o2 = np.float32(1 - 0.9), np.float32(1 - 0.999)
    for x, q, col, top, mant, bias, rand in ((gf * o1, m, 0, 8, 3, 7, r & 0xFFFF), (gf * gf * o2, v, 1, 15, 2, 15, r >> 16)):
        want, es = _oracle8(x, rand, top, mant, bias, col == 1)
        assert np.array_equal(e[-len(es):, col].cpu().numpy(), es) and np.array_equal(_np(q[-k:].float()), want)
        assert not q.view(torch.uint8)[:-k].any() and (e[:-len(es), col] == 1).all()
    rp = _formula(p0, gf.astype(np.float64), 0.0, 0.0, 1, 1e-3, 1e-2)[0]
    assert (np.abs(_np(p[-k:]) - rp) <= (2.0 ** -8 + 2 * U) * (np.abs(rp) + 1e-3) + 24 * U * 2e-3).all() and not p[:-k].any()
