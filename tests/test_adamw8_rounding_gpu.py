"""The 8-bit states' rounding with the stream of utils/rng.py under the caller's own two words, with and without the smallest second average
(optim.adamw8_step, hold_v), bit for bit against its definition: more tensors than a launch takes, fp32 and bf16 parameters among them."""
import numpy as np
import pytest
import torch

from test_optim_gpu import BF16, F32, U, _formula, _np, _oracle8

from od_wscl_amd.utils import rng

pytestmark = pytest.mark.gpu


def stream_words(key):
    """The key that makes adamw8_step draw from the stream with the words `key` (it adds 0x9E3779B9 key[0] to the second one)."""
    return key[0], (key[1] - 0x9E3779B9 * key[0]) & 0xFFFFFFFF


@pytest.mark.parametrize("hold_v", [False, True])
@pytest.mark.parametrize("gt", [F32, BF16])
def test_codes_over_two_launches(hold_v, gt):
    """Codes and scales equal; p: half a step of its type, and 24 u of lr times the ratio (as in test_optim_gpu), which is far over 1 where a
    held second average is zero."""
    from od_wscl_amd import optim
    sizes = [int(x) for x in np.random.RandomState(3).randint(1, 1500, 70)] + [9001, 1]
    gen = torch.Generator().manual_seed(9)
    p = [(torch.randn(n, generator=gen) * 0.05).to(BF16 if i % 3 == 1 else F32).cuda() for i, n in enumerate(sizes)]
    g = [(torch.randn(n, generator=gen) * torch.exp2(-30 * torch.rand(n, generator=gen))).to(gt).cuda() for n in sizes]
    st = [optim.state8_zeros(x) for x in p]
    m, v, e = ([s[k] for s in st] for k in range(3))
    b1, o1, b2, o2 = (np.float32(x) for x in (0.9, 1 - 0.9, 0.999, 1 - 0.999))
    zeros = 0
    for t in (1, 2, 3):
        before, pw = [[_np(x) for x in optim.state8_read(*s)] for s in st], [_np(x) for x in p]
        optim.adamw8_step(p, g, m, v, e, t, stream_words(rng.stream_key(5, t)), lr=1e-3, hold_v=hold_v)
        drawn = rng.bits(5, t, sum(sizes)).astype(np.int64)
        first = 0
        for i, n in enumerate(sizes):
            gf, r = g[i].float().cpu().numpy(), drawn[first:first + n]
            mm = before[i][0].astype(np.float32) * b1 + gf * o1
            vv = before[i][1].astype(np.float32) * b2 + gf * gf * o2
            for x, q, col, top, mant, bias, rand in ((mm, m[i], 0, 8, 3, 7, r & 0xFFFF), (vv, v[i], 1, 15, 2, 15, r >> 16)):
                want, es = _oracle8(x, rand, top, mant, bias, col == 1 and hold_v)
                assert np.array_equal(e[i][:, col].cpu().numpy(), es), (t, i, col)
                assert np.array_equal(_np(q.float()), want), (t, i, col)
                zeros += int(((want == 0) & (x != 0)).sum()) if col == 1 else 0
            rp, rm, rv = _formula(pw[i], gf.astype(np.float64), before[i][0], before[i][1], t, 1e-3, 1e-2)
            ratio = np.abs(rm) / (1 - 0.9 ** t) / (np.sqrt(rv / (1 - 0.999 ** t)) + 1e-8)
            half = 2.0 ** -8 if p[i].dtype == BF16 else U
            assert (np.abs(_np(p[i]) - rp) <= (half + 2 * U) * (np.abs(rp) + 1e-3 * ratio) + 24 * U * 1e-3 * (1 + ratio)).all(), (t, i)
            first += n
    assert (zeros > 0) == (not hold_v)
