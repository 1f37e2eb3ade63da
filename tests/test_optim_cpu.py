"""Argument checks of the optimiser's and the row norm's entry points that end before any launch, and the 8-bit states' layout, without a GPU."""
import copy
import ctypes
import math
import pickle

import pytest
import torch

from od_wscl_amd import _lib, layers, optim


def _arr(ctype, *values):
    return (ctype * len(values))(*values)


def test_cpu_tensors_are_refused():
    p = [torch.zeros(4)]
    s = optim.state8_zeros(p[0])
    for call in (lambda: optim.adamw_step(p, p, p, p, 1), lambda: optim.adamw8_step(p, p, [s[0]], [s[1]], [s[2]], 1, (0, 0)),
                 lambda: optim.grad_norm(p), lambda: optim.clip_grad_norm_(p, 1.0), lambda: layers.rms_norm(torch.zeros(2, 4)),
                 lambda: layers.rms_norm_fp8(torch.zeros(2, 4)), lambda: layers.RMSNorm(4)(torch.zeros(2, 4))):
        with pytest.raises(RuntimeError, match="not on the GPU"):
            call()
    q = torch.nn.Parameter(torch.zeros(4))
    q.grad = torch.zeros(4)
    for bits in (8, 32):
        with pytest.raises(RuntimeError, match="not on the GPU"):
            optim.AdamW([q], state_bits=bits).step()
    assert optim.AdamW([torch.nn.Parameter(torch.zeros(4))]).step() is None        # no gradients: nothing to do
    optim.adamw_step([], [], [], [], 1)


def test_optimiser_arguments():
    p = [torch.nn.Parameter(torch.zeros(4))]
    for bad in (dict(state_bits=16), dict(max_grad_norm=-1.0), dict(lr=-1.0), dict(lr=math.nan), dict(weight_decay=-0.1), dict(betas=(0.9,)),
                dict(betas=(0.9, 1.0)), dict(eps=0.0), dict(eps=math.inf)):
        with pytest.raises(ValueError):
            optim.AdamW(p, **bad)


def _with_a_state(**more):
    p = torch.nn.Parameter(torch.arange(6.0))
    opt = optim.AdamW([p], lr=2e-3, **more)
    src = torch.optim.AdamW([p], lr=3e-3, weight_decay=0.1)
    p.grad = torch.linspace(-1.0, 1.0, 6)
    src.step()
    opt.load_state_dict(src.state_dict())
    return opt


@pytest.mark.parametrize("way", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))], ids=["copy", "pickle"])
@pytest.mark.parametrize("bits", [8, 32])
def test_a_copied_optimiser_is_whole(way, bits):
    opt = _with_a_state(state_bits=bits, max_grad_norm=2.0, seed=7)
    got = way(opt)
    assert (got.state_bits, got.max_grad_norm, got.seed, got.capturable, got.grad_norm) == (bits, 2.0, 7, False, None)
    a, b = opt.state_dict(), got.state_dict()
    assert a["param_groups"] == b["param_groups"] and a["state"].keys() == b["state"].keys()
    for i in a["state"]:
        for k in ("step", "exp_avg", "exp_avg_sq"):
            assert torch.equal(a["state"][i][k], b["state"][i][k])
    with pytest.raises(RuntimeError, match="not on the GPU"):
        got.param_groups[0]["params"][0].grad = torch.ones(6)
        got.step()


def test_states_of_another_rule_are_refused():
    p = torch.nn.Parameter(torch.zeros(4))
    opt = optim.AdamW([p])
    for other in (torch.optim.AdamW([p], amsgrad=True), torch.optim.AdamW([p], maximize=True), torch.optim.Adam([p], weight_decay=0.1)):
        with pytest.raises(ValueError, match="amsgrad|maximize|coupled"):
            opt.load_state_dict(other.state_dict())
    opt.load_state_dict(torch.optim.AdamW([p]).state_dict())


def test_library_checks_come_before_launches():
    lib = _lib.lib()
    n, types, one = _arr(ctypes.c_int64, 8), _arr(ctypes.c_int, 0), _arr(ctypes.c_float, 1e-3)
    null, some, odd = _arr(ctypes.c_void_p, None), _arr(ctypes.c_void_p, 4096), _arr(ctypes.c_void_p, 4097)

    def adamw(p=some, g=some, m=some, v=some, n=n, types=types, b1=0.9, eps=1e-8, step=1, wg=0, count=1):
        return lib.odw_adamw(count, p, g, m, v, None, n, types, one, one, b1, 0.999, eps, step, None, None, 1.0, wg, None)
    assert adamw(count=0) == 0 and adamw(n=_arr(ctypes.c_int64, 0)) == 0            # nothing to do: nothing is launched
    for bad in (dict(p=null), dict(g=null), dict(m=null), dict(v=null), dict(p=odd), dict(g=odd), dict(m=odd), dict(p=None), dict(types=None),
                dict(n=_arr(ctypes.c_int64, -1)), dict(n=_arr(ctypes.c_int64, 1 << 41)), dict(types=_arr(ctypes.c_int, 4)), dict(b1=1.0), dict(b1=math.nan),
                dict(eps=0.0), dict(eps=math.nan), dict(step=0), dict(wg=-1), dict(count=-1)):
        assert adamw(**bad) == -1 and b"adamw" in lib.odw_last_error(), bad
    assert lib.odw_adamw8(1, some, some, some, some, null, None, n, types, one, one, 0.9, 0.999, 1e-8, 1, None, None, 1.0, 0, 0, 0, None) == -1
    assert lib.odw_adamw_advance(None, 0.9, 0.999, None, None) == -1
    need = lib.odw_grad_norm_workspace(1, n)
    assert 0 < need <= 64
    assert lib.odw_grad_norm(1, some, n, types, 1.0, some, None, 0, None) == -3 and b"workspace" in lib.odw_last_error()
    assert lib.odw_grad_norm(1, some, n, types, 0.0, some, some, need, None) == -1
    assert lib.odw_grad_norm(1, some, n, types, math.nan, some, some, need, None) == -1
    assert lib.odw_grad_norm(1, null, n, types, 1.0, some, some, need, None) == -1
    assert lib.odw_grad_norm(1, some, n, types, 1.0, None, some, need, None) == -1
    assert lib.odw_scale_tensors(1, some, n, types, None, None) == -1
    assert lib.odw_rms_norm(None, 4, None, 0, None, 2, 4, 1e-6, None, None, None, 0, None) == -1 and b"rms_norm" in lib.odw_last_error()
    assert lib.odw_rms_norm(None, 4, None, 0, None, 0, 4, 1e-6, None, None, None, 0, None) == 0
    assert lib.odw_rms_norm(4096, 4, None, 0, None, -1, 4, 1e-6, 4096, None, None, 0, None) == -1
    assert lib.odw_rms_norm(4096, 4, None, 0, None, 2, 0, 1e-6, 4096, None, None, 0, None) == -1
    assert lib.odw_rms_norm(4096, 4, 4096, 4, None, 2, 4, 1e-6, 4096, None, None, 0, None) == -1        # a residual without h
    assert lib.odw_rms_norm(4096, 4, None, 0, None, 2, 4, 1e-6, 4096, None, None, 8, None) == -1
    assert lib.odw_rms_norm_fp8(4096, 4, None, 0, None, 2, 4, 1e-6, 4096, None, None, 0, None) == -1
    assert lib.odw_rms_norm_bwd(None, 4, None, 0, None, 4, None, None, 2, 4, None, None, None, 0, None, 0, None) == -1
    assert lib.odw_rms_norm_bwd(4096, 4, None, 0, 4096, 4, None, 4096, 2, 4, None, None, 4096, 0, None, 0, None) == -3


def test_8_bit_states_hold_what_they_are_given():
    """Relative error at most half a grid step (2^-4 for the first average, 2^-3 for the second) down to the formats' normal numbers, and
    absolute below them: half of a lowest step for the first, 2^-10 of the scale, whose largest value is over 1.75 * 2^7 of it (2^-17 of
    the largest); the whole lowest step for the second, 2^-16 of the scale, because what is not zero is moved up to it, with the largest value over
    1.75 * 2^14 (under 2^-30 of it); a second write gives the same; shapes and empty tensors."""
    g = torch.Generator().manual_seed(1)
    for shape in ((0,), (), (1,), (255,), (3, 100), (513,)):
        m = torch.randn(shape, generator=g) * torch.exp(2 * torch.randn(shape, generator=g))
        v = m.square() * 0.01
        q = optim.state8_write(m, v)
        assert q[0].shape == m.shape and q[0].dtype == torch.float8_e4m3fn and q[1].dtype == torch.float8_e5m2
        assert q[2].shape == (-(-m.numel() // 256), 2) and q[2].dtype == torch.uint8
        rm, rv = optim.state8_read(*q)
        if m.numel():
            assert ((rm - m).abs() <= m.abs() * 2.0 ** -4 + m.abs().max() * 2.0 ** -17).all()
            assert ((rv - v).abs() <= v * 2.0 ** -3 + v.max() * 2.0 ** -30).all() and (rv[v > 0] > 0).all()
        again = optim.state8_read(*optim.state8_write(rm, rv))
        assert torch.equal(again[0], rm) and torch.equal(again[1], rv)
    z = optim.state8_zeros(torch.zeros(300))
    assert not any(x.any() for x in optim.state8_read(*z)) and optim.state8_write(torch.zeros(300), torch.zeros(300))[2].eq(1).all()
    bad = optim.state8_read(*optim.state8_write(torch.tensor([1.0, math.inf, math.nan]), torch.tensor([1.0, math.inf, math.nan])))
    assert all(x[0] == 1 and x[1:].isnan().all() for x in bad)
