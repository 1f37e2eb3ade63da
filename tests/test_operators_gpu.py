"""perf/operators.py: the package's calls give what the plain forms give, over two passes on the same state.

Bounds (u = 2^-24): norm: fp32 sums of up to 700 terms in another order, 64 u; a bf16 output may round the other way, one step of 2^-7 (where
the plain form rounds dresidual and dx twice, two); 8-bit codes: one step of 2^-3, 2^-9 for
the lowest.  clip, adamw: 64 u of what an update moves, and of the value.
adamw8: the plain form rounds values below the smallest normal code after an fp32 addition, so that one in 2^16 of those may differ."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
CASES = [
    {"op": "norm", "rows": 5, "dim": 700, "dtype": "f32", "residual": True, "grad": True},
    {"op": "norm", "rows": 9, "dim": 513, "dtype": "bf16", "residual": False, "grad": True},
    {"op": "norm", "rows": 3, "dim": 640, "dtype": "bf16", "residual": True, "grad": False},
    {"op": "norm8", "rows": 7, "dim": 601, "dtype": "f32", "residual": True},
    {"op": "clip", "tensors": "ragged", "count": 60, "total": 50001, "layout": 3, "grads": "bf16"},
    {"op": "adamw", "tensors": "ragged", "count": 60, "total": 50001, "layout": 4, "grads": "bf16", "clip": True, "copies": True},
    {"op": "adamw8", "tensors": "ragged", "count": 60, "total": 150001, "layout": 5, "grads": "f32", "clip": False, "copies": True},
    {"op": "adamw8", "tensors": "ragged", "count": 120, "total": 90001, "layout": 6, "grads": "bf16", "clip": False, "copies": False},
]


@pytest.fixture(scope="module")
def operators():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")
    spec = importlib.util.spec_from_file_location("operators_under_test", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _two_passes(mod, own, case):
    mod.own = own
    s = mod.prepare(dict(case), 11)
    mod.run(s)
    out = mod.run(s)
    parts = {k: s[k] for k in ("p", "g", "m", "v", "e", "copy", "grads") if k in s}        # (between the tensors lies what was there)
    return {k: v.clone() for k, v in out.items() if k not in ("p", "m", "v", "copy", "scales", "grads")}, parts


@pytest.mark.parametrize("case", CASES, ids=lambda c: "%s-%s" % (c["op"], c.get("dim", c.get("total"))))
def test_the_calls_give_what_the_plain_forms_give(operators, case):
    (want, parts), (got, own) = (_two_passes(operators, own, case) for own in (False, True))
    assert want.keys() == got.keys() and parts.keys() == own.keys()
    for k, w in want.items():
        g = got[k]
        assert g.dtype == w.dtype and g.shape == w.shape
        rel = {torch.float32: 64 * U, torch.bfloat16: 2.0 ** -6, torch.float8_e4m3fn: 2.0 ** -3}[w.dtype]
        w, g = w.double(), g.double()
        floor = 64 * U * w.abs().max() if k.startswith("d") else 2.0 ** -9 if k == "q" else 0.0
        assert ((g - w).abs() <= rel * w.abs() + floor).all(), k
    differ, codes = 0, 0
    for k, ws in parts.items():
        for w, g in zip(ws, own[k]):
            w, g = w.double(), g.double()
            if k == "e":
                assert torch.equal(w, g)
            elif k in "mv" and case["op"] == "adamw8":
                differ, codes = differ + int((w != g).sum()), codes + w.numel()
            else:
                half = 2.0 ** -7 if (k == "copy" or (k == "grads" and case["grads"] == "bf16")) else 64 * U
                assert ((g - w).abs() <= half * w.abs() + (64 * U * operators.LR * 8 if k in ("p", "copy") else 0.0)).all(), k
    assert differ <= codes * 2.0 ** -16 + 3
