"""8-bit codes of rows whose largest product is met twice: the products are equal in fp32 and their exact values are not."""
from fractions import Fraction

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _codes(x, w):
    """rne(448 t / max |t|), t = x w, in rationals, as the values the codes stand for."""
    t = [Fraction(float(a)) * Fraction(float(b)) for a, b in zip(x, w)]
    top = max(abs(v) for v in t)
    out = []
    for v in t:
        z = 448 * v / top
        e = -6
        while abs(z) >= Fraction(2) ** (e + 1):
            e += 1
        out.append(float(round(z * Fraction(2) ** (3 - e)) * Fraction(2) ** (e - 3)))       # (round() goes to the even one)
    return out


def _row():
    """448 t / max |t| of the last one is 17 - 2.6e-7 by the first product and 17 + 4.2e-7 by the second: codes 16 and 18."""
    return (np.array([1.0641474723815918, 1.1613094806671143, 1.679557204246521], np.float32),
            np.array([1.1451144218444824, 1.0493073463439941, 0.027531305328011513], np.float32))


@pytest.mark.parametrize("order", [(0, 1, 2), (1, 0, 2), (2, 1, 0), (2, 0, 1)])
@pytest.mark.parametrize("signs", [(1, 1, 1), (-1, 1, 1), (1, -1, -1), (-1, -1, -1)])
@pytest.mark.parametrize("gap", [1, 4, 64, 1025])
def test_equal_largest_products(order, signs, gap):
    """`gap` columns between the three: one thread's, two threads', two waves'; zeros elsewhere."""
    from od_wscl_amd import layers
    x3, w3 = (v[list(order)] for v in _row())
    assert x3[0] * w3[0] == x3[1] * w3[1] or x3[1] * w3[1] == x3[2] * w3[2] or x3[0] * w3[0] == x3[2] * w3[2]
    x, w = np.zeros(2 * gap + 1, np.float32), np.ones(2 * gap + 1, np.float32)
    x[::gap], w[::gap] = x3 * np.array(signs, np.float32), w3
    q, _ = layers.rms_norm_fp8(torch.from_numpy(x)[None].cuda(), torch.from_numpy(w).cuda(), eps=1e-6)
    assert q.float().cpu().numpy()[0, ::gap].tolist() == _codes(x[::gap], w[::gap])
    assert abs(_codes(x3, w3)[order.index(2)]) == 16.0
