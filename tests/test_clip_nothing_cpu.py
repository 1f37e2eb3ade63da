"""Clipping where no parameter has a gradient: nothing to do, as in torch.nn.utils.clip_grad_norm_ -- on the CPU too, since nothing is launched."""
import pytest
import torch

from od_wscl_amd import optim


def test_no_gradients():
    p = torch.nn.Parameter(torch.ones(3))
    for items in ([p, p], [], p, iter([p])):
        n = optim.clip_grad_norm_(items, 1.0)
        want = torch.nn.utils.clip_grad_norm_([p] if items is p else [], 1.0)
        assert n.shape == want.shape == () and n.dtype == want.dtype and n.item() == want.item() == 0.0
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            optim.clip_grad_norm_([p], bad)
    with pytest.raises(ValueError):
        optim.grad_norm([p])                    # (a norm of nothing is asked for by mistake)
