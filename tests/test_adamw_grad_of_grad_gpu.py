"""Gradients that require gradients themselves are clipped and applied like others."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("way", ["leaf", "create_graph"])
def test_a_gradient_that_requires_grad(way):
    from od_wscl_amd import optim
    x = torch.linspace(-2.0, 2.0, 9, device="cuda")
    p, q = torch.nn.Parameter(x.clone()), torch.nn.Parameter(x.clone())
    if way == "leaf":
        p.grad = (x * 3).requires_grad_(True)
    else:
        (p * p * 1.5).sum().backward(create_graph=True)
        assert p.grad.requires_grad
    q.grad = x * 3
    norms = []
    for t in (p, q):
        o = optim.AdamW([t], lr=0.1, max_grad_norm=1.0)
        o.step()
        norms.append(o.grad_norm.item())
    assert norms[0] == norms[1] and abs(norms[0] / (3 * x.norm().item()) - 1) < 1e-6 and torch.equal(p, q)
    p.grad = None
