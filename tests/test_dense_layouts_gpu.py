"""Gradients and parameters whose elements lie in another order without gaps (channels_last weights, transposed matrices)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def test_clip_and_norm():
    from od_wscl_amd import optim
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(16, 8, 3, 5, generator=gen).cuda()
    forms = (x.clone(), x.to(memory_format=torch.channels_last), x.permute(3, 1, 0, 2).contiguous().permute(2, 1, 3, 0))
    want = x.double().norm().item()
    for g in forms:
        assert torch.equal(g, x)
        before = g.data_ptr()
        n, c = optim.grad_norm([g], 1.0)
        assert abs(n.item() / want - 1) <= 2 * U
        assert torch.equal(optim.clip_grad_norm_([g], 1.0), n) and torch.equal(g, x * c) and g.data_ptr() == before
    p = torch.nn.Parameter(x.to(memory_format=torch.channels_last))
    p.grad = torch.randn_like(p)
    assert not p.grad.is_contiguous()
    optim.clip_grad_norm_([p], 1e-3)
    assert abs(p.grad.norm().item() / 1e-3 - 1) <= 1e-5
    rows = torch.zeros(4, 10, device="cuda")
    for bad in (rows[:, :9], rows[:1].expand(4, 10), rows[:, ::2]):
        with pytest.raises(ValueError, match="contiguous"):
            optim.clip_grad_norm_([bad], 1.0)
        assert optim.grad_norm([bad]).item() == 0.0
