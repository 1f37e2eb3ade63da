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


def _net(last, seed=3):
    torch.manual_seed(seed)
    net = torch.nn.ParameterList([torch.randn(16, 8, 3, 3), torch.randn(40, 30).t() if last else torch.randn(40, 30).t().contiguous(), torch.randn(7)]).cuda()
    if last:
        net[0].data = net[0].data.to(memory_format=torch.channels_last)
    return net


def _step(net, opt, t):
    for i, p in enumerate(net):
        p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(10 * t + i)).cuda()
        if t % 2:
            p.grad = p.grad.to(memory_format=torch.channels_last) if p.dim() == 4 else p.grad
    opt.step()


def test_adamw_on_channels_last_parameters():
    """An element's update does not depend on where it lies: the same bits as with contiguous parameters, and states as they lie."""
    from od_wscl_amd import optim
    a, b = _net(True), _net(False)
    assert not a[0].is_contiguous() and not a[1].is_contiguous() and all(torch.equal(p, q) for p, q in zip(a, b))
    oa, ob = (optim.AdamW(n.parameters(), lr=1e-2, weight_decay=0.1) for n in (a, b))
    for t in range(4):
        _step(a, oa, t)
        _step(b, ob, t)
    for p, q in zip(a, b):
        assert torch.equal(p, q) and oa.state[p]["exp_avg"].stride() == p.stride() and torch.equal(oa.state[p]["exp_avg_sq"], ob.state[q]["exp_avg_sq"])
    a[0].data = a[0].data.contiguous()                     # laid out anew: the averages follow
    b[1].data = b[1].data.t().contiguous().t()
    for t in range(4, 6):
        _step(a, oa, t)
        _step(b, ob, t)
    for p, q in zip(a, b):
        assert torch.equal(p, q) and oa.state[p]["exp_avg"].stride() == p.stride()


@pytest.mark.parametrize("laid_anew", [False, True])
def test_adamw_in_8_bits_on_channels_last_parameters(laid_anew):
    """A block's 256 elements are neighbours in memory; the state moves through a checkpoint, and with a parameter laid out anew, unrounded where the
    blocks stay the same ones."""
    from od_wscl_amd import optim
    a = _net(True)
    oa = optim.AdamW(a.parameters(), lr=1e-2, state_bits=8, seed=5)
    for t in range(3):
        _step(a, oa, t)
    st = oa.state[a[0]]
    flat = [st[k].permute(0, 2, 3, 1) for k in ("exp_avg", "exp_avg_sq")]
    assert all(x.is_contiguous() for x in flat) and st["scales"].shape == (-(-a[0].numel() // 256), 2)
    m, v = optim.state8_read(*flat, st["scales"])
    sd = oa.state_dict()
    assert torch.equal(sd["state"][0]["exp_avg"], m.permute(0, 3, 1, 2)) and torch.equal(sd["state"][0]["exp_avg_sq"], v.permute(0, 3, 1, 2))
    b = _net(True)
    for p, q in zip(a, b):
        q.data.copy_(p.data)
    ob = optim.AdamW(b.parameters(), lr=1e-2, state_bits=8, seed=5)
    ob.load_state_dict(sd)
    if laid_anew:       # other blocks: the averages are rounded once more, to nearest -- half a step of the largest value's
        a[0].data = a[0].data.contiguous()
        _step(a, oa, 3)
        _step(b, ob, 3)
        assert oa.state[a[0]]["exp_avg"].is_contiguous()
        # (a ratio of at most 7.3 * lr; m and the root of v each off by 2^-4 and 2^-4 of their blocks' largest)
        assert (a[0] - b[0]).abs().max().item() <= 7.3e-2 and torch.equal(a[1], b[1])
        return
    for t in range(3, 6):                                  # a resumed run continues bit for bit
        _step(a, oa, t)
        _step(b, ob, t)
    for p, q in zip(a, b):
        assert torch.equal(p, q)


def test_what_has_gaps_is_refused():
    from od_wscl_amd import optim
    p = torch.nn.Parameter(torch.zeros(4, 10, device="cuda")[:, :9])
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match="contiguous"):
        optim.AdamW([p]).step()
