"""Lazily negated views (torch's way to take the imaginary part of a conjugate): their memory holds the other sign."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _neg(t):
    n = torch._neg_view(t.neg())
    assert n.is_neg() and torch.equal(n, t)
    return n


def test_norm_of_rows():
    from od_wscl_amd import layers
    g = torch.Generator().manual_seed(1)
    x, r, w, dy, dh = (torch.randn(*s, generator=g).cuda() for s in ((6, 40), (6, 40), (40,), (6, 40), (6, 40)))

    def run(*t):
        a, b, c = (u.detach().requires_grad_(True) for u in t[:3])
        y, h = layers.rms_norm(a, c, residual=b)
        return (y, h) + torch.autograd.grad((y, h), (a, b, c), t[3:]) + layers.rms_norm_fp8(a, c, residual=b)
    want = run(x, r, w, dy, dh)
    for k in range(5):
        got = run(*(_neg(t) if i == k else t for i, t in enumerate((x, r, w, dy, dh))))
        for a, b in zip(got, want):
            assert torch.equal(a.float(), b.float()), k
    # an output as the imaginary part of what is conjugated later
    a = x.clone().requires_grad_(True)
    torch.complex(torch.zeros_like(x), layers.rms_norm(a)).conj().imag.backward(dy)
    b = x.clone().requires_grad_(True)
    layers.rms_norm(b).backward(-dy)
    assert torch.equal(a.grad, b.grad)


def test_optimiser():
    from od_wscl_amd import optim
    t = lambda: torch.full((8,), 2.0, device="cuda")          # noqa: E731
    for k in range(4):
        args = [[_neg(t())] if i == k else [t()] for i in range(4)]
        with pytest.raises(ValueError, match="negated"):
            optim.adamw_step(*args, 1)
    assert float(optim.grad_norm([_neg(t())])) == float(optim.grad_norm([t()]))
    n = _neg(t())
    optim.clip_grad_norm_([n], 1.0)
    assert torch.allclose(n, torch.full_like(n, 8 ** -0.5))
    p, q = (torch.nn.Parameter(t()) for _ in range(2))
    p.grad, q.grad = _neg(t()), t()
    for x in (p, q):
        optim.AdamW([x]).step()
    assert torch.equal(p, q)
