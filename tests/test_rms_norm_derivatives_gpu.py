"""Derivatives that layers.rms_norm does not have are refused, not taken for zero; so are traces, which would not hold the launches."""
import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["x", "weight", "residual"])
def test_forward_mode(which):
    from od_wscl_amd import layers
    x, w, r = (torch.randn(*s, device="cuda") for s in ((4, 32), (32,), (4, 32)))
    with fw.dual_level():
        args = dict(x=x, weight=w, residual=r)
        layers.rms_norm(**args)                                 # nothing carries a tangent: as ever
        args[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            layers.rms_norm(**args)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            layers.rms_norm(**args)
        args = {k: v.detach().requires_grad_(True) if k != which else v for k, v in args.items()}
        with pytest.raises(RuntimeError, match="forward-mode"):
            layers.rms_norm(**args)


def test_function_transforms():
    from od_wscl_amd import layers
    x = torch.randn(4, 32, device="cuda")
    for call in (lambda: torch.func.jvp(layers.rms_norm, (x,), (x,)), lambda: torch.func.vmap(layers.rms_norm)(x[None]),
                 lambda: torch.func.grad(lambda a: layers.rms_norm(a).sum())(x)):
        with pytest.raises(RuntimeError):
            call()


def test_traces():
    from od_wscl_amd import layers, optim
    x = torch.randn(4, 32, device="cuda")

    def step(a):
        optim.adamw_step([a], [a.clone()], [torch.zeros_like(a)], [torch.zeros_like(a)], 1)
        return a
    for f in (layers.RMSNorm(32).cuda(), lambda a: layers.rms_norm_fp8(a)[1], step, lambda a: optim.grad_norm([a]), lambda a: optim.clip_grad_norm_([a], 1.0)):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(f, (x.clone(),), check_trace=False)
