"""engine.FlatAdamW in the training step of engine.build_training_step, and a normalised residual head trained through the public
operators together: layers.RMSNorm + layers.linear.Linear + optim.AdamW with clipping.  -m gpu."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
U = 2.0 ** -24


def _engine(*more):
    import bench
    from od_wscl_amd import engine
    dev = torch.device("cuda", 0)
    cfg = bench.build_cfg(21)
    cfg.merge_from_list(["ODW.OPTIMIZER", "ADAMW", "SOLVER.BASE_LR", 1e-4, "SOLVER.WEIGHT_DECAY", 0.01, "SOLVER.WARMUP_ITERS", 0] + list(more))
    step, info = engine.build_training_step(cfg, dev, dtype="bf16x2f", world=1, seed=cfg.SEED)
    return cfg, step, info, bench.synthetic_batch(cfg.SEED, 1, 224, 160, 21, dev)


def _run(step, cfg, batch, it):
    from od_wscl_amd.utils.device_rand import DeviceRand
    return step(*batch, DeviceRand(cfg.SEED, first_stream=(1 << 20) + (it << 12), device="cuda"), iteration=it + 1)


@pytest.mark.parametrize("bits,clip", [(32, 0.0), (32, 0.05), (8, 0.05), (8, 0.0)])
def test_training_steps_update_as_the_formula_says(bits, clip):
    """Three steps; each one's update recomputed in fp64 from the gradients that the step left, the parameters before it and -- held in 8
    bits -- the averages before it.  Bounds as in test_optim_gpu: m, v 4 u of their terms a step, p half a step and 16 u of lr * 2 (of
    the ratio, at most 3.2 where a held average was rounded), the clip factor 2 u more."""
    cfg, step, info, batch = _engine("ODW.STATE_BITS", bits, "ODW.CLIP_NORM", clip)
    opt = step.optimizer
    assert "AdamW, %d-bit" % bits in info["optimizer"]
    for it in range(3):
        torch.cuda.synchronize()
        p0 = opt.flat_p.clone()
        m0, v0 = (x.clone() for x in opt._averages())
        losses, _ = _run(step, cfg, batch, it)
        torch.cuda.synchronize()
        assert opt.steps == it + 1 and all(torch.isfinite(v.detach()).all() for v in losses.values())
        # (with clipping the head cannot be updated before the backward is over)
        assert opt.early_done == (clip == 0.0)
        coef = 1.0
        if clip > 0.0:
            norm = opt.flat_g.double().square().sum().sqrt().item()
            assert abs(opt.grad_norm.item() / norm - 1) <= 2 * U and norm > clip      # it does clip
            coef = clip / (norm + 1e-6)
        t = it + 1
        m1, v1 = opt._averages()
        for name, (off, n) in opt.slices.items():
            part = slice(off, off + n)
            lr, wd = [(lr, wd) for s, k, lr, wd in opt.regions if s <= off < s + k][0]
            g = opt.flat_g[part].double() * coef
            m = 0.9 * m0[part].double() + (1 - 0.9) * g
            v = 0.999 * v0[part].double() + (1 - 0.999) * g * g
            ratio = m / (1 - 0.9 ** t) / ((v / (1 - 0.999 ** t)).sqrt() + 1e-8)
            want = p0[part].double() * (1 - lr * wd) - lr * ratio
            tol = 2 * U * (want.abs() + lr) + 24 * U * lr * (1 + ratio.abs())
            assert ((opt.flat_p[part].double() - want).abs() <= tol).all(), name
            if bits == 32:
                assert ((m1[part].double() - m).abs() <= 6 * U * (m0[part].double().abs() + g.abs()) + 1e-40).all(), name
                assert ((v1[part].double() - v).abs() <= 8 * U * (v0[part].double() + g * g) + 1e-40).all(), name
        if opt.flat_w16 is not None:
            assert torch.equal(opt.flat_w16, opt.flat_p[:opt.n_gemm].to(torch.bfloat16))


def test_a_resumed_optimiser_continues_bit_for_bit(tmp_path):
    """The checkpoint holds all that the next update reads: after two training steps, the same gradients give the same parameters and
    averages on the running engine and on a resumed one.  (A whole step would not: bias gradients are summed by atomics.)"""
    from od_wscl_amd.utils import checkpoint as ck
    cfg, step, _, batch = _engine("ODW.STATE_BITS", 8, "ODW.CLIP_NORM", 0.05)
    for it in range(2):
        _run(step, cfg, batch, it)
    path = str(tmp_path / "model.pth")
    ck.save_checkpoint(step.model, path, optimizer=step.optimizer, iteration=2)
    grads = step.optimizer.flat_g.clone()

    def update(opt):
        for _ in range(2):
            opt.early_done = False
            opt.flat_g.copy_(grads)
            opt.step()
        torch.cuda.synchronize()
        return opt.flat_p.clone(), [x.clone() for x in opt._averages()]
    want, averages = update(step.optimizer)
    slices = step.optimizer.slices
    del step
    torch.cuda.empty_cache()
    cfg, step, _, batch = _engine("ODW.STATE_BITS", 8, "ODW.CLIP_NORM", 0.05)
    assert ck.restore_training_state(step.optimizer, step.model, ck.load_checkpoint(step.model, path, map_location="cuda")) == 2
    got, averages2 = update(step.optimizer)
    for name, (off, n) in slices.items():
        for x, y in zip([want] + averages, [got] + averages2):
            assert torch.equal(x[off:off + n], y[off:off + n]), name


# ---- a head of one's own ---------------------------------------------------------------------------------------------------------------


class Head(torch.nn.Module):
    """y = out(norm(h + fc(norm(h)))): a residual block between row norms, on the package's Linear."""

    def __init__(self, dim, classes):
        super().__init__()
        from od_wscl_amd.layers import RMSNorm
        from od_wscl_amd.layers.linear import Linear
        self.norm1, self.fc, self.norm2, self.out = RMSNorm(dim), Linear(dim, dim), RMSNorm(dim), Linear(dim, classes)

    def forward(self, x):
        y, h = self.norm1(x), x
        y = self.fc.fused(y, relu=True, out_f32=True)
        y, h = self.norm2(y, residual=h)
        return self.out.fused(y, out_f32=True)


def _plain(head, x):
    """The same in fp64 from the same parameters: (output, gradients of its sum of squares)."""
    ps = {n: p.detach().double().requires_grad_(True) for n, p in head.named_parameters()}
    norm = lambda v, w: v / (v.square().mean(1, keepdim=True) + 1e-6).sqrt() * w       # noqa: E731
    h = x.double()
    y = torch.relu(norm(h, ps["norm1.weight"]) @ ps["fc.weight"].t().contiguous() + ps["fc.bias"])
    y = norm(h + y, ps["norm2.weight"]) @ ps["out.weight"].t().contiguous() + ps["out.bias"]
    grads = torch.autograd.grad(y.square().mean(), list(ps.values()))
    return y.detach(), dict(zip(ps, grads))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_normalised_residual_head_trains(bits):
    """Run together in the fp32-grade mode: outputs and gradients against fp64 (bound: products of 256 terms in planes that drop 2^-23 and
    less, sums in fp32: 2^-16 of the largest value is 64 roundings), then steps whose updates see the weights of the step before."""
    from od_wscl_amd import optim
    torch.manual_seed(1)
    head = Head(256, 24).cuda()
    opt = optim.AdamW(head.parameters(), lr=1e-3, weight_decay=0.01, state_bits=bits, max_grad_norm=0.1)
    for it in range(4):
        x = torch.randn(300, 256, device="cuda")
        opt.zero_grad()
        y = head(x)
        y.square().mean().backward()
        want, grads = _plain(head, x)
        assert (y.double() - want).abs().max() <= 2.0 ** -16 * want.abs().max()
        for n, p in head.named_parameters():
            assert (p.grad.double() - grads[n]).abs().max() <= 2.0 ** -14 * grads[n].abs().max() + 1e-9, n
        before = {n: p.detach().clone() for n, p in head.named_parameters()}
        opt.step()
        total = torch.stack([p.grad.double().square().sum() for p in head.parameters()]).sum().sqrt().item()
        assert abs(opt.grad_norm.item() / total - 1) <= 2 * U
        for n, p in head.named_parameters():
            assert 0 < (p.detach() - before[n]).abs().max().item() <= 4e-3, n
