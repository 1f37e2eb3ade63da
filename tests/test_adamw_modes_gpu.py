"""engine.FlatAdamW in the other precision modes of the training step: with bf16 operands alone (a shadow of the weights), and in the fp32-grade mode
(none); and its update as one of several ranks' -- gradients already summed."""
import pytest
import torch

from test_adamw_engine_gpu import U, _run

pytestmark = pytest.mark.gpu


def _engine(dtype, *more):
    import bench
    from od_wscl_amd import engine
    dev = torch.device("cuda", 0)
    cfg = bench.build_cfg(21)
    cfg.merge_from_list(["ODW.OPTIMIZER", "ADAMW", "SOLVER.BASE_LR", 1e-4, "SOLVER.WEIGHT_DECAY", 0.01, "SOLVER.WARMUP_ITERS", 0] + list(more))
    step, _ = engine.build_training_step(cfg, dev, dtype=dtype, world=1, seed=cfg.SEED)
    return cfg, step, bench.synthetic_batch(cfg.SEED, 1, 224, 160, 21, dev)


@pytest.mark.parametrize("dtype,bits,clip,world", [("bf16", 8, 0.0, 1), ("bf16", 32, 0.05, 1), ("bf16x3", 32, 0.0, 1), ("bf16x3", 8, 0.05, 1),
                                                   ("bf16x2f", 8, 0.05, 4), ("bf16x2f", 32, 0.0, 4)])
def test_two_steps_update_as_the_formula_says(dtype, bits, clip, world):
    """Bounds as in test_adamw_engine_gpu."""
    cfg, step, batch = _engine(dtype, "ODW.STATE_BITS", bits, "ODW.CLIP_NORM", clip)
    opt = step.optimizer
    opt.world = world                                       # (no exchange: what is in the buffer stands for the ranks' sum)
    for it in range(2):
        torch.cuda.synchronize()
        p0, (m0, v0) = opt.flat_p.clone(), [x.clone() for x in opt._averages()]
        _run(step, cfg, batch, it)
        torch.cuda.synchronize()
        coef = 1.0 / world
        if clip > 0.0:
            norm = opt.flat_g.double().square().sum().sqrt().item() / world
            assert abs(opt.grad_norm.item() / norm - 1) <= 4 * U
            coef *= min(1.0, clip / (norm + 1e-6 / world))
        for name, (off, n) in opt.slices.items():
            part, t = slice(off, off + n), it + 1
            lr, wd = [(lr, wd) for s, k, lr, wd in opt.regions if s <= off < s + k][0]
            g = opt.flat_g[part].double() * coef
            m, v = 0.9 * m0[part].double() + (1 - 0.9) * g, 0.999 * v0[part].double() + (1 - 0.999) * g * g
            ratio = m / (1 - 0.9 ** t) / ((v / (1 - 0.999 ** t)).sqrt() + 1e-8)
            want = p0[part].double() * (1 - lr * wd) - lr * ratio
            assert ((opt.flat_p[part].double() - want).abs() <= 2 * U * (want.abs() + lr) + 24 * U * lr * (1 + ratio.abs())).all(), name
        assert (opt.flat_w16 is None) == (dtype == "bf16x3")
        if opt.flat_w16 is not None:
            assert torch.equal(opt.flat_w16, opt.flat_p[:opt.n_gemm].to(torch.bfloat16))
