"""A training step that fails in the body's backward, behind the head's early update, and the same step again."""
import pytest
import torch

from test_adamw_engine_gpu import U, _engine, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_the_retried_step_is_the_heads_next_update(bits):
    """The failed step leaves the head updated with number 1; the retried one updates it with number 2 and everything else with 1, each as the formula
    says (bounds as in test_adamw_engine_gpu)."""
    cfg, step, _, batch = _engine("ODW.STATE_BITS", bits)
    opt, heads = step.optimizer, step.model.roi_heads
    ready = heads.head_grads_ready

    def fails():
        ready()
        raise RuntimeError("the body's backward fails")
    start = opt.flat_p.clone()
    heads.head_grads_ready = fails
    with pytest.raises(RuntimeError, match="body's backward"):
        _run(step, cfg, batch, 0)
    heads.head_grads_ready = ready
    torch.cuda.synchronize()
    assert opt.steps == 0 and opt.head_ahead == 1
    p0, (m0, v0) = opt.flat_p.clone(), [x.clone() for x in opt._averages()]
    assert not torch.equal(p0[:opt.n_gemm], start[:opt.n_gemm]) and torch.equal(p0[opt.n_gemm:], start[opt.n_gemm:])
    _run(step, cfg, batch, 0)
    torch.cuda.synchronize()
    assert opt.steps == 1 and opt.head_ahead == 1
    for name, (off, n) in opt.slices.items():
        part, t = slice(off, off + n), 2 if off < opt.n_gemm else 1
        lr, wd = [(lr, wd) for s, k, lr, wd in opt.regions if s <= off < s + k][0]
        g = opt.flat_g[part].double()
        m, v = 0.9 * m0[part].double() + (1 - 0.9) * g, 0.999 * v0[part].double() + (1 - 0.999) * g * g
        ratio = m / (1 - 0.9 ** t) / ((v / (1 - 0.999 ** t)).sqrt() + 1e-8)
        want = p0[part].double() * (1 - lr * wd) - lr * ratio
        assert ((opt.flat_p[part].double() - want).abs() <= 2 * U * (want.abs() + lr) + 24 * U * lr * (1 + ratio.abs())).all(), name
