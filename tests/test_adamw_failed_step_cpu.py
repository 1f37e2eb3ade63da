"""engine.FlatAdamW's numbers: what a step that fails behind head_grads_ready leaves, the ranks' mean and the clip factor -- recorded, without a GPU."""
import pytest
import torch


class Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        from od_wscl_amd.layers.linear import Linear
        self.conv = torch.nn.Conv2d(3, 40, 3)
        self.fc = Linear(24, 16)


def _optimizer(monkeypatch, *more, world=1):
    from od_wscl_amd import engine, optim
    from od_wscl_amd.config import make_defaults
    calls = []

    def adamw_step(p, g, m, v, step, **k):
        calls.append(dict(k, sizes=[x.numel() for x in p], step=step))

    def adamw8_step(p, g, m, v, e, step, key, **k):
        calls.append(dict(k, sizes=[x.numel() for x in p], step=step, key=key))
    monkeypatch.setattr(optim, "adamw_step", adamw_step)
    monkeypatch.setattr(optim, "adamw8_step", adamw8_step)
    monkeypatch.setattr(optim, "grad_norm", lambda grads, max_norm: (torch.tensor(6.0), ("coef", max_norm)))
    cfg = make_defaults()
    cfg.merge_from_list(["ODW.OPTIMIZER", "ADAMW"] + list(more))
    net = Net()
    return engine.build_optimizer(cfg, net, world), net, calls


def _step(opt, fails=False):
    opt.begin_step()
    if fails:
        opt._update((0,), paced=160)          # (head_grads_ready: on the side stream; then the backward fails)
    else:
        opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_failed_step_is_an_update_of_the_head_alone(monkeypatch, bits):
    opt, net, calls = _optimizer(monkeypatch, "ODW.STATE_BITS", bits)
    head, rest = [24 * 16], [40 * 27, 40 + 16]
    for fails in (False, True, False, False, True, True, False):
        _step(opt, fails)
    assert [c["step"] for c in calls if c["sizes"] == head] == [1, 2, 3, 4, 5, 6, 7]
    assert [c["step"] for c in calls if c["sizes"] == rest] == [1, 2, 3, 4] and opt.steps == 4
    if bits == 8:
        keys = [c["key"] for c in calls]
        assert len(set(keys)) == len(keys) == 11
    sd = opt.state_dict(net)
    steps = {n: float(sd["state"][i]["step"]) for i, n in enumerate(opt._param_order(net))}
    assert steps == {"conv.weight": 4, "conv.bias": 4, "fc.weight": 7, "fc.bias": 4}
    again, net2, calls2 = _optimizer(monkeypatch, "ODW.STATE_BITS", bits)
    again.load_state_dict(net2, sd)
    _step(again)
    assert [c["step"] for c in calls2] == [8, 5]
    sd["state"][0]["step"] = torch.tensor(3.0)
    with pytest.raises(ValueError, match="different numbers"):
        again.load_state_dict(net2, sd)


def test_a_first_step_that_fails(monkeypatch):
    opt, net, calls = _optimizer(monkeypatch)
    _step(opt, True)
    sd = opt.state_dict(net)
    assert [float(st["step"]) for st in sd["state"].values()] == [1.0]
    again, net2, calls2 = _optimizer(monkeypatch)
    again.load_state_dict(net2, sd)
    _step(again)
    assert [c["step"] for c in calls2] == [2, 1]


def test_a_refused_update_is_not_counted(monkeypatch):
    from od_wscl_amd import optim
    opt, _, calls = _optimizer(monkeypatch)

    def refuse(*a, **k):
        raise RuntimeError("refused")
    good = optim.adamw_step
    monkeypatch.setattr(optim, "adamw_step", refuse)
    with pytest.raises(RuntimeError):
        _step(opt, True)
    monkeypatch.setattr(optim, "adamw_step", good)
    _step(opt)
    assert [c["step"] for c in calls] == [1, 1]


@pytest.mark.parametrize("world", [1, 4])
def test_the_mean_over_the_ranks(monkeypatch, world):
    """Gradients arrive summed: the update takes them times 1 / world, and their sum's norm is clipped to world times the limit."""
    opt, _, calls = _optimizer(monkeypatch, "ODW.CLIP_NORM", 0.5, world=world)
    opt.exchange.world = 1                       # (no exchange: the numbers of the update alone)
    _step(opt)
    assert [c["grad_mult"] for c in calls] == [1.0 / world] * 2 and [c["grad_scale"] for c in calls] == [("coef", 0.5 * world)] * 2
    assert float(opt.grad_norm) == 6.0 / world
