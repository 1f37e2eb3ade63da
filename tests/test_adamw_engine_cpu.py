"""engine.FlatAdamW without a GPU: configuration, state layout, checkpoints between 32 and 8 bits and torch.optim.AdamW."""
import pytest
import torch


class Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.conv = torch.nn.Conv2d(3, 40, 3)
        self.frozen = torch.nn.Conv2d(4, 4, 1)
        self.out = torch.nn.Conv2d(4, 2, 1)
        for p in self.frozen.parameters():
            p.requires_grad_(False)


def _cfg(*more):
    from od_wscl_amd.config import make_defaults
    cfg = make_defaults()
    cfg.merge_from_list(["SOLVER.BASE_LR", 0.01, "SOLVER.STEPS", (5, 8), "SOLVER.WARMUP_ITERS", 2, "ODW.OPTIMIZER", "ADAMW"] + list(more))
    return cfg


def test_configuration():
    from od_wscl_amd import engine
    from od_wscl_amd.config import make_defaults
    assert type(engine.build_optimizer(make_defaults(), Net())) is engine.FlatSGD
    o = engine.build_optimizer(_cfg("ODW.CLIP_NORM", 2.0, "ODW.STATE_BITS", 8), Net())
    assert type(o) is engine.FlatAdamW and o.bits == 8 and o.clip_norm == 2.0 and not hasattr(o, "flat_m")
    assert sum(x.numel() for st in o.state8 for x in st[:2]) == 2 * o.total
    for bad in (["ODW.STATE_BITS", 4], ["ODW.CLIP_NORM", -1.0], ["ODW.OPTIMIZER", "LION"], ["ODW.OPTIMIZER", "SGD", "ODW.CLIP_NORM", 1.0]):
        with pytest.raises(ValueError):
            engine.build_optimizer(_cfg(*bad), Net())


@pytest.mark.parametrize("bits", [32, 8])
def test_state_round_trips_through_a_checkpoint_and_torch(tmp_path, bits):
    from od_wscl_amd import engine, optim
    from od_wscl_amd.utils import checkpoint as ck
    cfg = _cfg("ODW.STATE_BITS", bits)
    torch.manual_seed(0)
    a = Net()
    oa = engine.build_optimizer(cfg, a)
    assert oa.state_dict(a)["state"] == {}                     # before the first step
    m, v = torch.randn_like(oa.flat_p), torch.rand_like(oa.flat_p)
    if bits == 8:
        for (s, n, _, _), st in zip(oa.regions, oa.state8):
            optim.state8_write(m[s:s + n], v[s:s + n], out=st)
    else:
        oa.flat_m.copy_(m)
        oa.flat_v.copy_(v)
    oa.steps, oa.sched_steps, oa.lr_scale = 6, 6, engine.lr_factor(cfg, 6)
    path = str(tmp_path / "model_0000006.pth")
    ck.save_checkpoint(a, path, optimizer=oa, iteration=6)
    saved = torch.load(path)
    trainable = [(n, p) for n, p in Net().named_parameters() if p.requires_grad]
    ref = torch.optim.AdamW([{"params": [p], "lr": 0.01} for _, p in trainable], 0.01)
    ref.load_state_dict(saved["optimizer"])
    assert len(ref.state_dict()["state"]) == len(trainable) and float(ref.state_dict()["state"][0]["step"]) == 6
    assert abs(saved["optimizer"]["param_groups"][1]["lr"] - 0.01 * 2 * 0.1) < 1e-12
    for source in (saved["optimizer"], ref.state_dict()):
        b = Net()
        ob = engine.build_optimizer(cfg, b)
        rest = ck.load_checkpoint(b, path)
        assert ck.restore_training_state(ob, b, dict(rest, optimizer=source)) == 6
        assert ob.steps == 6 and ob.lr_scale == oa.lr_scale
        want, got = oa._averages(), ob._averages()
        for n, (off, k) in oa.slices.items():
            for x, y in zip(want, got):
                assert torch.equal(x[off:off + k], y[off:off + k]), n
            assert torch.equal(oa.flat_p[off:off + k], ob.flat_p[off:off + k]), n        # (the padding between them is uninitialised)
    other = engine.build_optimizer(_cfg("ODW.STATE_BITS", 40 - bits), Net())      # the other width reads it too
    c = Net()
    oc = engine.build_optimizer(_cfg("ODW.STATE_BITS", 40 - bits), c)
    oc.load_state_dict(c, saved["optimizer"])
    assert oc.steps == 6
    for n, (off, k) in oa.slices.items():
        x, y = (o._averages()[0][off:off + k] for o in (oc, oa))
        assert (x - y).abs().max() <= 2.0 ** -4 * y.abs().max(), n
    sgd = engine.FlatSGD(_cfg(), a)
    sgd.first = False
    with pytest.raises(ValueError, match="SGD"):
        other.load_state_dict(c, sgd.state_dict(a))
    torch_state = {i: dict(st) for i, st in saved["optimizer"]["state"].items()}
    torch_state[0]["step"] = torch.tensor(7.0)
    with pytest.raises(ValueError, match="different numbers"):
        other.load_state_dict(c, {"state": torch_state, "param_groups": saved["optimizer"]["param_groups"]})


def test_schedule_does_not_touch_the_averages():
    from od_wscl_amd import engine
    o = engine.build_optimizer(_cfg(), Net())
    o.first = False
    o.flat_m.fill_(1.0)
    o.set_iteration(4)
    o.set_iteration(5)                                          # SGD rescales its momentum at this jump of 10
    assert abs(o.lr_scale - 0.1) < 1e-12 and (o.flat_m == 1).all()


def test_states_of_another_rule_are_refused():
    from od_wscl_amd import engine
    net = Net()
    groups = [{"params": [p]} for p in net.parameters() if p.requires_grad]
    o = engine.build_optimizer(_cfg(), net)
    for other in (torch.optim.AdamW(groups, amsgrad=True), torch.optim.AdamW(groups, maximize=True), torch.optim.Adam(groups, weight_decay=0.1)):
        with pytest.raises(ValueError, match="amsgrad|maximize|coupled"):
            o.load_state_dict(net, other.state_dict())
