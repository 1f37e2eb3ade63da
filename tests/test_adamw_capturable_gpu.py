"""optim.AdamW(capturable=True) where parameters do not step alike: groups of other betas and eps, missing gradients, reloads."""
import pytest
import torch

pytestmark = pytest.mark.gpu
SHAPES = ((30, 40), (40,), (7, 3), ())


def _pair(bits=32):
    from od_wscl_amd import optim

    def params():
        g = torch.Generator().manual_seed(21)
        return [torch.nn.Parameter(torch.randn(s, generator=g).cuda()) for s in SHAPES]
    a, b = params(), params()
    groups = lambda ps: [{"params": ps[:1]}, {"params": ps[1:3], "betas": (0.8, 0.99)}, {"params": ps[3:], "eps": 1e-6}]     # noqa: E731
    return a, b, optim.AdamW(groups(a), lr=1e-2, capturable=True, state_bits=bits), torch.optim.AdamW(groups(b), lr=1e-2)


def _gradients(a, b, t, without=()):
    for i, (p, q) in enumerate(zip(a, b)):
        g = torch.randn(p.shape, generator=torch.Generator().manual_seed(100 * t + i)).cuda()
        p.grad, q.grad = (None, None) if i in without else (g, g.clone())


def _near(a, b):
    """(the products' parameters are not set to torch's in between: a few roundings of lr = 1e-2 a step)"""
    for p, q in zip(a, b):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("parted", [False, True])
def test_groups_of_other_rules_and_missing_gradients(parted):
    from od_wscl_amd import optim
    a, b, ours, ref = _pair()
    for t in range(1, 9):
        _gradients(a, b, t, {3: (2,), 5: (0, 1), 6: (1,)}.get(t, ()) if parted else ())
        if t == 7 and parted:                              # another rule for one parameter's group
            for o in (ours, ref):
                o.param_groups[1]["betas"] = (0.85, 0.98)
        ours.step()
        ref.step()
        _near(a, b)
    steps = [float(ours.state_dict()["state"][i]["step"]) for i in range(4)]
    assert steps == [float(ref.state_dict()["state"][i]["step"]) for i in range(4)]
    again = optim.AdamW([{"params": a[:1]}, {"params": a[1:3]}, {"params": a[3:]}], capturable=True)
    again.load_state_dict(ours.state_dict())
    for t in range(9, 12):
        _gradients(a, b, t)
        again.step()
        ref.step()
        _near(a, b)
    assert [float(again.state_dict()["state"][i]["step"]) for i in range(4)] == [s + 3 for s in steps]


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_groups(bits):
    """Replays of a step of three rules against the same steps taken eagerly; a step that would part them is not captured."""
    a, b, ours, _ = _pair(bits)
    twin = _pair(bits)[2]
    b = [p for g in twin.param_groups for p in g["params"]]
    _gradients(a, b, 0)
    ours.step()
    twin.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ours.step()
    for t in range(1, 5):
        held = [p.grad for p in a]
        _gradients(b, b, t)
        for h, q in zip(held, b):
            h.copy_(q.grad)
        graph.replay()
        twin.step()
        torch.cuda.synchronize()
        for p, q in zip(a, b):
            assert torch.equal(p, q)
        assert [float(x["step"]) for x in ours.state_dict()["state"].values()] == [t + 1.0] * 4
    a[1].grad = None                                       # shares its counter with a[2]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="step counter"):
                ours.step()
            a[0].grad.mul_(1.0)
        finally:
            graph.capture_end()


def test_one_fill_for_many_parameters():
    """The first step makes one counter for all parameters of a rule."""
    from od_wscl_amd import optim
    ps = [torch.nn.Parameter(torch.zeros(3, device="cuda")) for _ in range(50)]
    o = optim.AdamW(ps, capturable=True)
    for p in ps:
        p.grad = torch.ones_like(p)
    o.step()
    assert len(set(id(o.state[p]["step"]) for p in ps)) == 1


@pytest.mark.parametrize("bad", [dict(max_workgroups=-1), dict(lr=-1.0), dict(eps=0.0), dict(betas=(1.0, 0.9)), dict(grad_mult=float("nan")),
                                 dict(copies=[]), dict(exp_avgs=[torch.zeros(7)]), dict(grad_scale=torch.ones(2))], ids=lambda d: list(d)[0])
def test_a_refused_step_leaves_its_number(bad):
    from od_wscl_amd import optim
    one = lambda: [torch.ones(8, device="cuda")]           # noqa: E731
    step = torch.full((1,), 4, dtype=torch.int64, device="cuda")
    args = dict(params=one(), grads=one(), exp_avgs=one(), exp_avg_sqs=one(), step=step)
    with pytest.raises((ValueError, RuntimeError)):
        optim.adamw_step(**{**args, **bad})
    assert int(step) == 4 and torch.equal(args["params"][0], one()[0])
    optim.adamw_step(**args)
    assert int(step) == 5
