"""The AdamW object's states of parameters in another order without gaps, through checkpoints, without a GPU."""
import copy

import pytest
import torch

from od_wscl_amd import optim


@pytest.mark.parametrize("bits", [32, 8])
def test_states_lie_like_their_parameter(bits):
    x = torch.randn(8, 5, 3, 3)
    ps = [torch.nn.Parameter(v) for v in (x.to(memory_format=torch.channels_last), torch.randn(6, 40).t(), torch.randn(1, 7, 1, 3).permute(2, 3, 0, 1), torch.randn(()))]
    src = torch.optim.AdamW(ps)
    for p in ps:
        p.grad = torch.randn_like(p)
    src.step()
    opt = optim.AdamW(ps, state_bits=bits)
    opt.load_state_dict(src.state_dict())
    for p in ps:
        st = opt.state[p]
        order = optim._order(p)
        assert all(optim._flat(st[k], order).is_contiguous() and st[k].shape == p.shape for k in ("exp_avg", "exp_avg_sq"))
    first = opt.state_dict()["state"]
    for i, p in enumerate(ps):
        want = src.state[p]["exp_avg"]
        assert torch.equal(first[i]["exp_avg"], want) if bits == 32 else (first[i]["exp_avg"] - want).abs().max() <= 2.0 ** -4 * want.abs().max()
    again = optim.AdamW(ps, state_bits=bits)
    again.load_state_dict(opt.state_dict())
    twin = copy.deepcopy(opt)
    for other in (again, twin):
        for i, st in other.state_dict()["state"].items():
            assert torch.equal(st["exp_avg"], first[i]["exp_avg"]) and torch.equal(st["exp_avg_sq"], first[i]["exp_avg_sq"])
