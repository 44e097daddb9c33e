"""The optimiser's state through state_dict and load_state_dict, without a GPU."""

import pytest
import torch

from torchft_amd import Muon

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(20, 30), (40, 10), (16, 16)]


def optimizer(dtype, seed):
    """One with momenta, as after a step (a step needs a GPU); the last weight has had no gradient yet."""
    g = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype)) for s in SHAPES]
    opt = Muon([{"params": ps[:1], "lr": 0.1}, {"params": ps[1:], "weight_decay": 0.3}])
    for p in ps[:2]:
        opt.state[p]["momentum"] = torch.randn(p.shape, generator=g) * 1e-3
    return ps, opt


@pytest.mark.parametrize("dtype", DTYPES)
def test_momentum_is_restored_in_float32(dtype):
    """Bit for bit, whatever the weights' type; options come along."""
    ps, opt = optimizer(dtype, 1)
    qs, again = optimizer(dtype, 2)
    again.load_state_dict(opt.state_dict())
    for p, q in zip(ps[:2], qs):
        m = again.state[q]["momentum"]
        assert m.dtype == torch.float32 and torch.equal(m, opt.state[p]["momentum"])
    assert "momentum" not in again.state[qs[2]]
    assert [g["lr"] for g in again.param_groups] == [0.1, 0.02]
    assert [g["weight_decay"] for g in again.param_groups] == [0.0, 0.3]
    saved = opt.state_dict()["state"]
    assert all(s["momentum"].dtype == torch.float32 for s in saved.values())


@pytest.mark.parametrize("dtype", DTYPES)
def test_momentum_of_another_type(dtype):
    """A momentum that was saved in 16 bits is taken as the numbers that it holds."""
    ps, opt = optimizer(dtype, 3)
    state = opt.state_dict()
    state["state"] = {k: {"momentum": v["momentum"].to(torch.bfloat16)} for k, v in state["state"].items()}
    qs, again = optimizer(dtype, 4)
    again.load_state_dict(state)
    for p, q in zip(ps[:2], qs):
        m = again.state[q]["momentum"]
        assert m.dtype == torch.float32 and torch.equal(m, opt.state[p]["momentum"].to(torch.bfloat16).float())


def test_hooks_of_the_caller():
    """A hook before loading may replace the state, one after it finds the momenta as they are; nothing is left behind."""
    ps, opt = optimizer(torch.bfloat16, 5)
    qs, again = optimizer(torch.bfloat16, 6)
    seen = []

    def doubled(_, state):
        state = dict(state)
        state["state"] = {k: {"momentum": 2 * v["momentum"]} for k, v in state["state"].items()}
        return state
    again.register_load_state_dict_pre_hook(doubled)
    again.register_load_state_dict_post_hook(lambda o: seen.append(o.state[qs[0]]["momentum"].clone()))
    for n in (1, 2):
        again.load_state_dict(opt.state_dict())
        assert torch.equal(again.state[qs[1]]["momentum"], 2 * opt.state[ps[1]]["momentum"])
        assert len(seen) == n and torch.equal(seen[-1], 2 * opt.state[ps[0]]["momentum"])


def test_a_state_that_does_not_fit():
    """Refused as by any optimiser, and loading works afterwards."""
    ps, opt = optimizer(torch.bfloat16, 7)
    other = Muon([torch.nn.Parameter(torch.zeros(3, 4, dtype=torch.bfloat16))])
    with pytest.raises(ValueError):
        other.load_state_dict(opt.state_dict())
    qs, again = optimizer(torch.bfloat16, 8)
    again.load_state_dict(opt.state_dict())
    assert torch.equal(again.state[qs[0]]["momentum"], opt.state[ps[0]]["momentum"])
