"""What the optimiser takes as its parameters, without a GPU."""

import pytest
import torch

from torchft_amd import Muon


def matrix():
    return torch.nn.Parameter(torch.zeros(4, 6))


def test_a_group_of_vectors_is_refused():
    """At once, by either way in, and the optimiser is left as it was."""
    vector = torch.nn.Parameter(torch.zeros(4))
    for bad in ([vector], [matrix(), vector], [{"params": [matrix()]}, {"params": [vector]}]):
        with pytest.raises(AssertionError, match="2D"):
            Muon(bad)
    opt = Muon([matrix()])
    for bad in ({"params": vector}, {"params": [matrix(), vector]}, {"params": iter([vector])}, {"params": [("bias", vector)]}):
        with pytest.raises((AssertionError, ValueError)):
            opt.add_param_group(bad)
        assert len(opt.param_groups) == 1
    with pytest.raises(AssertionError, match="2D"):
        opt.add_param_group({"params": [vector]})


def test_a_group_of_matrices_is_taken():
    opt = Muon([matrix()], lr=0.1)
    opt.add_param_group({"params": (p for p in [matrix(), matrix()]), "lr": 0.3})
    assert [len(g["params"]) for g in opt.param_groups] == [1, 2] and [g["lr"] for g in opt.param_groups] == [0.1, 0.3]


def test_options_out_of_range():
    """Of a group as of the optimiser, before anything is added."""
    for name, value in (("lr", -0.1), ("weight_decay", -1.0), ("momentum", 1.0), ("momentum", -0.1)):
        with pytest.raises(AssertionError, match="out of range"):
            Muon([matrix()], **{"lr": 0.1, name: value})
        opt = Muon([matrix()])
        with pytest.raises(AssertionError, match="out of range"):
            opt.add_param_group({"params": [matrix()], name: value})
        assert len(opt.param_groups) == 1
