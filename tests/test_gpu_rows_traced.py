"""A backward pass of the row operators under a trace is refused like a forward pass; a mode that looks on changes nothing."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

pytestmark = pytest.mark.gpu


def steps():
    import torchft_amd as t

    def leaf(*shape):
        return torch.randn(*shape, device="cuda", requires_grad=True)

    order = t.sort_by_expert(torch.randint(0, 4, (70, 2), device="cuda"), 4)
    ids = torch.randint(0, 50, (70,), device="cuda")
    return {
        "norm": (lambda x, w, r: sum(t.rms_norm(x, w, r)), (leaf(70, 40), leaf(40), leaf(70, 40))),
        "dropout": (lambda x, r: t.dropout(x, 0.5, 1, residual=r), (leaf(70, 40), leaf(70, 40))),
        "embedding": (lambda table: t.embedding(ids, table), (leaf(50, 40),)),
        "dispatch": (lambda x: t.dispatch(x, order), (leaf(70, 40),)),
        "combine": (lambda rows, w: t.combine(rows, order, w), (leaf(140, 40), leaf(70, 2))),
    }


@pytest.mark.parametrize("name", ["norm", "dropout", "embedding", "dispatch", "combine"])
def test_backward(name):
    from torch.utils.flop_counter import FlopCounterMode
    run, leaves = steps()[name]
    y = run(*leaves)
    dy = torch.randn_like(y)
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    with pytest.raises(RuntimeError, match="trace of the call"):
        make_fx(lambda g: torch.autograd.grad(y, leaves, g, retain_graph=True))(dy)
    with FlopCounterMode(display=False):
        got = (run(*leaves), *torch.autograd.grad(y, leaves, dy))
    assert all(torch.equal(a, b) for a, b in zip(got, (y, *want)))
