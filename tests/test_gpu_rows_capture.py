"""A backward pass captured beside an eager graph of the same leaves is refused, and captured once that is gone."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def steps():
    import torchft_amd as t

    def leaf(*shape):
        return torch.randn(*shape, device="cuda", requires_grad=True)

    ids = torch.randint(0, 50, (70,), device="cuda")
    chosen = torch.randint(0, 4, (70, 2), device="cuda")
    order = t.sort_by_expert(chosen, 4)
    return {
        "norm": (lambda x, w, r: sum(t.rms_norm(x, w, r)), (leaf(70, 40), leaf(40), leaf(70, 40))),
        "dropout": (lambda x, r: t.dropout(x, 0.5, 1, residual=r), (leaf(70, 40), leaf(70, 40))),
        "embedding": (lambda table: t.embedding(ids, table), (leaf(50, 40),)),
        "dispatch": (lambda x: t.dispatch(x, order), (leaf(70, 40),)),
        "combine": (lambda rows, w: t.combine(rows, order, w), (leaf(140, 40), leaf(70, 2))),
    }


@pytest.mark.parametrize("name", ["norm", "dropout", "embedding", "dispatch", "combine"])
def test_eager_graph_lives(name):
    run, leaves = steps()[name]
    eager = run(*leaves)
    dy = torch.randn_like(eager)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run(*leaves)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            torch.autograd.grad(y, leaves, dy)
    torch.autograd.grad(eager, leaves, dy)  # the process and the eager graph are well
    del eager, y
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(run(*leaves), leaves, dy)
    for seed in range(3):
        dy.copy_(torch.randn(dy.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        want = torch.autograd.grad(run(*leaves), leaves, dy)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        torch.cuda.synchronize()
