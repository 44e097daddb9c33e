"""A captured backward pass beside an eager graph of the same leaves is refused where the leaves lie behind other operators too, and
taken where no gradient goes to that graph's nodes."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def leaf(*shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", dtype=dtype, requires_grad=True)


def steps():
    import torchft_amd as t

    ids = torch.randint(0, 50, (70,), device="cuda")
    order = t.sort_by_expert(torch.randint(0, 4, (70, 2), device="cuda"), 4)
    low = torch.bfloat16
    return {
        "norm": (lambda x, w, r: sum(t.rms_norm(x.to(low), w * 2, r.to(low))), (leaf(70, 40), leaf(40), leaf(70, 40))),
        "dropout": (lambda x, r: t.dropout((x * 2).tanh(), 0.5, 1, residual=r.exp()), (leaf(70, 40), leaf(70, 40))),
        "embedding": (lambda table: t.embedding(ids, table.to(low)), (leaf(50, 40),)),
        "dispatch": (lambda x: t.dispatch(x.view(70, 40), order), (leaf(40 * 70),)),
        "combine": (lambda rows, w: t.combine(rows.to(low), order, w.softmax(1)), (leaf(140, 40), leaf(70, 2))),
        "run": (lambda table, w: t.dropout(t.rms_norm(t.embedding(ids, table.to(low)), w.to(low)), 0.5, 1), (leaf(50, 40), leaf(40))),
    }


@pytest.mark.parametrize("name", ["norm", "dropout", "embedding", "dispatch", "combine", "run"])
def test_leaves_behind_other_operators(name):
    run, leaves = steps()[name]
    eager = run(*leaves)
    dy = torch.randn_like(eager)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run(*leaves)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            torch.autograd.grad(y, leaves, dy)
        y = run(*leaves)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            y.backward(dy)
    assert all(v.grad is None for v in leaves)
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


def test_nodes_that_get_no_gradient():
    """Rows of an eager graph that lives, and a gradient of the weight alone."""
    import torchft_amd as t
    rows, w, dy = leaf(70, 40), leaf(40), torch.randn(70, 40, device="cuda")
    x = rows * 2
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(t.rms_norm(x, w), w, dy)
    for seed in range(3):
        dy.copy_(torch.randn(dy.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, torch.autograd.grad(t.rms_norm(x, w), w, dy)[0])
        torch.cuda.synchronize()
