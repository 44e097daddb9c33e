"""The row operators in a row, as examples/experts.py uses them: its gradients against 64 bits, its run, its serving."""

import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

SIZES = dict(width=72, hidden=40, vocab=101, layers=2, experts=5)


@pytest.fixture(scope="module")
def example():
    import experts
    return experts


def plain(p, ids, choices, keep, factor):
    """The model in 64 bits; keep: what every layer's dropout leaves."""
    h = p["table"][ids] * p["table"].shape[1] ** 0.5
    routes = []

    def norm(h, w):
        return h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-6) * w

    for i in range(SIZES["layers"]):
        y = norm(h, p[f"{i}.norm"])
        best = (y @ p[f"{i}.router"].t()).topk(choices, dim=1)
        routes.append(best.indices)
        weights = best.values.softmax(1)
        out = torch.zeros_like(y)
        for s in range(choices):
            for e in range(SIZES["experts"]):
                some = (best.indices[:, s] == e).nonzero()[:, 0]
                z = torch.nn.functional.silu(y[some] @ p[f"{i}.{e}.up"].t()) @ p[f"{i}.{e}.down"].t()
                out = out.index_add(0, some, z * weights[some, s, None])
        h = h + torch.where(keep[i], out * factor, 0.0)
    return norm(h, p["norm"]) @ p["head"].t(), routes


def test_gradients(example):
    """In fp32 with plain linear layers: every gradient, through both layers, within 1e-4 of its norm.  (The longest sums
    have 101 terms and a dozen operators follow each other: about 101 2^-24 a step, 1e-4 in all with its condition.)"""
    import rows_reference as ref
    tokens, choices, rate, seed = 64, 2, 0.25, 9
    p = example.parameters(seed=3, device="cuda", **SIZES)
    for w in p.values():
        w.requires_grad_()
    ids = torch.randint(0, SIZES["vocab"], (tokens,), generator=torch.Generator().manual_seed(1))
    dy = torch.randn(tokens, SIZES["vocab"], generator=torch.Generator().manual_seed(2))
    logits = example.forward(p, ids.cuda(), SIZES["layers"], SIZES["experts"], choices, rate, seed, linear=lambda x, w: x @ w.t(), dtype=torch.float32)
    names = list(p)
    got = torch.autograd.grad(logits, [p[n] for n in names], dy.cuda(), allow_unused=True)
    wide = {n: w.detach().cpu().double().requires_grad_() for n, w in p.items()}
    keep = [(ref.bits16(seed, i, tokens * SIZES["width"]) >= 16384).view(tokens, -1) for i in range(SIZES["layers"])]
    want_logits, _ = plain(wide, ids, choices, keep, 65536 / (65536 - 16384))
    assert (logits.detach().cpu().double() - want_logits).norm() <= 1e-4 * want_logits.norm()
    want = torch.autograd.grad(want_logits, [wide[n] for n in names], dy.double(), allow_unused=True)
    for n, a, b in zip(names, got, want):
        if b is None or not b.any():
            assert a is None or not a.any(), n
        else:
            assert (a.cpu().double() - b).norm() <= 1e-4 * b.norm(), n


def test_run(example):
    """Two replicas take the same steps; the trained model answers."""
    sizes = dict(SIZES, vocab=128, width=64, hidden=96)
    results = example.run(2, steps=3, tokens=128, choices=2, rate=0.1, **sizes)
    (a, losses), (b, others) = results
    assert all(torch.equal(a[n], b[n]) for n in a)
    assert all(torch.isfinite(torch.tensor(x)).all() for x in (losses, others))
    first = example.parameters(seed=1, device="cuda", **sizes)
    assert all(not torch.equal(a[n], first[n]) for n in ("table", "head", "norm", "0.norm", "0.router"))
    logits = example.serve(a, torch.arange(1, device="cuda"), sizes["layers"], sizes["experts"], 2)
    assert logits.shape == (1, 128) and torch.isfinite(logits).all()
    assert example.serve(a, torch.arange(7, device="cuda"), sizes["layers"], sizes["experts"], 2).shape == (7, 128)
