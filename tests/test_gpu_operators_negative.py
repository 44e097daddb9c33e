"""Tensors that torch holds as the negative of what lies in memory (imaginary parts of conjugates)."""

import pytest
import torch

from test_gpu_orthogonal import gradient

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ta():
    import torchft_amd
    return torchft_amd


def negative(t):
    """t as a view of -t: stored by rows, or with gaps where it has one column."""
    if t.shape[1] == 1:
        view = torch.complex(torch.zeros_like(t), -t).conj().imag
        view = view if view.is_neg() else torch._neg_view(-t)
    else:
        view = torch._neg_view(-t)
    assert view.is_neg() and torch.equal(view, t)
    return view


@pytest.mark.parametrize("shape", [(70, 1), (70, 96), (3, 500)])
def test_mxfp4(ta, shape):
    x = gradient(*shape, torch.float32, 190).cuda()
    w = gradient(40, shape[1], torch.float32, 191).cuda()
    for got, want in zip(ta.quantize_mxfp4_both(negative(x)), ta.quantize_mxfp4_both(x)):
        assert torch.equal(got.dequantize(), want.dequantize())
    kept = ta.quantize_mxfp4(w)
    assert torch.equal(ta.linear_mxfp4(negative(x), kept), ta.linear_mxfp4(x, kept))
    assert torch.equal(ta.linear_mxfp4(negative(x), negative(w)), ta.linear_mxfp4(x, w))
    results = []
    for f in (negative, lambda t: t):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        ta.linear_mxfp4(f(a) if a.shape[1] > 1 else a, b).backward(f(gradient(shape[0], 40, torch.float32, 192).cuda()))
        results.append((a.grad, b.grad))
    assert all(torch.equal(g, h) for g, h in zip(*results))


@pytest.mark.parametrize("shape", [(70, 1), (70, 96), (3, 500)])
def test_orthogonal(ta, shape):
    x = gradient(*shape, torch.float32, 193).cuda()
    assert torch.equal(ta.orthogonalize(negative(x)), ta.orthogonalize(x))
    w, m = gradient(*shape, torch.float32, 194).cuda(), gradient(*shape, torch.float32, 195).cuda()
    want = [t.clone() for t in (w, m)]
    ta.muon_([want[0]], [x], [want[1]], lr=0.1, weight_decay=0.1)
    for which in range(3):
        args = [t.clone() for t in (w, x, m)]
        args[which] = negative(args[which])
        ta.muon_([args[0]], [args[1]], [args[2]], lr=0.1, weight_decay=0.1)
        assert torch.equal(args[0], want[0]) and torch.equal(args[2], want[1])
