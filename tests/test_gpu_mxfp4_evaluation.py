"""Layers on ordinary weights without gradients: the bytes of those with, and no more work than they need."""

import pytest
import torch

import mx_reference as ref
from test_gpu_mxfp4 import DTYPES, close, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def m():
    import torchft_amd.mxfp4 as m
    m._ready(torch.device("cuda", torch.cuda.current_device()))
    return m


@pytest.fixture
def quantised(m, monkeypatch):
    """The directions that are asked for along either axis."""
    calls, quantize = [], m._quantize

    def counted(x, by_rows, by_columns):
        calls.append((by_rows, by_columns))
        return quantize(x, by_rows, by_columns)
    monkeypatch.setattr(m, "_quantize", counted)
    return calls


SHAPES = [(1, 70, 333), (16, 64, 1000), (40, 100, 64), (64, 11000, 64), (130, 257, 512), (2000, 300, 700)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_without_gradients(m, quantised, shape, dtype):
    t, n, k = shape
    x, w = values(t, k, dtype, 120), values(n, k, torch.float32, 121)
    gx, gw = x.cuda().requires_grad_(), torch.nn.Parameter(w.cuda())
    with torch.no_grad():
        y = m.linear_mxfp4(gx, gw)
    with torch.inference_mode():
        again = m.linear_mxfp4(gx, gw)
    plain = m.linear_mxfp4(gx.detach(), gw.detach())
    assert quantised == [(True, False)] * 3  # the weight, along its rows
    assert torch.equal(y, again) and torch.equal(y, plain) and not y.requires_grad and y.dtype == dtype
    assert torch.equal(y, m.linear_mxfp4(gx.detach(), m.quantize_mxfp4(gw)))
    a, b = ref.quantize(x)[0], ref.quantize(w)[0]
    close(y, a @ b.t(), ref.product_bound(a, b, dtype))
    close(m.linear_mxfp4(gx, gw).detach(), a @ b.t(), ref.product_bound(a, b, dtype))


def test_shapes_without_gradients(m):
    w = torch.nn.Parameter(values(50, 100, torch.bfloat16, 122).cuda())
    x = values(24, 100, torch.bfloat16, 123).cuda()
    with torch.no_grad():
        flat = m.linear_mxfp4(x, w)
        assert torch.equal(m.linear_mxfp4(x.view(2, 3, 4, 100), w), flat.view(2, 3, 4, 50))
        assert torch.equal(m.linear_mxfp4(x[0], w), m.linear_mxfp4(x[:1], w)[0])
        assert torch.equal(m.linear_mxfp4(x.t().contiguous().t(), w), flat)
        for t, n, k in ((0, 5, 7), (5, 0, 7), (5, 7, 0)):
            y = m.linear_mxfp4(torch.zeros(t, k, device="cuda"), torch.nn.Parameter(torch.zeros(n, k, device="cuda")))
            assert y.shape == (t, n) and not y.any()


def test_one_gradient_of_two(m, quantised):
    """Frozen inputs of a training step: nothing is quantised along an axis that no gradient contracts."""
    x, w = values(80, 300, torch.bfloat16, 124).cuda(), values(40, 300, torch.bfloat16, 125).cuda()
    m.linear_mxfp4(x.clone().requires_grad_(), w).sum().backward()
    assert quantised == [(True, True), (True, False)]  # w; dy along n
    del quantised[:]
    m.linear_mxfp4(x, w.clone().requires_grad_()).sum().backward()
    assert quantised == [(True, False), (True, True), (False, True)]  # w; x; dy along the tokens
