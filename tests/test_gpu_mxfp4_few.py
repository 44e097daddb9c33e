"""Layers whose weight is kept in 4 bits, from one row of x to more than the kernel of few rows takes."""

import pytest
import torch

import mx_reference as ref
from test_gpu_mxfp4 import DTYPES, close, operand, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mx():
    import torchft_amd
    return torchft_amd


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    """Whole calls in the native helper, and the way round it."""
    import torchft_amd.mxfp4 as m
    m._ready(torch.device("cuda", torch.cuda.current_device()))
    if request.param == "python":
        monkeypatch.setattr(m, "_native", None)
        monkeypatch.setattr(m, "_ready", lambda device: None)
    return request.param


# rows of x, of the weight, columns: either side of 16, 32 and 64 rows, of panels of 256 columns, of what the
# kernel quantises itself, and of the weights that are too large for it
LAYERS = [(1, 1, 1), (1, 33, 31), (2, 500, 257), (3, 17, 4100), (7, 90, 512), (15, 1030, 255), (16, 64, 1000), (17, 64, 1000),
          (31, 31, 2049), (32, 200, 256), (33, 100, 300), (48, 15, 1536), (63, 300, 100), (64, 17, 1540), (64, 11000, 64),
          (65, 100, 300), (1, 20000, 96), (4, 130, 33000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", LAYERS)
def test_layer(mx, path, shape, dtype):
    m, n, k = shape
    x = values(m, k, dtype, 21)
    w, wv = operand(mx, n, k, torch.float32, 22)
    xv = ref.quantize(x)[0]
    y = mx.linear_mxfp4(x.cuda(), w)
    assert y.dtype == dtype
    close(y, xv @ wv.t(), ref.product_bound(xv, wv, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 5, 20, 64, 70])
def test_rows_at_any_address(mx, path, rows, dtype):
    """Rows of x that start at any element, lie apart, or are every second column of another matrix."""
    n, k = 70, 333
    big = values(2 * rows + 1, 2 * k + 9, dtype, 23)
    gpu = big.cuda()
    w, wv = operand(mx, n, k, torch.float32, 24)
    for at in ((slice(0, rows), slice(3, 3 + k)), (slice(1, 2 * rows, 2), slice(4, 4 + k)), (slice(0, rows), slice(1, 1 + 2 * k, 2)),
               (slice(rows, 2 * rows), slice(8, 8 + k))):
        xv = ref.quantize(big[at])[0]
        close(mx.linear_mxfp4(gpu[at], w), xv @ wv.t(), ref.product_bound(xv, wv, dtype))
    line = gpu[:1, 5:5 + k].expand(rows, k)
    xv = ref.quantize(big[:1, 5:5 + k].expand(rows, k))[0]
    close(mx.linear_mxfp4(line, w), xv @ wv.t(), ref.product_bound(xv, wv, dtype))


@pytest.mark.parametrize("rows", [1, 16, 17, 64, 65])
def test_corners(mx, path, rows):
    """A NaN or an infinity makes its row's results NaN, and no other's; zeros give zeros; scales far apart."""
    n, k = 40, 600
    x = values(rows, k, torch.float32, 25)
    x[rows - 1] = 0.0
    x[rows // 2, 299] = float("nan") if rows > 1 else 1.0
    x[0] *= 2.0 ** 100
    wide = values(n, k, torch.float32, 26)
    wide[7] *= 2.0 ** -110
    wide[9, 598] = float("inf")
    w, wv = mx.quantize_mxfp4(wide.cuda()), ref.quantize(wide)[0]
    y = mx.linear_mxfp4(x.cuda(), w).cpu()
    xv = ref.quantize(x)[0]
    nan = torch.isnan(xv).any(1)[:, None] | torch.isnan(wv).any(1)[None]
    assert torch.equal(torch.isnan(y), nan)
    xz, wz = torch.nan_to_num(xv), torch.nan_to_num(wv)
    off = (y.double() - xz @ wz.t()).abs() - ref.product_bound(xz, wz, torch.float32)
    assert off[~nan].max().item() <= 0


def test_paths_agree(mx, monkeypatch):
    """A layer is the product of the quantised matrices, whichever way the call goes; on another stream too."""
    import torchft_amd.mxfp4 as m
    x, w = values(64, 520, torch.bfloat16, 27).cuda(), mx.quantize_mxfp4(values(90, 520, torch.bfloat16, 28).cuda())
    torch.cuda.synchronize()
    for rows in (1, 3, 16, 40, 64):
        here = mx.linear_mxfp4(x[:rows], w)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            there = mx.linear_mxfp4(x[:rows], w)
        side.synchronize()
        assert torch.equal(here, there)
        with monkeypatch.context() as without:
            without.setattr(m, "_native", None)
            without.setattr(m, "_ready", lambda device: None)
            assert torch.equal(here, mx.linear_mxfp4(x[:rows], w))
            a = mx.quantize_mxfp4(x[:rows])
            assert torch.equal(a.dequantize(), mx.MXFP4Tensor(a.buffer, a.shape, a.dtype).dequantize())


def test_graph_of_one_token(mx):
    """A captured layer of one row gives the eager bytes on every replay."""
    xs = values(4, 700, torch.bfloat16, 29).cuda()
    w = mx.quantize_mxfp4(values(130, 700, torch.bfloat16, 30).cuda())
    want = [mx.linear_mxfp4(xs[i:i + 1], w) for i in range(4)]
    static = xs[:1].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mx.linear_mxfp4(static, w)
    for i in (0, 1, 2, 3, 1):
        static.copy_(xs[i:i + 1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
        assert torch.equal(mx.linear_mxfp4(xs[i:i + 1], w), want[i])


def test_buffers_that_do_not_hold_their_matrix(mx):
    x = torch.ones(4, 600, device="cuda")
    whole = mx.quantize_mxfp4(x)
    for buffer in (whole.buffer[:-8], whole.buffer[16:], whole.buffer.view(torch.int32), whole.buffer[::2],
                   torch.cat([whole.buffer, whole.buffer])[8:]):
        bad = mx.MXFP4Tensor(buffer, whole.shape, whole.dtype)
        for call in (lambda: mx.linear_mxfp4(x, bad), lambda: mx.matmul_mxfp4(whole, bad), lambda: mx.matmul_mxfp4(bad, whole), bad.dequantize):
            with pytest.raises(AssertionError, match="buffer"):
                call()
