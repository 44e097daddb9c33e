"""A matrix of more rows than one launch takes: quantised, read back and multiplied."""

import pytest
import torch

pytestmark = pytest.mark.gpu

PERIOD = 4096


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_rows_than_a_launch(dtype):
    """2^28 rows and more of a few columns, the same 4096 over and over but for the last: 40 GB of codes."""
    import torchft_amd as mx
    rows, cols = (1 << 28) + PERIOD + 3, 5
    if torch.cuda.mem_get_info()[1] < 150 << 30:
        pytest.skip("needs 150 GB of device memory")
    g = torch.Generator("cuda").manual_seed(140)
    part = torch.randn(PERIOD, cols, device="cuda", generator=g).to(dtype)
    x = part.repeat(-(-rows // PERIOD), 1)[:rows]
    x[-1] *= 2
    w = mx.quantize_mxfp4(torch.randn(20, cols, device="cuda", generator=g))
    small = mx.quantize_mxfp4(part)
    values, products = small.dequantize(), mx.matmul_mxfp4(small, w)

    def check(got, want):
        whole = rows // PERIOD * PERIOD
        assert (got[:whole].view(-1, PERIOD, want.shape[1]) == want).all()
        assert torch.equal(got[whole:-1], want[:rows - whole - 1]) and torch.equal(got[-1], 2 * want[rows - whole - 1])
    m = mx.quantize_mxfp4(x)
    check(m.dequantize(), values)
    check(mx.matmul_mxfp4(m, w), products)
    del m
    check(mx.linear_mxfp4(x, w), products)
    t = mx.quantize_mxfp4(x, 0)  # [cols, rows]
    assert torch.equal(t.dequantize()[:, :PERIOD], mx.quantize_mxfp4(part, 0).dequantize())
