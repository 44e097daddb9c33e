"""4-bit microscaled matrices, host side: sizes and refusals of the C entries, without a GPU."""

import ctypes

import pytest
import torch

from torchft_amd import MXFP4Tensor, _lib

F32, BF16 = 0, 2


def test_bytes():
    L = _lib.load()
    for rows, cols in ((1, 1), (1, 256), (3, 257), (4096, 14336), (333, 1001), (2 ** 20, 2 ** 20)):
        panels, even = -(-cols // 256), rows + rows % 2
        assert L.tftq_mx_bytes(rows, cols) == panels * (rows * 128 + even * 8)
    assert L.tftq_mx_bytes(0, 7) == 0 and L.tftq_mx_bytes(7, 0) == 0
    for rows, cols in ((-1, 4), (4, -1), (2 ** 31, 4), (4, 2 ** 31)):
        assert L.tftq_mx_bytes(rows, cols) == -3


def test_entries_refuse_before_they_launch():
    """Every call below returns before it touches a device (there is none here)."""
    L = _lib.load()
    buf = (ctypes.c_uint8 * 4096)()
    at = (ctypes.addressof(buf) + 15) & ~15
    assert L.tftq_mx_quantize(3, at, 2, 32, 32, at, None, -1, None) == -2
    assert L.tftq_mx_quantize(F32, at, -1, 32, 32, at, None, -1, None) == -3
    assert L.tftq_mx_quantize(F32, at, 2, 2 ** 31, 2 ** 31, at, None, -1, None) == -3
    assert L.tftq_mx_quantize(F32, at, 2, 32, 32, None, None, -1, None) == -1
    assert L.tftq_mx_quantize(F32, None, 2, 32, 32, at, None, -1, None) == -1
    assert L.tftq_mx_quantize(F32, at, 2, 32, 31, at, None, -1, None) == -1
    assert L.tftq_mx_quantize(F32, at, 2, 32, 32, at + 8, None, -1, None) == -1
    assert L.tftq_mx_quantize(F32, None, 0, 32, 32, None, None, -1, None) == 0
    assert L.tftq_mx_dequantize(9, at, 2, 32, at, 32, -1, None) == -2
    assert L.tftq_mx_dequantize(BF16, at, 2, 32, at, 16, -1, None) == -1
    assert L.tftq_mx_dequantize(BF16, at + 4, 2, 32, at, 32, -1, None) == -1
    assert L.tftq_mx_dequantize(BF16, None, 0, 32, None, 32, -1, None) == 0
    assert L.tftq_mx_product(9, at, 2, at, 2, 32, at, 2, -1, None) == -2
    assert L.tftq_mx_product(F32, at, 2, at, -2, 32, at, 2, -1, None) == -3
    assert L.tftq_mx_product(F32, at, 2, at, 2, 32, at, 1, -1, None) == -1
    assert L.tftq_mx_product(F32, None, 2, at, 2, 32, at, 2, -1, None) == -1
    assert L.tftq_mx_product(F32, at, 2, at, 2, 32, None, 2, -1, None) == -1
    assert L.tftq_mx_product(F32, None, 0, None, 2, 32, None, 2, -1, None) == 0


def test_blocks_that_do_not_fit():
    codes, scales = torch.zeros(4, 2, 16, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    for bad in ((codes.int(), scales, 64), (codes, scales, 65), (codes, scales, 32), (codes[:, :1], scales, 64),
                (codes[..., :15], scales, 64)):
        with pytest.raises(AssertionError):
            MXFP4Tensor.from_blocks(*bad)
    with pytest.raises(AssertionError, match="GPU"):
        MXFP4Tensor.from_blocks(codes, scales, 64)


def test_linear_refuses_before_it_launches():
    L = _lib.load()
    buf = (ctypes.c_uint8 * 65536)()
    at = (ctypes.addressof(buf) + 15) & ~15

    def size(dtype=BF16, x=at, m=100, stride=512, n=40, k=512):
        return L.tftq_mx_linear_workspace(dtype, x, m, stride, n, k)

    def call(dtype=BF16, x=at, m=100, stride=512, b=at, n=40, k=512, out=at, out_stride=40, workspace=at, bytes=1 << 40):
        return L.tftq_mx_linear(dtype, x, m, stride, b, n, k, out, out_stride, workspace, bytes, -1, None)
    assert size() == L.tftq_mx_bytes(100, 512)  # x, quantised in a launch of its own
    assert size(m=1) == 0 and size(m=0) == 0 and size(k=0) == 0
    assert size(dtype=7) == call(dtype=7) == -2
    for bad in (dict(m=-1), dict(n=-1), dict(k=-1), dict(m=2 ** 31), dict(n=2 ** 31), dict(k=2 ** 31)):
        assert size(**bad) == call(**bad) == -3
    assert call(m=0, x=None) == 0 and call(n=0, b=None) == 0
    assert call(x=None) == call(b=None) == call(out=None) == call(b=at + 8) == -1
    assert call(stride=511) == call(out_stride=39) == -1
    assert call(bytes=L.tftq_mx_bytes(100, 512) - 1) == -4
    assert call(workspace=None) == call(workspace=at + 8) == -1
