"""4-bit matrices whose buffer is part of a larger one: what they hold, and products with them."""

import pytest
import torch

import mx_reference as ref
from test_gpu_mxfp4 import close, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("longer", [0, 3])
@pytest.mark.parametrize("shape", [(7, 200), (7, 700), (80, 512), (33, 1025)])
def test_part_of_a_larger_buffer(shape, longer):
    import torchft_amd as mx
    x = values(*shape, torch.float32, 100)
    m = mx.quantize_mxfp4(x.cuda())
    size = m.buffer.numel()
    for offset in (0, 16, 4096):
        large = torch.full((offset + size + longer,), 0x5a, dtype=torch.uint8, device="cuda")
        large[offset:offset + size] = m.buffer
        view = mx.MXFP4Tensor(large[offset:], m.shape, m.dtype)
        assert torch.equal(view.scales, m.scales) and torch.equal(view.codes, m.codes)
        assert torch.equal(view.scales.cpu(), ref.quantize(x)[1])
        assert torch.equal(view.dequantize(), m.dequantize())
        again = mx.MXFP4Tensor.from_blocks(view.codes, view.scales, shape[1], torch.float32)
        assert torch.equal(again.dequantize(), m.dequantize())
        t = values(5, shape[1], torch.float32, 101)
        av, bv = ref.quantize(t)[0], ref.quantize(x)[0]
        close(mx.linear_mxfp4(t.cuda(), view), av @ bv.t(), ref.product_bound(av, bv, torch.float32))
        close(mx.matmul_mxfp4(view, mx.quantize_mxfp4(t.cuda())), bv @ av.t(), ref.product_bound(bv, av, torch.float32))
