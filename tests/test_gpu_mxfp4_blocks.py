"""Codes and scales of a checkpoint in any order of storage."""

import pytest
import torch

import mx_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [32, 100, 256, 512, 700, 1024])
def test_from_blocks_of_any_order(cols):
    """Stored block by block, as a part of a larger matrix along either axis, every second row, one row for all."""
    import torchft_amd as mx
    rows, blocks = 10, -(-cols // 32)
    g = torch.Generator().manual_seed(200 + cols)
    codes = torch.randint(0, 256, (rows, blocks, 16), generator=g).to(torch.uint8).cuda()
    scales = torch.randint(100, 140, (rows, blocks), generator=g).to(torch.uint8).cuda()

    def stored(t, order):
        return t.permute(order).contiguous().permute([order.index(i) for i in range(t.dim())])

    def part(t):
        large = torch.full((2 * rows + 3, blocks + 5, *t.shape[2:]), 0x77, dtype=torch.uint8, device="cuda")
        view = large[3::2, 2:2 + blocks]
        view.copy_(t)
        return view
    want = mx.MXFP4Tensor.from_blocks(codes, scales, cols)
    each = torch.stack([codes & 15, codes >> 4], -1).view(rows, blocks, 32).long().cpu()
    values = torch.where(each > 7, -1.0, 1.0) * ref.GRID[each % 8] * torch.exp2(scales.cpu().double() - 127)[..., None]
    assert torch.equal(want.dequantize(torch.float32).cpu().double(), values.view(rows, -1)[:, :cols])
    for c, s in ((stored(codes, [1, 0, 2]), stored(scales, [1, 0])), (stored(codes, [2, 0, 1]), scales), (stored(codes, [2, 1, 0]), stored(scales, [1, 0])),
                 (part(codes), part(scales)), (codes, stored(scales, [1, 0]))):
        assert torch.equal(c, codes) and torch.equal(s, scales)
        got = mx.MXFP4Tensor.from_blocks(c, s, cols)
        assert torch.equal(got.scales, want.scales) and torch.equal(got.codes, want.codes)
        assert torch.equal(got.dequantize(), want.dequantize())
    line = mx.MXFP4Tensor.from_blocks(codes[:1].expand(rows, -1, -1), scales[:1].expand(rows, -1), cols)
    assert torch.equal(line.dequantize(), want.dequantize()[:1].expand(rows, -1))
