"""4-bit matrices whose buffer is part of a larger one, without a GPU."""

import pytest
import torch

from torchft_amd import MXFP4Tensor, _lib

SHAPES = [(1, 1), (3, 33), (4, 256), (3, 512), (5, 700), (6, 1000), (1, 2049)]


@pytest.mark.parametrize("longer", [0, 3, 64])
@pytest.mark.parametrize("offset", [0, 8, 16, 3, 4096])
@pytest.mark.parametrize("shape", SHAPES)
def test_codes_and_scales(shape, offset, longer):
    """Those of the bytes from where the buffer starts, one panel or several, an even or odd number of rows."""
    rows, cols = shape
    size = _lib.load().tftq_mx_bytes(rows, cols)
    g = torch.Generator().manual_seed(size + offset)
    whole = torch.randint(0, 256, (offset + size + longer,), generator=g).to(torch.uint8)
    m = MXFP4Tensor(whole[offset:], shape, torch.float32)
    own = whole[offset:offset + size]
    panels, even = -(-cols // 256), rows + rows % 2
    codes, scales = own[:panels * rows * 128].tolist(), own[panels * rows * 128:].tolist()
    blocks = -(-cols // 32)
    want_codes = [[codes[(b // 8 * rows + r) * 128 + b % 8 * 16:][:16] for b in range(blocks)] for r in range(rows)]
    want_scales = [[scales[(b // 8 * even + r) * 8 + b % 8] for b in range(blocks)] for r in range(rows)]
    assert m.codes.tolist() == want_codes
    assert m.scales.tolist() == want_scales
