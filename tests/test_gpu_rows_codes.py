"""Codes of a norm in 8 bits, of rows and weights of whole numbers, against whole numbers.

A code is the number of e4m3 nearest to 448 h w / max |h w|, the even one of two that are as near.  With whole h and w its
quotient lies beside or on a border where whole products say so: no rounding is in the way, and no code may differ.
"""

import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu

BF, HALF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def t():
    import torchft_amd
    return torchft_amd


def codes_of(h, w):
    """The codes of whole numbers h (rows) and w (a weight for every column), int64; products below 2^43."""
    p = (h * w).abs()
    most = p.amax(1, keepdim=True)
    # 1024 times the borders between the numbers of e4m3 that are not negative, whole numbers
    values = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double() * 1024
    borders = ((values[1:] + values[:-1]) / 2).long().tolist()
    code = torch.zeros_like(p)
    for j, border in enumerate(borders):  # between code j and j + 1
        quotient, at = p * (448 * 1024), most * border
        code += (quotient > at) | ((quotient == at) & (j % 2 == 1))
    return code.to(torch.uint8) | torch.where(h * w < 0, 128, 0).to(torch.uint8)


def whole(shape, bits, more, g):
    """Whole numbers of up to `bits` bits, times powers of two up to 2^more."""
    return torch.randint(1 - 2 ** bits, 2 ** bits, shape, generator=g) << torch.randint(0, more + 1, shape, generator=g)


# of the rows and of the weight: type, bits, powers of two; narrow numbers have many quotients on borders
NUMBERS = [(BF, 8, 9, BF, 8, 9), (BF, 4, 0, None, 0, 0), (BF, 7, 0, BF, 3, 0), (BF, 8, 4, F32, 24, 0), (BF, 6, 0, F32, 7, 0),
           (HALF, 11, 4, HALF, 11, 4), (HALF, 6, 0, None, 0, 0), (HALF, 11, 2, F32, 24, 0), (F32, 21, 0, F32, 21, 0), (F32, 7, 0, F32, 4, 0),
           (F32, 24, 0, None, 0, 0), (F32, 10, 0, None, 0, 0)]
SHAPES = [(900, 3), (400, 40), (200, 130), (100, 333), (70, 600), (50, 1030), (30, 2900), (20, 4480), (12, 8200), (6, 16390), (4, 33001)]


@pytest.mark.parametrize("numbers", NUMBERS, ids=lambda n: f"{str(n[0])[6:]}-{n[1]}-{str(n[3])[6:]}-{n[4]}")
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_nearest(t, shape, numbers):
    dtype, bits, more, weight_dtype, weight_bits, weight_more = numbers
    g = torch.Generator().manual_seed(shape[1] + bits)
    h = whole(shape, bits, more, g)
    w = whole((shape[1],), weight_bits, weight_more, g) if weight_dtype else torch.ones(shape[1], dtype=torch.int64)
    h[1] = 0
    h[:, 0], w[0] = 2 ** bits - 1, 2 ** max(1, weight_bits) - 1  # no row but that is all zeros
    h[1] = 0
    x, weight = h.to(dtype), w.to(weight_dtype) if weight_dtype else None
    assert torch.equal(x.long(), h) and (weight is None or torch.equal(weight.long(), w))
    on = weight.cuda() if weight_dtype else None
    want = codes_of(h, w)
    want[1] = 0
    residual = whole(shape, max(1, bits - 1), 0, g).to(dtype)  # x - residual may be rounded, and then has another h
    got = t.rms_norm_fp8(x.cuda(), on)
    same = (x.float() - residual.float()).to(dtype)
    with_residual, kept = t.rms_norm_fp8(same.cuda(), on, residual.cuda())
    back = kept.cpu().long()
    want_back = codes_of(back, w)
    for rows, codes, h_ in ((got, want, h), (with_residual, want_back, back)):
        own = rows.codes.cpu().view(torch.uint8)
        some = h_.any(1)  # a row of zeros has codes of zeros, whose sign does not matter
        zero = (h_ * w) == 0
        assert torch.equal(torch.where(zero, own & 127, own)[some], torch.where(zero, 0, codes)[some]), \
            f"{int((torch.where(zero, own & 127, own) != torch.where(zero, 0, codes))[some].sum())} codes of {own.numel()} are not the nearest"
        assert not (own[~some] & 127).any()
        y = ref.norm(h_.to(torch.float64).to(dtype), weight, None, 1e-6)[0]
        scale = y.abs().amax(1, keepdim=True)[some] / 448
        assert ((rows.scales.cpu().double()[some] - scale).abs() <= scale * (shape[1] / 2 + 16) * ref.U).all()


def test_wide_ranges(t):
    """Products beyond fp32's range whose y is within it, and rows of very small numbers."""
    g = torch.Generator().manual_seed(5)
    for dtype in (BF, F32):
        h, w = whole((9, 700), 7, 0, g), whole((700,), 5, 0, g)
        h[:, 0], w[0] = 127, 31
        want = codes_of(h, w)
        zero = h * w == 0
        for a, b in ((2.0 ** 45, 2.0 ** 100), (2.0 ** -50, 2.0 ** 100), (2.0 ** 45, 2.0 ** -90), (2.0 ** -50, 2.0 ** -60)):
            rows = t.rms_norm_fp8((h.double() * a).to(dtype).cuda(), (w.double() * b).to(dtype).cuda(), eps=0.0)
            own = rows.codes.cpu().view(torch.uint8)
            assert torch.equal(torch.where(zero, own & 127, own), torch.where(zero, 0, want))
