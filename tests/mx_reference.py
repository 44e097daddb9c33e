"""4-bit microscaled matrices in 64 bits on the CPU, straight from the formats' definition."""

import torch

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def quantize(x):
    """(values, scale bytes) of a matrix's rows in blocks of 32: values [rows, cols] in float64, NaN in
    a block with an infinity or a NaN; bytes [rows, blocks]."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = torch.zeros(rows, blocks * 32, dtype=torch.float64)
    v[:, :cols] = x.double()
    v = v.view(rows, blocks, 32)
    bad = ~torch.isfinite(v).all(-1)
    v = torch.where(bad[..., None], 0.0, v)
    amax = v.abs().amax(-1)
    _, e = torch.frexp(amax)  # amax = f 2^e with f in [1/2, 1): floor(log2 amax) = e - 1
    byte = torch.where(amax == 0, 0, (e - 3).clamp(-127, 127) + 127)
    scale = torch.ldexp(torch.ones_like(amax), byte - 127)[..., None]
    q = v.abs() / scale
    # nearest grid value, ties to the even index: of the distances, the smaller; of equal ones, the even
    distance = (q[..., None] - GRID).abs()
    at = distance.argmin(-1)  # the first of equal ones
    up = (at + 1).clamp(max=7)
    tie = distance.gather(-1, at[..., None])[..., 0] == distance.gather(-1, up[..., None])[..., 0]
    at = torch.where(tie & (at % 2 == 1), up, at)
    out = torch.copysign(GRID[at], v) * scale
    out = torch.where(bad[..., None], float("nan"), out).reshape(rows, blocks * 32)[:, :cols]
    return out, torch.where(bad, 255, byte).to(torch.uint8)


def product_bound(a, b, dtype):
    """How far an element of a @ b.T (float64 values) may be off when it is summed in float32 in any order
    and rounded once to dtype: k - 1 additions and the products' own roundings, each of at most half a
    unit (products of 4-bit numbers are exact; an adder that drops bits below its width: a whole unit)
    of the largest partial sum, at most sum |a b|."""
    k = a.shape[1]
    sums = a.abs() @ b.abs().t()
    bits = {torch.float32: 24, torch.float16: 11, torch.bfloat16: 8}[dtype]
    return sums * (2 * max(k, 1) * 2.0 ** -24) + (a @ b.t()).abs() * 2.0 ** -bits * 1.001 + torch.finfo(dtype).smallest_normal * 2.0 ** -bits * 2
