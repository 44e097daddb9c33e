"""The row operators from their definitions, in 64 bits on the CPU, and how far a kernel may be from them.

A result is rounded once: by at most half a step, ``eps / 2`` of its value, of its type (and half of the smallest
subnormal number's step).  Behind that stand the fp32 operations before it; each is off by at most 2^-24 of its
result, and a sum of n terms in any order by n 2^-24 of the sum of their magnitudes.
"""

import torch

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24  # of an fp32 operation


def half_step(want, dtype):
    info = torch.finfo(dtype)
    return want.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def close(got, want, bound, dtype):
    """``got`` within ``bound`` (absolute, of what comes before the last rounding) and one rounding of ``want``."""
    assert got.dtype == dtype and tuple(got.shape) == tuple(want.shape), (got.dtype, got.shape, want.shape)
    got = got.detach().cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    over = want.abs() + bound > torch.finfo(dtype).max  # may round to infinity
    error = (got - want).abs()
    allowed = bound + half_step(want.abs() + bound, dtype)
    bad = (error > allowed) & ~over & ~want.isnan() & ~(got == want)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, the worst by {float((error / allowed)[bad].max())} of what it may be"


def bits16(seed, offset, count):
    """The generator's 16-bit numbers, with Python's whole numbers."""
    out = []
    for block in range(-(-count // 8)):
        c = [block & 0xFFFFFFFF, block >> 32, offset & 0xFFFFFFFF, offset >> 32 & 0xFFFFFFFF]
        k = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [b >> 32 ^ c[1] ^ k[0], b & 0xFFFFFFFF, a >> 32 ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [k[0] + 0x9E3779B9 & 0xFFFFFFFF, k[1] + 0xBB67AE85 & 0xFFFFFFFF]
        for word in c:
            out += [word & 0xFFFF, word >> 16]
    return torch.tensor(out[:count])


def norm(x, weight, residual, eps):
    """(y, h, 1 / root) of CPU tensors; h as it is rounded."""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    wide = h.double()
    r = 1 / torch.sqrt(wide.square().mean(-1, keepdim=True) + eps)
    return wide * r * (1 if weight is None else weight.double()), h, r


def norm_error(y, n):
    """fp32 before the rounding of y: the mean square is off by (n + 2) U of it at most, its root by half that and 3 U, and two products."""
    return y.abs() * ((n / 2 + 8) * U)


def norm_backward(dy, dh, h, weight, eps):
    """(dx, dw, how far fp32 may be from dx, from dw)."""
    n = h.shape[-1]
    dy, h = dy.double(), h.double()
    w = torch.ones(n, dtype=torch.float64) if weight is None else weight.double()
    r = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    g = dy * w
    along = (g * h).mean(-1, keepdim=True)
    dx = r * (g - h * r * r * along)
    # g and h c as they are subtracted: c = r^2 mean(g h), whose sum is off by n U of that of the magnitudes
    off = (g * h).abs().mean(-1, keepdim=True)
    error = r * (g.abs() * (n / 2 + 12) * U + h.abs() * r * r * off * (2.5 * n + 24) * U)
    if dh is not None:
        dx = dx + dh.double()
        error = error + dx.abs() * U * 2
    each = dy * h * r
    rows = each.reshape(-1, n)
    dw = rows.sum(0)
    return dx, dw, error, rows.abs().sum(0) * ((rows.shape[0] + n / 2 + 10) * U)


def places(chosen, experts):
    """(order, position, offsets) of [tokens, k] choices."""
    flat = chosen.reshape(-1).tolist()
    key = [e if 0 <= e < experts else experts for e in flat]
    order = sorted(range(len(key)), key=lambda i: key[i])
    position = [0] * len(key)
    for at, i in enumerate(order):
        position[i] = at
    offsets = [sum(1 for k in key if k < e) for e in range(experts + 1)] if len(key) * experts < 100000 else \
        torch.searchsorted(torch.tensor(sorted(key)), torch.arange(experts + 1)).tolist()
    return (torch.tensor(order, dtype=torch.int32), torch.tensor(position, dtype=torch.int32).reshape(chosen.shape if chosen.dim() == 2 else (-1, 1)),
            torch.tensor(offsets, dtype=torch.int32))
