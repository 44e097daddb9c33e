"""4-bit microscaled matrices on the GPU: quantisation by values, products and gradients against 64 bits."""

import pytest
import torch

import mx_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1), (1, 31), (3, 32), (5, 33), (32, 5), (2, 255), (33, 257), (257, 33), (130, 512), (64, 1000), (301, 300)]


@pytest.fixture(scope="module")
def mx():
    import torchft_amd
    return torchft_amd


def values(m, n, dtype, seed):
    """Normal over four decades from row to row, with zeros, ties and every corner of the types."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, n, generator=g) * 10.0 ** (torch.rand(m, 1, generator=g) * 4 - 3.5)
    flat = x.view(-1)
    pick = torch.randperm(flat.numel(), generator=g)
    some = pick[: flat.numel() // 4]
    flat[some] = (torch.randint(-28, 29, (some.numel(),), generator=g) / 4.0)  # ties at the smallest step
    flat[pick[: flat.numel() // 16]] = 0.0
    return x.to(dtype)


def check_matrix(got, x):
    """`got` is the matrix of x's rows."""
    want, byte = ref.quantize(x)
    assert got.shape == x.shape and got.dtype == x.dtype
    assert torch.equal(got.scales.cpu(), byte)
    assert got.codes.shape == (x.shape[0], -(-x.shape[1] // 32), 16)
    v = got.dequantize(torch.float32).cpu().double()
    assert torch.equal(torch.isnan(v), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(v), torch.nan_to_num(want))
    assert torch.equal(torch.signbit(v) & ~torch.isnan(want), torch.signbit(want) & ~torch.isnan(want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize(mx, shape, dtype):
    x = values(*shape, dtype, 1)
    gpu = x.cuda()
    check_matrix(mx.quantize_mxfp4(gpu), x)
    check_matrix(mx.quantize_mxfp4(gpu, 0), x.t().contiguous())
    rows, cols = mx.quantize_mxfp4_both(gpu)
    check_matrix(rows, x)
    check_matrix(cols, x.t().contiguous())


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_strided(mx, dtype):
    """Slices that start anywhere, rows apart, transposes, expanded rows."""
    big = values(150, 700, dtype, 2).cuda()
    for view in (big[3:140, 5:601], big[:, 8:264], big[::2], big.t(), big.t()[7:300, 1:90], big[:, ::3],
                 big[:1].expand(40, -1), big[:, 4:5], big[5:6, 1:], big[:0], big[:, :0]):
        rows, cols = mx.quantize_mxfp4_both(view)
        check_matrix(rows, view.cpu())
        check_matrix(cols, view.cpu().t().contiguous())
        check_matrix(mx.quantize_mxfp4(view), view.cpu())


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_corners(mx, dtype):
    """Largest and smallest numbers, infinities and NaN (their block, rows and columns alike, is NaN)."""
    info = torch.finfo(dtype)
    x = torch.zeros(70, 96, dtype=dtype)
    tiny = info.smallest_normal * info.eps
    x[0, :4] = torch.tensor([info.max, -info.max, info.max / 4, 1.0])
    x[1, :4] = torch.tensor([tiny, -tiny, 3 * tiny, 0.0])
    x[2, 32:36] = torch.tensor([info.smallest_normal, tiny, -info.smallest_normal / 2, 5 * tiny])
    x[3, 40] = float("inf")
    x[35, 41] = float("-inf")
    x[36, 95] = float("nan")
    x[37] = -0.0
    x[38, :] = 2.0 ** -100 if dtype != torch.float16 else 2.0 ** -20
    x[39, ::3] = 7.0
    x[69, :] = tiny
    rows, cols = mx.quantize_mxfp4_both(x.cuda())
    check_matrix(rows, x)
    check_matrix(cols, x.t().contiguous())


@pytest.mark.parametrize("dtype", DTYPES)
def test_dequantize_types(mx, dtype):
    """Rounded once to the type asked for, into its subnormal numbers and past its largest one."""
    x = values(40, 300, torch.float32, 3)
    x[7] *= 1e-38
    x[8] *= 1e30
    x[9] *= 1e-6
    m = mx.quantize_mxfp4(x.cuda())
    assert torch.equal(m.dequantize(dtype).cpu().float(), ref.quantize(x)[0].to(dtype).float())


@pytest.mark.parametrize("cols", [1, 31, 32, 33, 255, 256, 257, 600])
def test_from_blocks(mx, cols):
    """What a checkpoint holds goes in and comes out; codes past the last column count as zero."""
    g = torch.Generator().manual_seed(cols)
    blocks = -(-cols // 32)
    codes = torch.randint(0, 256, (9, blocks, 16), generator=g).to(torch.uint8)
    scales = torch.randint(100, 140, (9, blocks), generator=g).to(torch.uint8)
    m = mx.MXFP4Tensor.from_blocks(codes.cuda(), scales.cuda(), cols)
    assert torch.equal(m.scales.cpu(), scales)
    each = torch.stack([codes & 15, codes >> 4], -1).view(9, blocks, 32).long()
    want = torch.where(each > 7, -1.0, 1.0) * ref.GRID[each % 8] * torch.exp2(scales.double() - 127)[..., None]
    want = want.view(9, -1)[:, :cols]
    assert torch.equal(m.dequantize(torch.float32).cpu().double(), want)
    past = torch.stack([m.codes.cpu() & 15, m.codes.cpu() >> 4], -1).view(9, -1)[:, cols:]
    assert not past.any()


def operand(mx, m, k, dtype, seed):
    x = values(m, k, dtype, seed)
    return mx.quantize_mxfp4(x.cuda()), ref.quantize(x)[0]


def close(got, want, bound):
    off = (got.cpu().double() - want).abs()
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert worst <= 0, f"off by {worst} more than the bound"


PRODUCTS = [(1, 1, 1), (1, 40, 33), (7, 5, 256), (16, 16, 257), (17, 100, 600), (33, 129, 513), (64, 64, 1024), (65, 300, 31),
            (128, 128, 512), (130, 1000, 300), (257, 511, 700), (1000, 1, 64), (1, 1000, 4100)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", PRODUCTS)
def test_product(mx, shape, dtype):
    m, n, k = shape
    (a, av), (b, bv) = operand(mx, m, k, dtype, 4), operand(mx, n, k, torch.float32, 5)
    close(mx.matmul_mxfp4(a, b, dtype), av @ bv.t(), ref.product_bound(av, bv, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3000, 3500, 500), (4100, 4099, 256), (1700, 2000, 1024)])
def test_product_of_many_tiles(mx, shape, dtype):
    """Enough tiles for the larger kernels, with partial ones at both edges."""
    m, n, k = shape
    g = torch.Generator("cuda").manual_seed(6)
    x = torch.randn(m, k, device="cuda", generator=g)
    w = torch.randn(n, k, device="cuda", generator=g) * torch.exp2(torch.randint(-9, 9, (n, 1), device="cuda", generator=g).float())
    a, b = mx.quantize_mxfp4(x), mx.quantize_mxfp4(w)
    av, bv = a.dequantize().double(), b.dequantize().double()
    got, want = mx.matmul_mxfp4(a, b, dtype).double(), av @ bv.t()
    assert ((got - want).abs() - ref.product_bound(av, bv, dtype)).max().item() <= 0


def test_product_extreme_scales(mx):
    """Scales whose product passes float32's range on either side, and NaN blocks, which make their rows NaN."""
    x = torch.ones(40, 64)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] = 0
    x[3, 40] = float("nan")
    w = torch.ones(50, 64)
    w[0] *= 1e30
    w[1] *= 1e-30
    w[2, 3] = float("inf")
    a, b = mx.quantize_mxfp4(x.cuda()), mx.quantize_mxfp4(w.cuda())
    got = mx.matmul_mxfp4(a, b, torch.float32).cpu()
    want = (ref.quantize(x)[0] @ ref.quantize(w)[0].t())
    assert torch.isnan(got[3]).all() and torch.isnan(got[:, 2]).all()
    rest = torch.ones_like(got, dtype=torch.bool)
    rest[3], rest[:, 2] = False, False
    assert torch.isinf(got[0, 0]) and got[0, 0] > 0  # 64e60
    rest[0, 0] = False
    assert (got[rest].double() - want[rest]).abs().le(want[rest].abs() * 2.0 ** -20 + 2.0 ** -126).all()


def test_empty_sizes(mx):
    for m, n, k in ((0, 5, 7), (5, 0, 7), (5, 7, 0), (0, 0, 0)):
        x = torch.zeros(m, k, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        w = torch.zeros(n, k, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        y = mx.linear_mxfp4(x, w)
        assert y.shape == (m, n) and not y.any()
        y.sum().backward()
        assert x.grad.shape == x.shape and not x.grad.any() and w.grad.shape == w.shape and not w.grad.any()


TRAINED = [(1, 1, 1), (3, 40, 33), (64, 64, 64), (100, 257, 300), (511, 130, 1001), (1, 500, 70)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", TRAINED)
def test_linear_and_its_gradient(mx, shape, dtype):
    """The formula's: every product of operands quantised along the contracted axis, in 64 bits."""
    t, n, k = shape
    x, w, dy = values(t, k, dtype, 7), values(n, k, torch.float32, 8), values(t, n, dtype, 9)
    gx, gw = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = mx.linear_mxfp4(gx, gw)
    y.backward(dy.cuda())
    assert y.dtype == dtype and gx.grad.dtype == dtype and gw.grad.dtype == torch.float32

    def q(v):
        return ref.quantize(v)[0]
    for got, a, b in ((y.detach(), q(x), q(w)), (gx.grad, q(dy), q(w.t())), (gw.grad, q(dy.t()), q(x.t()))):
        close(got, a @ b.t(), ref.product_bound(a, b, got.dtype))


def test_gradient_against_differences(mx):
    """On matrices of -3 to 3 in which every block's largest magnitude is 4 to 6, quantisation along either axis
    changes nothing (its step is 1 or less there), and the layer is exactly bilinear: half the
    difference over a step of one in both directions is the derivative, without an error."""
    g = torch.Generator().manual_seed(10)
    t, n, k = 64, 32, 96

    def grid(rows, cols):
        v = torch.randint(-3, 4, (rows, cols), generator=g).float()
        v[::32] = 4.0
        v[:, ::32] = 4.0
        return v
    x, w, dy = grid(t, k), grid(n, k), grid(t, n)
    gx, gw = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = mx.linear_mxfp4(gx, gw)
    y.backward(dy.cuda())

    def loss(a, b):
        return (mx.linear_mxfp4(a.cuda(), b.cuda()).cpu().double() * dy.double()).sum().item()
    for _ in range(12):
        i, j, c = (int(torch.randint(1, s, (1,), generator=g)) for s in (32, 32, 32))
        for base, grad, at, other in ((x, gx.grad, (i, c), w), (w, gw.grad, (j, c), x)):
            up, down = base.clone(), base.clone()
            up[at], down[at] = (base[at] + 1).clamp(max=3), (base[at] - 1).clamp(min=-3)
            step = (up[at] - down[at]).item()
            got = (loss(up, other) - loss(down, other)) if base is x else (loss(other, up) - loss(other, down))
            assert got / step == grad[at].item()


def test_leading_dimensions_and_frozen_inputs(mx):
    x = values(24, 100, torch.bfloat16, 11).cuda()
    w = values(50, 100, torch.bfloat16, 12).cuda()
    flat = mx.linear_mxfp4(x, w)
    assert torch.equal(mx.linear_mxfp4(x.view(2, 3, 4, 100), w), flat.view(2, 3, 4, 50))
    assert torch.equal(mx.linear_mxfp4(x[0], w), mx.linear_mxfp4(x[:1], w)[0])
    kept = mx.quantize_mxfp4(w)
    assert torch.equal(mx.linear_mxfp4(x, kept), flat)
    for wants_x in (True, False):
        gx, gw = x.clone().requires_grad_(wants_x), w.clone().requires_grad_(not wants_x)
        mx.linear_mxfp4(gx.view(6, 4, 100), gw).sum().backward()
        both = x.clone().requires_grad_(), w.clone().requires_grad_()
        mx.linear_mxfp4(*both).sum().backward()
        if wants_x:
            assert torch.equal(gx.grad, both[0].grad) and gw.grad is None
        else:
            assert torch.equal(gw.grad, both[1].grad) and gx.grad is None


def test_another_stream_and_graph(mx):
    """The calls go to the current stream; a captured call gives the eager bytes on every replay."""
    x, w = values(40, 512, torch.bfloat16, 13).cuda(), values(70, 512, torch.bfloat16, 14).cuda()
    want = mx.linear_mxfp4(x, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = mx.linear_mxfp4(x, w)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    static = x.clone()
    with torch.cuda.graph(graph):
        out = mx.linear_mxfp4(static, w)
    for scale in (1.0, 2.0, 0.5, -1.0):
        static.copy_(x * scale)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want * scale)


def test_refusals(mx):
    x = torch.zeros(4, 64, device="cuda")
    m = mx.quantize_mxfp4(x)
    with pytest.raises(AssertionError, match="2D"):
        mx.quantize_mxfp4(x[0])
    with pytest.raises(AssertionError, match="fp32, fp16 and bf16"):
        mx.quantize_mxfp4(x.double())
    with pytest.raises(AssertionError, match="GPU"):
        mx.quantize_mxfp4(x.cpu())
    with pytest.raises(AssertionError, match="numbers of columns"):
        mx.matmul_mxfp4(m, mx.quantize_mxfp4(x[:, :63]))
    with pytest.raises(AssertionError, match="number of columns"):
        mx.linear_mxfp4(x[:, :63], x)
    with pytest.raises(AssertionError, match="fp32, fp16 and bf16"):
        mx.matmul_mxfp4(m, m, torch.float64)
    with pytest.raises(AssertionError, match="no gradient product"):
        mx.linear_mxfp4(x.clone().requires_grad_(), m)
    with pytest.raises(AssertionError, match="same device"):
        mx.linear_mxfp4(x.cpu(), m)
    codes, scales = m.codes, m.scales
    for bad in ((codes.int(), scales, 64), (codes, scales, 65), (codes, scales, 32), (codes[:, :1], scales, 64), (codes[..., :15], scales, 64)):
        with pytest.raises(AssertionError):
            mx.MXFP4Tensor.from_blocks(*bad)


def test_past_four_gib(mx):
    """A matrix whose codes, and whose source, pass 2^32 bytes."""
    rows, cols = 1 << 20, 8448
    g = torch.Generator("cuda").manual_seed(15)
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    part = torch.randn(4096, cols, device="cuda", generator=g).to(torch.bfloat16)
    for i in range(0, rows, 4096):
        x[i:i + 4096] = part
    x[-1] *= 2
    m, t = mx.quantize_mxfp4_both(x)
    small = mx.quantize_mxfp4(part)
    v = m.dequantize()
    assert torch.equal(v[-4096:-1], small.dequantize()[:-1]) and torch.equal(v[-1], 2 * small.dequantize()[-1])
    assert torch.equal(v[524288:528384], v[:4096])
    del v, x
    a = mx.quantize_mxfp4(torch.randn(5, cols, device="cuda", generator=g))
    y, want = mx.matmul_mxfp4(a, m), mx.matmul_mxfp4(a, small)
    assert torch.equal(y[:, -4096:-1], want[:, :-1]) and torch.equal(y[:, -1], 2 * want[:, -1])
    z = t.dequantize()  # [cols, rows]
    assert torch.equal(z[:, -4096:-32], z[:, :4064])
