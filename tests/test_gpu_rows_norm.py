"""Root-mean-square norm on the GPU, its gradients and its output in 8 bits, against 64 bits."""

import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu

EPS = 1e-6
# every number of lanes to a row and their borders in both directions, rows beyond registers, odd ends
SHAPES = [(1, 1), (3, 7), (5, 8), (33, 31), (7, 64), (260, 65), (4, 127), (19, 129), (2, 257), (9, 512), (3, 513), (6, 1001),
          (1, 1024), (5, 2047), (300, 130), (2, 4096), (3, 4097), (2, 8191), (3, 16390), (2, 33000), (1, 65537)]


@pytest.fixture(scope="module")
def t():
    import torchft_amd
    return torchft_amd


def values(rows, cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * 10.0 ** (torch.rand(rows, 1, generator=g) * 3 - 2)
    x[torch.rand(rows, cols, generator=g) < 0.02] *= 20
    return x.to(dtype)


def check(t, x, weight, residual, dy, dh, grads=True):
    """One forward and backward pass; CPU tensors in."""
    gx, gw, gr = (None if v is None else v.cuda().requires_grad_(grads) for v in (x, weight, residual))
    got = t.rms_norm(gx, gw, gr, EPS)
    y, h = (got, None) if residual is None else got
    want, want_h, _ = ref.norm(x, weight, residual, EPS)
    ref.close(y, want, ref.norm_error(want, x.shape[-1]), x.dtype)
    if residual is not None:
        assert torch.equal(h.detach().cpu(), want_h)
    if not grads:
        assert not y.requires_grad
        return
    inputs = [v for v in (gx, gw, gr) if v is not None]
    outputs, dout = [y], [dy.cuda()]
    if residual is not None:
        outputs.append(h)
        dout.append(dh.cuda())
    d = list(torch.autograd.grad(outputs, inputs, dout))
    dx, dw, ex, ew = ref.norm_backward(dy, dh if residual is not None else None, want_h, weight, EPS)
    ref.close(d.pop(0), dx, ex, x.dtype)
    if weight is not None:
        ref.close(d.pop(0), dw, ew, weight.dtype)
    if residual is not None:
        ref.close(d.pop(0), dx, ex, x.dtype)


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_norm(t, shape, dtype):
    x, r, dy, dh = (values(*shape, dtype, s) for s in range(4))
    w = (1 + values(1, shape[1], torch.float32, 5)[0]).to(dtype)
    check(t, x, w, r, dy, dh)
    check(t, x, w.float(), None, dy, None)
    check(t, x, None, r, dy, dh)
    check(t, x, w, r, dy, dh, grads=False)


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_many_rows(t, dtype):
    """More rows than the backward pass has teams for."""
    for shape in ((9000, 24), (40000, 8), (2500, 600)):
        x, dy = values(*shape, dtype, 1), values(*shape, dtype, 2)
        check(t, x, (1 + values(1, shape[1], torch.float32, 5)[0]).to(dtype), None, dy, None)


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_fp8(t, shape, dtype):
    """A code is off by half a step of its 4 bits, or by one where fp32 lies on the other side of a border."""
    x, r = values(*shape, dtype, 1), values(*shape, dtype, 2)
    w = (1 + values(1, shape[1], torch.float32, 5)[0]).to(dtype)
    for residual in (None, r):
        got = t.rms_norm_fp8(x.cuda(), w.cuda(), None if residual is None else residual.cuda(), EPS)
        rows, h = (got, None) if residual is None else got
        y, want_h, _ = ref.norm(x, w, residual, EPS)
        if residual is not None:
            assert torch.equal(h.cpu(), want_h)
        assert rows.codes.dtype == torch.float8_e4m3fn and rows.codes.shape == x.shape and rows.scales.shape == (shape[0], 1)
        amax = y.abs().amax(1, keepdim=True)
        slack = (shape[1] / 2 + 16) * ref.U
        want_scale = torch.where(amax / 448 < 2.0 ** -126, 1.0, amax / 448)
        scale = rows.scales.cpu().double()
        assert ((scale - want_scale).abs() <= want_scale * slack).all()
        v = rows.codes.cpu().float().double()
        # half of a step: 2^-4 of the number, 2^-10 below 2^-6
        allowed = torch.maximum(v.abs() / 16, torch.tensor(2.0 ** -10, dtype=torch.float64)) * scale + y.abs() * slack
        assert ((v * scale - y).abs() <= allowed).all()
        for out in ref.DTYPES:
            values_ = rows.dequantize(out)
            assert torch.equal(values_.cpu(), (rows.codes.cpu().float() * rows.scales.cpu()).to(out))
        assert rows.dequantize().dtype == dtype


@pytest.mark.parametrize("shape", [(40000, 3), (3000, 64), (700, 333), (90, 2900), (60, 4480), (20, 8000), (6, 16390), (4, 40001)])
def test_fp8_nearest(t, shape):
    """Codes of fp32 rows are the nearest: two results of 64 bits lie on two sides of a border once in 10^14 codes."""
    x, r, w = values(*shape, torch.float32, 1), values(*shape, torch.float32, 2), 1 + values(1, shape[1], torch.float32, 5)[0]
    for residual in (None, r):
        got = t.rms_norm_fp8(x.cuda(), w.cuda(), None if residual is None else residual.cuda(), EPS)
        rows = got if residual is None else got[0]
        y, _, _ = ref.norm(x, w, residual, EPS)
        z = y / (y.abs().amax(1, keepdim=True) / 448)
        step = torch.exp2(torch.frexp(z.abs().clamp(min=2.0 ** -6)).exponent.double() - 4)  # e4m3: 4 bits, 2^-9 at least
        assert torch.equal(rows.codes.cpu().double(), (z / step).round() * step)


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_orders(t, dtype):
    """Slices, transposes, heads inside wider rows, expanded rows, more dimensions, empty ones."""
    big = values(64, 600, dtype, 3).cuda()
    w = {}
    for view in (big[3:40, 5:405], big[::2, 1:130], big.t(), big[:1].expand(9, -1), big.view(8, 8, 600)[:, :, 7:100], big[:, ::3],
                 big.view(64, 5, 120)[:, 1:4], big.view(8, 8, 600).transpose(0, 1), big[5], big[:, 4:5], big[:0], big[:, :0], big.view(2, 32, 600)[:, :1]):
        n = view.shape[-1]
        weight = w.setdefault(n, (1 + values(1, n, torch.float32, n)[0]).to(dtype)) if n else torch.zeros(0, dtype=dtype)
        x = view.cpu()
        y = t.rms_norm(view, weight.cuda(), None, EPS)
        want = ref.norm(x, weight, None, EPS)[0] if n else torch.zeros(x.shape, dtype=torch.float64)
        ref.close(y, want, ref.norm_error(want, n), dtype)
        y, h = t.rms_norm(view.contiguous(), weight.cuda(), view, EPS)
        assert torch.equal(h.cpu(), (x.float() + x.float()).to(dtype))
        leaf = view.detach().requires_grad_()
        got = t.rms_norm(leaf, weight.cuda(), None, EPS)
        dy = torch.full_like(got, 0.5)
        if n and x.numel():
            dx, _, ex, _ = ref.norm_backward(dy.cpu(), None, x, weight, EPS)
            ref.close(torch.autograd.grad(got.sum() * 0.5, leaf)[0], dx, ex, dtype)
        else:
            assert torch.autograd.grad(got.sum(), leaf)[0].shape == leaf.shape


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_heads(t, dtype):
    """Queries and keys inside wider rows, heads before tokens, groups of one row, rows long and short; without a copy of x."""
    for heads, d in ((5, 64), (3, 33), (1, 128), (7, 4), (2, 1100), (2, 9000), (2, 40000)):
        wide = values(6, 3 * heads * d, dtype, d).cuda().view(2, 3, 3, heads, d)
        w = (1 + values(1, d, torch.float32, d)[0]).to(dtype)
        for view in (wide[:, :, 1], wide[:, :, 2, :, : max(1, d - 1)], wide[:, :, 0].transpose(1, 2), wide[:, :, :2], wide[:, 1, 1:]):
            n = view.shape[-1]
            x = view.cpu()
            leaf = view.detach().requires_grad_()
            weight = w[:n].cuda().requires_grad_()
            y = t.rms_norm(leaf, weight, None, EPS)
            want, h, _ = ref.norm(x, w[:n], None, EPS)
            ref.close(y, want, ref.norm_error(want, n), dtype)
            dy = values(x.numel() // n, n, dtype, 5).view(x.shape)
            dx, dw = torch.autograd.grad(y, (leaf, weight), dy.cuda())
            want, dw_want, error, dw_error = ref.norm_backward(dy, None, x, w[:n], EPS)
            ref.close(dx, want, error, dtype)
            ref.close(dw, dw_want, dw_error, dtype)
            y, h = t.rms_norm(view, weight.detach(), view, EPS)
            assert torch.equal(h.cpu(), (x.float() + x.float()).to(dtype))


def test_no_rows(t):
    """A batch without tokens: the weight's gradient is zeros."""
    x = torch.empty(0, 40, device="cuda", requires_grad=True)
    w = torch.ones(40, device="cuda", requires_grad=True)
    dx, dw = torch.autograd.grad(t.rms_norm(x, w).sum(), (x, w))
    assert dx.shape == (0, 40) and torch.equal(dw.cpu(), torch.zeros(40))


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_corners(t, dtype):
    """Rows of zeros, infinities and NaN are no other row's matter."""
    x = values(8, 300, dtype, 1)
    x[1] = 0
    x[3, 7] = float("inf")
    x[5, 250] = float("nan")
    dy = values(8, 300, dtype, 2)
    y = t.rms_norm(x.cuda(), None, None, EPS).cpu()
    clean = [0, 1, 2, 4, 6, 7]
    want = ref.norm(x[clean], None, None, EPS)[0]
    ref.close(y[clean], want, ref.norm_error(want, 300), dtype)
    assert y[5].isnan().all() and y[3, 7].isnan() and (y[3, :7] == 0).all()
    leaf = x.cuda().requires_grad_()
    dx = torch.autograd.grad(t.rms_norm(leaf, None, None, EPS), leaf, dy.cuda())[0].cpu()
    want, _, error, _ = ref.norm_backward(dy[clean], None, x[clean], None, EPS)
    ref.close(dx[clean], want, error, dtype)
    rows = t.rms_norm_fp8(x.cuda(), None, None, EPS)
    assert rows.scales[1].item() == 1 and rows.scales[5].item() == 1
    assert rows.dequantize().cpu()[5].isnan().all() and not rows.dequantize().cpu()[clean].isnan().any()


def test_some_gradients(t):
    """Each of the inputs alone, and each of the outputs alone."""
    x, r, dy = (values(10, 200, torch.float32, s).cuda() for s in range(3))
    w = (1 + values(1, 200, torch.float32, 5)[0]).cuda()
    every = [v.clone().requires_grad_() for v in (x, w, r)]
    y, h = t.rms_norm(every[0], every[1], every[2])
    full = torch.autograd.grad(y, every, dy, retain_graph=True)
    for i in range(3):
        some = [v.clone().requires_grad_(k == i) for k, v in enumerate((x, w, r))]
        y1, h1 = t.rms_norm(*some)
        assert torch.equal(torch.autograd.grad(y1, some[i], dy)[0], full[i])
    only = torch.autograd.grad(h, every, dy, allow_unused=True, retain_graph=True)
    assert torch.equal(only[0], dy) and torch.equal(only[2], dy) and only[1] is None
    z = t.rms_norm(every[0])
    assert torch.equal(torch.autograd.grad(z.sum(), every[0])[0], torch.autograd.grad(t.rms_norm(every[0]), every[0], torch.ones_like(x))[0])


def test_differences(t):
    """Gradients against differences of the operator itself."""
    g = torch.Generator().manual_seed(7)
    x, r, dy, dh = (torch.randn(4, 33, generator=g).cuda() for _ in range(4))
    w = (1 + 0.3 * torch.randn(33, generator=g)).cuda()
    leaves = [v.requires_grad_() for v in (x, w, r)]
    y, h = t.rms_norm(*leaves)
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))

    def loss(*args):
        with torch.no_grad():
            y, h = t.rms_norm(*args)
        return float((y.double() * dy.double()).sum() + (h.double() * dh.double()).sum())

    step = 2.0 ** -6
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        towards = torch.randn(leaf.shape, generator=g).cuda()
        args = lambda s: [v.detach() + s * towards if k == i else v.detach() for k, v in enumerate(leaves)]  # noqa: E731
        slope = (loss(*args(step)) - loss(*args(-step))) / (2 * step)
        along = float((grad.double() * towards.double()).sum())
        # the third derivative along |towards| of about sqrt(n), step^2 / 6 of it, and fp32 noise over the step
        assert abs(slope - along) <= 2e-2 * (abs(along) + float(grad.double().norm()) * float(towards.double().norm()) * 0.1)


def test_second_derivative_is_refused(t):
    x = torch.randn(3, 40, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(t.rms_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once"):
        dx.sum().backward()


def test_streams_and_graph(t):
    """Another stream than the tensors' own; a captured forward and backward pass, replayed with other numbers."""
    x, r, dy, dh = (values(50, 520, torch.bfloat16, s).cuda() for s in range(4))
    w = torch.ones(520, device="cuda")
    leaves = [v.clone().requires_grad_() for v in (x, w, r)]

    def step():
        y, h = t.rms_norm(*leaves)
        return (y.detach(), h.detach(), *torch.autograd.grad((y, h), leaves, (dy, dh)))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (11, 12, 13):
        with torch.no_grad():
            leaves[0].copy_(values(50, 520, torch.bfloat16, seed))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step(), out))
        torch.cuda.synchronize()
