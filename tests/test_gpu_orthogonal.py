"""Newton-Schulz orthogonalisation and Muon's step on the GPU against 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# Relative error (2-norms).  Rounding to 22 bits, or float32 products: at most 6e-6 in a simulation over
# these sizes and spectra; to 11 bits, diagonals and remainders apart: at most 1.3e-3, beside the result's
# own rounding (2^-9 / sqrt(3) of each element for bfloat16, 2^-12 / sqrt(3) for float16: 1.7e-3, 2.1e-4
# of evenly spread mantissas).  Twice that.
PRECISE, HALF = 1.2e-5, 2.6e-3
ROUNDING = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}


@pytest.fixture(scope="module")
def ta():
    import torchft_amd
    return torchft_amd


def bound(dtype, precise):
    return (PRECISE if precise else HALF) + ROUNDING[dtype]


def reference(u, coefficients=((A, B, C),) * 5, eps=1e-7):
    x = u.double()
    if x.shape[0] > x.shape[1]:
        return reference(u.t(), coefficients, eps).t()
    x = x / max(x.norm().item(), eps)
    for a, b, c in coefficients:
        s = x @ x.t()
        x = a * x + (b * s + c * s @ s) @ x
    return x


def gradient(m, n, dtype, seed, kind="low", device="cpu"):
    g = torch.Generator(device).manual_seed(seed)
    x = torch.randn(m, n, generator=g, device=device)
    if kind == "low":
        r = max(1, min(m, n) // 8)
        x = 0.02 * x + torch.randn(m, r, generator=g, device=device) @ torch.randn(r, n, generator=g, device=device) / math.sqrt(r)
    return (x * 1e-3).to(dtype)


def check(got, want, limit):
    got, want = got.double().to(want.device), want.double()
    assert got.shape == want.shape and torch.isfinite(got).all()
    off = (got - want).norm().item() / max(want.norm().item(), 1e-300)
    assert off <= limit, f"off by {off:.2e}, {limit:.2e} are allowed"
    rms = want.norm() / math.sqrt(want.numel())
    worst = ((got - want).abs() / torch.maximum(rms, want.abs())).max().item()
    assert worst <= 40 * limit, f"an element is off by {worst:.2e}"


SHAPES = [(1, 1), (1, 777), (777, 1), (3, 5), (31, 64), (64, 64), (65, 63), (66, 129), (130, 257), (300, 1000), (1000, 300), (512, 512)]


@pytest.mark.parametrize("kind", ["even", "low"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(ta, shape, dtype, kind):
    x = gradient(*shape, dtype, 1, kind)
    got = ta.orthogonalize(x.cuda())
    assert got.dtype == dtype
    check(got, reference(x), bound(dtype, dtype != torch.bfloat16))


@pytest.mark.parametrize("shape", [(2048, 2048), (1100, 4096), (4096, 1100), (4100, 4099), (2560, 9000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_larger(ta, shape, dtype):
    """Enough tiles for the larger kernels, with partial ones at the edges."""
    x = gradient(*shape, dtype, 2, device="cuda")
    check(ta.orthogonalize(x), reference(x), bound(dtype, dtype == torch.float32))


@pytest.mark.parametrize("precise", [False, True])
@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_types(ta, dtype, out, precise):
    x = gradient(96, 200, dtype, 3)
    got = ta.orthogonalize(x.cuda(), out_dtype=out, precise=precise)
    assert got.dtype == out
    check(got, reference(x), bound(out, precise))


def test_list_of_more_matrices_than_a_launch_takes(ta):
    shapes = [(8 * (i % 7) + 1, 13 * (i % 5) + 2) for i in range(60)] + [(0, 5), (200, 300), (5, 0), (300, 200)]
    xs = [gradient(*s, torch.float32, 4 + i) for i, s in enumerate(shapes)]
    got = ta.orthogonalize([x.cuda() for x in xs])
    for x, y in zip(xs, got):
        assert y.shape == x.shape
        if x.numel():
            check(y, reference(x), bound(torch.float32, True))
    alone = [ta.orthogonalize(x.cuda()) for x in xs]
    assert all(torch.equal(a, b) for a, b in zip(got[:60], alone[:60]))


@pytest.mark.parametrize("precise", [False, True])
def test_strides(ta, precise):
    """Slices that start anywhere, rows apart, stored by columns, every third column."""
    big = gradient(300, 500, torch.float32, 5)
    gpu = big.cuda()
    for at in ((slice(3, 130), slice(1, 260)), (slice(None), slice(5, 6)), (slice(0, 300, 2), slice(0, 64)), (slice(7, 8), slice(None)),
               (slice(0, 90), slice(0, 500, 3))):
        for pick, ref in ((gpu[at], big[at]), (gpu.t()[at[::-1]], big.t()[at[::-1]])):
            check(ta.orthogonalize(pick, precise=precise), reference(ref), bound(torch.float32, precise))


def test_sizes_of_gradients(ta):
    """The result does not depend on the gradient's size, down to eps; nothing under- or overflows on the way."""
    x = gradient(70, 90, torch.float32, 6)
    want = reference(x)
    for scale in (1e-25, 1e-10, 1.0, 1e20, 1e38):
        check(ta.orthogonalize((x * scale).cuda(), eps=1e-35), want, bound(torch.float32, True))
    small = x * 1e-12
    check(ta.orthogonalize(small.cuda()), reference(small), bound(torch.float32, True))
    zero = torch.zeros(40, 50, device="cuda")
    assert not ta.orthogonalize(zero).any()
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[3, 4] = bad
        got = ta.orthogonalize([y.cuda(), x.cuda()])
        assert torch.isnan(got[0]).all()
        check(got[1], want, bound(torch.float32, True))


def test_coefficients_of_every_iteration(ta):
    table = ((A, B, C),) * 4 + ((2.0, -1.5, 0.5), (1.875, -1.25, 0.375))
    x = gradient(80, 200, torch.float32, 7)
    check(ta.orthogonalize(x.cuda(), steps=6, coefficients=table), reference(x, table), bound(torch.float32, True))
    check(ta.orthogonalize(x.cuda(), steps=1), reference(x, ((A, B, C),)), bound(torch.float32, True))


def step_reference(w, g, m, lr, decay, momentum, nesterov):
    m = momentum * m.double() + (1 - momentum) * g.double()
    u = g.double() + momentum * (m - g.double()) if nesterov else m
    scale = math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
    return reference(u) * scale, m


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("grad_dtype", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_muon(ta, dtype, grad_dtype, nesterov):
    shapes = [(130, 70), (64, 64), (33, 200), (1, 50)]
    g = torch.Generator().manual_seed(8)
    ws = [(torch.randn(s, generator=g) * 0.02).to(dtype) for s in shapes]
    gs = [gradient(*s, grad_dtype, 9) for s in shapes]
    ms = [gradient(*s, torch.float32, 10) for s in shapes]
    gw, gg, gm = ([t.cuda() for t in ts] for ts in (ws, gs, ms))
    version = gw[0]._version
    ta.muon_(gw, gg, gm, lr=0.3, weight_decay=0.2, momentum=0.9, nesterov=nesterov)
    assert gw[0]._version > version
    for w, gr, m, w2, g2, m2 in zip(ws, gs, ms, gw, gg, gm):
        o, want_m = step_reference(w, gr, m, 0.3, 0.2, 0.9, nesterov)
        assert torch.equal(g2.cpu(), gr)
        assert (m2.cpu().double() - want_m).abs().le(want_m.abs() * 2.0 ** -22 + gr.double().abs() * 2.0 ** -22).all()
        want = (1 - 0.3 * 0.2) * w.double() - 0.3 * o
        # the step's error, and the weight's rounding and its two products' in float32
        off = (w2.cpu().double() - want).norm().item()
        assert off <= 0.3 * o.norm().item() * (PRECISE if dtype != torch.bfloat16 else HALF) + want.norm().item() * (ROUNDING[dtype] + 2.0 ** -22)


@pytest.mark.parametrize("order", ["weights", "grads", "momenta", "all"])
def test_muon_on_other_orders(ta, order):
    """Tensors of one matrix that are stored in different orders, or with gaps; what lies between stays."""
    g = torch.Generator().manual_seed(11)
    w, gr, m = torch.randn(50, 80, generator=g), gradient(50, 80, torch.float32, 12), gradient(50, 80, torch.float32, 13)
    want = [t.clone().cuda() for t in (w, gr, m)]
    ta.muon_(*([t] for t in want), lr=0.1)

    def other(t, name):
        if order not in (name, "all"):
            return t.cuda(), None
        base = torch.full((80, 120), 7.0, device="cuda")
        view = base.t()[10:60]
        view.copy_(t)
        return view, base
    views = [other(t, n) for t, n in ((w, "weights"), (gr, "grads"), (m, "momenta"))]
    ta.muon_(*([v] for v, _ in views), lr=0.1)
    for (v, base), t in zip(views, want):
        assert torch.allclose(v, t, rtol=1e-4, atol=1e-6)
        if base is not None:
            assert (base.t()[:10] == 7).all() and (base.t()[60:] == 7).all()


def test_optimizer(ta):
    """The optimiser's steps are the function's, group by group; a weight without a gradient stays."""
    g = torch.Generator().manual_seed(14)
    ps = [torch.nn.Parameter(torch.randn(s, generator=g).cuda()) for s in ((20, 30), (40, 10), (16, 16))]
    ws, ms = [p.detach().clone() for p in ps[:2]], [torch.zeros_like(p, dtype=torch.float32) for p in ps[:2]]
    opt = ta.Muon([{"params": ps[:1], "lr": 0.1}, {"params": ps[1:], "weight_decay": 0.3}], lr=0.2)
    third = ps[2].detach().clone()
    for i in range(3):
        gs = [gradient(*w.shape, torch.float32, 20 + i).cuda() for w in ws]
        for p, gr in zip(ps, gs):
            p.grad = gr.clone()
        assert opt.step(lambda: 1.5) == 1.5
        ta.muon_(ws[:1], gs[:1], ms[:1], lr=0.1)
        ta.muon_(ws[1:], gs[1:], ms[1:], lr=0.2, weight_decay=0.3)
    assert all(torch.equal(p, w) for p, w in zip(ps, ws)) and torch.equal(ps[2], third)
    again = ta.Muon([{"params": ps[:1]}, {"params": ps[1:]}])
    again.load_state_dict(opt.state_dict())
    assert torch.equal(again.state[ps[0]]["momentum"], ms[0])


def test_another_stream_and_graph(ta):
    x = gradient(200, 300, torch.bfloat16, 15).cuda()
    want = ta.orthogonalize(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ta.orthogonalize(x)
    side.synchronize()
    assert torch.equal(got, want)
    static, other = x.clone(), gradient(200, 300, torch.bfloat16, 16).cuda()
    want_other = ta.orthogonalize(other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ta.orthogonalize(static)
    for source, result in ((x, want), (other, want_other), (x, want), (other, want_other)):
        static.copy_(source)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, result)
        assert torch.equal(ta.orthogonalize(source), result)


def test_refusals(ta):
    x = torch.zeros(4, 6, device="cuda")
    with pytest.raises(AssertionError, match="2D"):
        ta.orthogonalize(x[0])
    with pytest.raises(AssertionError, match="fp32, fp16 and bf16"):
        ta.orthogonalize(x.double())
    with pytest.raises(AssertionError, match="GPU"):
        ta.orthogonalize(x.cpu())
    with pytest.raises(AssertionError, match="same dtype"):
        ta.orthogonalize([x, x.half()])
    with pytest.raises(AssertionError, match="same device"):
        ta.orthogonalize([x, x.cpu()])
    with pytest.raises(AssertionError, match="iteration"):
        ta.orthogonalize(x, steps=0)
    with pytest.raises(AssertionError, match="coefficients"):
        ta.orthogonalize(x, steps=3, coefficients=((1.0, 2.0, 3.0),) * 2)
    with pytest.raises(AssertionError, match="lengths"):
        ta.muon_([x], [x], [], lr=0.1)
    with pytest.raises(AssertionError, match="other shapes"):
        ta.muon_([x], [x.t()], [x], lr=0.1)
    with pytest.raises(AssertionError, match="same dtype"):
        ta.muon_([x], [x], [x.half()], lr=0.1)
    with pytest.raises(AssertionError, match="out of range"):
        ta.muon_([x], [x], [x], lr=-0.1)
    with pytest.raises(AssertionError, match="2D"):
        ta.Muon([torch.nn.Parameter(x[0])])
    assert ta.orthogonalize([]) == [] and ta.orthogonalize(x[:0]).shape == (0, 6)
    ta.muon_([], [], [], lr=0.1)
