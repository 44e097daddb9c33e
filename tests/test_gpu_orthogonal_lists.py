"""Newton-Schulz orthogonalisation and Muon's step on lists: many small matrices, those that take three
products a product beside those that take one."""

import math

import pytest
import torch

from test_gpu_orthogonal import DTYPES, HALF, PRECISE, ROUNDING, bound, check, gradient, reference, step_reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ta():
    import torchft_amd
    return torchft_amd


# enough tiles of 32 x 32 for the tiles of 64 x 64, from one panel of 64 columns to several
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(64, 640), (128, 128), (129, 65), (300, 300), (190, 450)])
def test_24_of_one_shape(ta, shape, dtype):
    xs = [gradient(*shape, dtype, 30 + i) for i in range(24)]
    for x, y in zip(xs, ta.orthogonalize([x.cuda() for x in xs])):
        check(y, reference(x), bound(dtype, dtype != torch.bfloat16))


@pytest.mark.parametrize("dtype", DTYPES)
def test_step_of_a_long_list(ta, dtype):
    """More than a launch takes, sides either side of 64, empty ones between them."""
    shapes = [((20, 70, 65, 200)[i % 4], (90, 64, 33, 130, 71)[i % 5]) for i in range(40)]
    shapes[11], shapes[25] = (0, 40), (40, 0)
    g = torch.Generator().manual_seed(31)
    ws = [(torch.randn(s, generator=g) * 0.02).to(dtype) for s in shapes]
    gs = [gradient(*s, dtype, 32 + i) if s[0] and s[1] else torch.zeros(s, dtype=dtype) for i, s in enumerate(shapes)]
    ms = [torch.zeros(s) for s in shapes]
    gw, gg, gm = ([t.cuda() for t in ts] for ts in (ws, gs, ms))
    ta.muon_(gw, gg, gm, lr=0.1, weight_decay=0.1)
    for w, gr, m, w2, m2 in zip(ws, gs, ms, gw, gm):
        if not w.numel():
            continue
        o, want_m = step_reference(w, gr, m, 0.1, 0.1, 0.95, True)
        assert (m2.cpu().double() - want_m).abs().le(want_m.abs() * 2.0 ** -22 + gr.double().abs() * 2.0 ** -22).all()
        want = (1 - 0.1 * 0.1) * w.double() - 0.1 * o
        off = (w2.cpu().double() - want).norm().item()
        assert off <= 0.1 * o.norm().item() * (PRECISE if dtype != torch.bfloat16 else HALF) + want.norm().item() * (ROUNDING[dtype] + 2.0 ** -22)


def test_singular_values(ta):
    """What the step is for: every direction that the momentum has comes out at about the same length.  The
    polynomial of five iterations maps every singular value from 3e-3 of the norm to 1 of it to between .65 and 1.25."""
    x = gradient(200, 600, torch.float32, 60, "even")
    s = torch.linalg.svdvals(ta.orthogonalize(x.cuda()).cpu().double())
    assert 0.6 <= s.min().item() and s.max().item() <= 1.3
    assert math.isclose((s ** 2).sum().item(), ta.orthogonalize(x.cuda()).double().norm().item() ** 2, rel_tol=1e-6)


def test_gradient_of_zero_keeps_a_weight(ta):
    """A zero momentum has no direction: the weight only decays."""
    w = torch.randn(70, 90, generator=torch.Generator().manual_seed(61)).cuda()
    want = w * (1 - 0.1 * 0.5)
    m = torch.zeros_like(w)
    ta.muon_([w], [torch.zeros_like(w)], [m], lr=0.1, weight_decay=0.5)
    assert (w - want).abs().le(want.abs() * 2.0 ** -22).all() and not m.any()


# few tiles and long sums: workgroups share a tile
WIDE = [[(64, 4096)], [(1, 5000)], [(9000, 40)], [(70, 20000)], [(600, 5000)], [(1030, 9000)], [(256, 16384), (33, 900), (700, 1000)],
        [(64, 1024), (2000, 65), (128, 128), (300, 3000)]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shapes", WIDE)
def test_long_and_narrow(ta, shapes, dtype):
    xs = [gradient(*s, dtype, 70 + i, device="cuda") for i, s in enumerate(shapes)]
    got = ta.orthogonalize(xs)
    for x, y in zip(xs, got):
        check(y, reference(x), bound(dtype, dtype == torch.float32 or min(x.shape) < 64))
    for _ in range(3):  # whichever workgroup is the last one
        assert all(torch.equal(a, b) for a, b in zip(got, ta.orthogonalize(xs)))


def test_graph_of_shared_tiles(ta):
    x = gradient(80, 6000, torch.bfloat16, 80).cuda()
    other = gradient(80, 6000, torch.bfloat16, 81).cuda()
    want = ta.orthogonalize(x), ta.orthogonalize(other)
    static = x.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ta.orthogonalize(static)
    for i in (0, 1, 1, 0, 1):
        static.copy_((x, other)[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
        assert torch.equal(ta.orthogonalize((x, other)[i]), want[i])
