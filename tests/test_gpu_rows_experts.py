"""Tokens to experts and back on the GPU, against a sort and 64-bit sums on the CPU."""

import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def t():
    import torchft_amd
    return torchft_amd


def choices(tokens, k, experts, dropped=0.0, seed=1):
    g = torch.Generator().manual_seed(seed)
    score = torch.rand(tokens, experts, generator=g) * torch.linspace(0.5, 1, experts)
    chosen = score.topk(min(k, experts), dim=1).indices if k <= experts else torch.randint(0, experts, (tokens, k), generator=g)
    return torch.where(torch.rand(chosen.shape, generator=g) < dropped, -1, chosen)


@pytest.mark.parametrize("tokens,k,experts", [(1, 1, 1), (1, 2, 8), (0, 2, 8), (5, 3, 4), (63, 1, 2), (64, 4, 255), (128, 2, 256), (300, 3, 257),
                                              (1000, 4, 61), (4096, 4, 8), (4097, 4, 7), (5000, 4, 8), (3000, 6, 300), (17000, 1, 70000), (33, 7, 3)])
def test_sort(t, tokens, k, experts):
    """Stable, with choices that name no expert behind all; both types of numbers."""
    chosen = choices(tokens, k, min(experts, 400), 0.1) if tokens else torch.zeros(0, k, dtype=torch.int64)
    if tokens > 40:
        chosen[7, 0], chosen[9, 0], chosen[11, 0] = experts, 2 ** 31 - 1, -2 ** 31
        chosen[20, :] = experts - 1
    order, position, offsets = ref.places(chosen, experts)
    for dtype in (torch.int64, torch.int32):
        got = t.sort_by_expert(chosen.to(dtype).cuda(), experts)
        assert got.order.dtype == got.position.dtype == got.offsets.dtype == torch.int32
        assert torch.equal(got.order.cpu(), order) and torch.equal(got.position.cpu(), position) and torch.equal(got.offsets.cpu(), offsets)
        assert torch.equal(got.counts.cpu(), offsets[1:] - offsets[:-1])


def check(t, tokens, k, experts, cols, dtype, dropped, weight_dtype, stride=0):
    g = torch.Generator().manual_seed(cols)
    chosen = choices(tokens, k, experts, dropped)
    order, position, offsets = ref.places(chosen, experts)
    used, n = int(offsets[-1]), tokens * k
    x, dy = (torch.randn(tokens, cols, generator=g).to(dtype) for _ in range(2))
    rows, dsorted = (torch.randn(n, cols, generator=g).to(dtype) for _ in range(2))
    weights = torch.rand(tokens, k, generator=g).to(weight_dtype)
    at, live = position.long(), position < used
    own = t.sort_by_expert(chosen.cuda(), experts)
    leaf = x.cuda().requires_grad_()
    got = t.dispatch(leaf, own)
    want = torch.zeros(n, cols, dtype=dtype)
    want[at[live]] = x[torch.arange(tokens)[:, None].expand(-1, k)[live]]
    assert torch.equal(got.detach().cpu(), want)
    dx, = torch.autograd.grad(got, leaf, dsorted.cuda())
    each = torch.where(live[:, :, None], dsorted.double()[at], 0.0)
    ref.close(dx, each.sum(1), each.abs().sum(1) * k * ref.U, dtype)
    if stride:  # rows inside wider ones
        wide = torch.zeros(n, cols + stride, dtype=dtype, device="cuda")
        wide[:, 1:cols + 1] = rows.cuda()
        r = wide[:, 1:cols + 1].detach().requires_grad_()
    else:
        r = rows.cuda().requires_grad_()
    w = weights.cuda().requires_grad_()
    y = t.combine(r, own, w)
    each = torch.where(live[:, :, None], rows.double()[at] * weights.double()[:, :, None], 0.0)
    ref.close(y, each.sum(1), each.abs().sum(1) * (k + 1) * ref.U, dtype)
    drows, dw = torch.autograd.grad(y, (r, w), dy.cuda())
    want = torch.zeros(n, cols, dtype=torch.float64)
    token, slot = torch.arange(tokens)[:, None].expand(-1, k)[live], torch.arange(k)[None].expand(tokens, -1)[live]
    want[at[live]] = dy.double()[token] * weights.double()[token, slot][:, None]
    ref.close(drows, want, want.abs() * ref.U, dtype)
    dots = torch.where(live[:, :, None], rows.double()[at] * dy.double()[:, None], 0.0)
    ref.close(dw, dots.sum(2), dots.abs().sum(2) * (cols + 1) * ref.U, weight_dtype)
    ones = torch.where(live[:, :, None], rows.double()[at], 0.0)
    ref.close(t.combine(rows.cuda(), own), ones.sum(1), ones.abs().sum(1) * k * ref.U, dtype)


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("tokens,k,experts,cols", [(1, 1, 1, 1), (1, 2, 8, 512), (37, 3, 5, 33), (200, 2, 8, 64), (70, 6, 61, 777), (50, 8, 16, 1030),
                                                   (33, 2, 4, 2050), (20, 4, 8, 4100), (9, 2, 3, 8200), (6, 3, 4, 17000), (4000, 5, 64, 24)])
def test_there_and_back(t, tokens, k, experts, cols, dtype):
    check(t, tokens, k, experts, cols, dtype, 0.0, torch.float32)
    check(t, tokens, k, experts, cols, dtype, 0.3, dtype, stride=5)
    check(t, tokens, k, experts, cols, dtype, 1.0, torch.float32)


def test_other_elements(t):
    """Rows of bytes and of whole numbers travel as they are; rows in 8 bits with their scales."""
    chosen = choices(40, 2, 5, 0.2)
    own = t.sort_by_expert(chosen.cuda(), 5)
    order, position, offsets = ref.places(chosen, 5)
    for cols in (1, 15, 16, 33, 1000, 5003):
        for dtype in (torch.uint8, torch.int16, torch.int32):
            x = torch.randint(0, 100, (40, cols)).to(dtype)
            got = t.dispatch(x.cuda(), own).cpu()
            want = torch.zeros(80, cols, dtype=dtype)
            want[: offsets[-1]] = x[order[: offsets[-1]].long() // 2]
            assert torch.equal(got, want)
    x = torch.randn(40, 300, device="cuda")
    rows = t.rms_norm_fp8(x)
    sent = t.dispatch(rows, own)
    assert torch.equal(sent.dequantize(torch.float32), t.dispatch(rows.dequantize(torch.float32), own))


def test_masked_rows_may_hold_anything(t):
    """What lies in places without an expert, and the weights of such choices, reach no result."""
    chosen = choices(30, 2, 4, 0.5)
    own = t.sort_by_expert(chosen.cuda(), 4)
    used = int(own.offsets[-1])
    rows = torch.randn(60, 100, device="cuda")
    weights = torch.rand(30, 2, device="cuda")
    dirty, loose = rows.clone(), weights.clone()
    dirty[used:] = float("nan")
    loose[(chosen < 0).cuda()] = float("inf")
    dy = torch.randn(30, 100, device="cuda")
    results = []
    for r, w in ((rows, weights), (dirty, loose)):
        r, w = r.requires_grad_(), w.requires_grad_()
        y = t.combine(r, own, w)
        results.append((y.detach(), *torch.autograd.grad(y, (r, w), dy)))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert not results[0][1][used:].any()


def test_some_gradients(t):
    chosen = choices(30, 2, 4, 0.2)
    own = t.sort_by_expert(chosen.cuda(), 4)
    rows, weights, dy = torch.randn(60, 100, device="cuda"), torch.rand(30, 2, device="cuda"), torch.randn(30, 100, device="cuda")
    r, w = rows.clone().requires_grad_(), weights.clone().requires_grad_()
    full = torch.autograd.grad(t.combine(r, own, w), (r, w), dy)
    assert torch.equal(torch.autograd.grad(t.combine(r, own, weights), r, dy)[0], full[0])
    assert torch.equal(torch.autograd.grad(t.combine(rows, own, w), w, dy)[0], full[1])
    flat = t.sort_by_expert(chosen[:, 0].cuda(), 4)
    one = weights[:, 0].clone().requires_grad_()
    assert torch.autograd.grad(t.combine(rows[:30], flat, one).sum(), one)[0].shape == (30,)


def test_graph(t):
    """Replays with other choices, between eager calls of the same leaves."""
    chosen = choices(5000, 4, 16, 0.1).cuda()
    x = torch.randn(5000, 72, device="cuda", requires_grad=True)
    w = torch.rand(5000, 4, device="cuda", requires_grad=True)
    dy = torch.randn(5000, 72, device="cuda")

    def step():
        order = t.sort_by_expert(chosen, 16)
        y = t.combine(t.dispatch(x, order), order, w)
        return (order.position, order.offsets, y.detach(), *torch.autograd.grad(y, (x, w), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2, 3):
        chosen.copy_(choices(5000, 4, 16, 0.1, seed))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step(), out))
        torch.cuda.synchronize()
