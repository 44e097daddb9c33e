"""Embedding lookup and its gradient on the GPU, against 64 bits."""

import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def t():
    import torchft_amd
    return torchft_amd


def check(t, ids, table, scale=1.0, padding=None, id_dtype=torch.int64, seed=1):
    """CPU tensors in; the table's gradient is the whole table."""
    dtype, (vocab, cols) = table.dtype, table.shape
    leaf = table.cuda().requires_grad_()
    y = t.embedding(ids.to(id_dtype).cuda(), leaf, scale, padding)
    inside = (ids >= 0) & (ids < vocab)
    rows = torch.zeros(*ids.shape, cols, dtype=torch.float64)
    rows[inside] = table.double()[ids[inside].long()]
    factor = float(torch.tensor(scale, dtype=torch.float32))
    ref.close(y, rows * factor, (rows * factor).abs() * ref.U, dtype)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(seed)).to(dtype)
    dtable, = torch.autograd.grad(y, leaf, dy.cuda())
    if padding is not None:
        inside = inside & (ids != padding)
    want, size, count = (torch.zeros(vocab, w, dtype=torch.float64) for w in (cols, cols, 1))
    some = dy.double()[inside]
    want.index_add_(0, ids[inside].long(), some)
    size.index_add_(0, ids[inside].long(), some.abs())
    count.index_add_(0, ids[inside].long(), torch.ones(some.shape[0], 1, dtype=torch.float64))
    ref.close(dtable, want * factor, size * abs(factor) * (count + 2) * ref.U, dtype)
    return dtable


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("vocab,cols,n", [(1, 1, 1), (5, 3, 40), (300, 64, 31), (300, 65, 33), (1000, 130, 257), (700, 1000, 300), (257, 2050, 100),
                                          (50, 4099, 64), (70000, 9, 4097), (65536, 16, 5000), (255, 31, 16384), (256, 40, 17000), (90000, 24, 20000)])
def test_embedding(t, vocab, cols, n, dtype):
    g = torch.Generator().manual_seed(vocab + n)
    table = torch.randn(vocab, cols, generator=g).to(dtype)
    even = torch.randint(0, vocab, (n,), generator=g)
    text = (vocab ** torch.rand(n, generator=g, dtype=torch.float64) - 1).long().clamp(0, vocab - 1)
    check(t, even, table, 1.0)
    check(t, text, table, 3.3, id_dtype=torch.int32)
    check(t, torch.full((n,), vocab // 2), table, 0.5)  # one token all over
    check(t, text, table, -1.0, padding=0)


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_outside(t, dtype):
    """A part of a vocabulary: numbers below and above have zeros and no gradient, the largest ones too."""
    table = torch.randn(100, 70).to(dtype)
    ids = torch.randint(-50, 200, (6, 70), generator=torch.Generator().manual_seed(3))
    ids[0, :4] = torch.tensor([2 ** 31 - 1, -2 ** 31, 100, -1])
    check(t, ids, table)
    check(t, ids, table, id_dtype=torch.int32)
    wide = ids.clone()
    wide[0, :3] = torch.tensor([2 ** 62, -2 ** 62, 2 ** 32 + 5])
    check(t, wide, table)
    check(t, torch.full((40,), -1), table)


def test_skewed_and_long(t):
    """Two tokens that alternate, runs that end with their chunks, and runs of exactly one chunk and of several."""
    g = torch.Generator().manual_seed(5)
    table = torch.randn(40, 48, generator=g)
    for n in (32, 64, 4096, 8192, 8193, 40000):
        chunk = 32
        while chunk * chunk * 8 < n:
            chunk *= 2
        check(t, torch.arange(n) % 2, table)
        check(t, (torch.arange(n) // chunk) % 40, table)
        check(t, ((torch.arange(n) + chunk // 2) // chunk) % 40, table)
        check(t, (torch.arange(n) // (3 * chunk)) % 40, table)


@pytest.mark.parametrize("n, cols", [(8192, 512), (8192, 4100), (8193, 2100), (40000, 512), (270001, 512)])
def test_long_runs(t, n, cols):
    """Runs beside the borders of 16, 64 and 256 tokens, at sizes where those are taken; whole numbers add up exactly in any order."""
    rows = n // 16 + 2
    table = torch.zeros(rows, cols, device="cuda", requires_grad=True)
    dy = torch.randint(-2, 3, (n, cols), device="cuda", dtype=torch.float32)  # sums below 2^24
    at = torch.arange(n, device="cuda")
    for run in (16, 64, 256):
        for ids in (at // run, (at + run // 2) // run, at // (3 * run), (at // run).clamp(max=3), at * 0 + 7):
            ids = ids[torch.randperm(n, device="cuda")]
            got, = torch.autograd.grad(t.embedding(ids, table), table, dy)
            assert torch.equal(got, torch.zeros(rows, cols, device="cuda").index_add_(0, ids, dy))


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_orders(t, dtype):
    """Tables inside wider ones and transposed, numbers in any order, no tokens, no columns, more dimensions."""
    big = torch.randn(60, 90).to(dtype)
    ids = torch.randint(0, 30, (7, 8), generator=torch.Generator().manual_seed(1))
    for table in (big[10:50, 3:70], big.t()[:50], big[::2], big[:30, :1]):
        on = big.cuda().as_strided(table.shape, table.stride(), table.storage_offset())
        y = t.embedding(ids.cuda().t(), on)
        assert torch.equal(y.cpu(), table[ids.t()])
        leaf = on.detach().requires_grad_()
        d, = torch.autograd.grad(t.embedding(ids.cuda().t(), leaf).float().sum(), leaf)
        count = torch.bincount(ids.flatten(), minlength=table.shape[0]).to(dtype)
        assert torch.equal(d.cpu(), count[:, None].expand(table.shape))
    leaf = big.cuda().requires_grad_()
    y = t.embedding(torch.empty(0, 3, dtype=torch.int64, device="cuda"), leaf)
    assert y.shape == (0, 3, 90) and not torch.autograd.grad(y.sum(), leaf)[0].any()
    y = t.embedding(torch.tensor(4, device="cuda"), leaf, 2.0)
    assert torch.equal(y.cpu(), big[4] * 2)
    assert t.embedding(ids.cuda(), big.cuda()[:, :0]).shape == (7, 8, 0)
    assert not t.embedding(ids.cuda(), big.cuda()[:0]).any()


def test_same_bits_twice(t):
    """Sums have one order."""
    table = torch.randn(500, 256, device="cuda", requires_grad=True)
    ids = torch.randint(0, 500, (9000,), device="cuda").square() // 500
    dy = torch.randn(9000, 256, device="cuda")
    a, b = (torch.autograd.grad(t.embedding(ids, table), table, dy)[0] for _ in range(2))
    assert torch.equal(a, b)


def test_graph(t):
    """Replays with other tokens, between eager calls of the same leaf."""
    table = torch.randn(3000, 130, device="cuda", requires_grad=True)
    ids, dy = torch.randint(0, 3000, (20000,), device="cuda"), torch.randn(20000, 130, device="cuda")

    def step():
        y = t.embedding(ids, table, 2.0)
        return y.detach(), torch.autograd.grad(y, table, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2, 3):
        ids.copy_(torch.randint(0, 3000, (20000,), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step(), out))
        torch.cuda.synchronize()
