"""The row operators past 2^31 elements, on rows and numbers of tokens that take the launches for large sizes."""

import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu

ROWS, COLS = 524300, 4096  # 2^31 elements and 12 rows more


@pytest.fixture(scope="module")
def t():
    import torchft_amd
    return torchft_amd


@pytest.fixture(autouse=True)
def memory():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB of GPU memory")
    yield
    torch.cuda.empty_cache()


def far(dtype=torch.bfloat16, rows=ROWS, cols=COLS):
    x = torch.zeros(rows, cols, dtype=dtype, device="cuda")
    x[-20:] = torch.randn(20, cols, generator=torch.Generator().manual_seed(1)).to(dtype)
    return x


def test_norm(t):
    x, w = far().requires_grad_(), torch.ones(COLS, device="cuda", dtype=torch.bfloat16)
    y, h = t.rms_norm(x, w, x.detach())
    want, want_h, _ = ref.norm(x.detach()[-20:].cpu(), w.cpu(), x.detach()[-20:].cpu(), 1e-6)
    assert torch.equal(h.detach()[-20:].cpu(), want_h) and not y[:-20].any()
    ref.close(y[-20:], want, ref.norm_error(want, COLS), torch.bfloat16)
    dy = far()
    dx, = torch.autograd.grad(y, x, dy)
    want, _, error, _ = ref.norm_backward(dy[-20:].cpu(), None, want_h, w.cpu(), 1e-6)
    ref.close(dx[-20:], want, error, torch.bfloat16)
    rows = t.rms_norm_fp8(x.detach(), w)
    values = rows.dequantize()
    assert not values[:-20].any()
    alone = t.rms_norm_fp8(x.detach()[-20:], w)
    assert torch.equal(values[-20:], alone.dequantize()) and torch.equal(rows.scales[-20:], alone.scales)


def test_dropout(t):
    x = torch.ones(ROWS * COLS + 5, dtype=torch.bfloat16, device="cuda")
    y = t.dropout(x, 0.5, 11, 3)
    first = (ROWS * COLS - 24) // 8
    # the generator's numbers of the last blocks: the counter begins there
    keep = []
    for block in range(first, first + 4):
        c, k = [block & 0xFFFFFFFF, block >> 32, 3, 0], [11, 0]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [b >> 32 ^ c[1] ^ k[0], b & 0xFFFFFFFF, a >> 32 ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [k[0] + 0x9E3779B9 & 0xFFFFFFFF, k[1] + 0xBB67AE85 & 0xFFFFFFFF]
        keep += [n >= 32768 for word in c for n in (word & 0xFFFF, word >> 16)]
    assert torch.equal(y[first * 8:].cpu().float(), torch.tensor(keep[:29]).float() * 2)


def test_embedding(t):
    table = far().requires_grad_()
    ids = torch.tensor([ROWS - 1, 3, ROWS - 20, ROWS - 1], device="cuda")
    y = t.embedding(ids, table)
    assert torch.equal(y, table.detach()[ids])
    d, = torch.autograd.grad(y, table, torch.ones_like(y))
    assert (d[-1] == 2).all() and (d[-20] == 1).all() and (d[3] == 1).all()
    assert int((d != 0).any(1).sum()) == 3


def test_experts(t):
    tokens, k = ROWS // 2, 2
    x = far(rows=tokens).requires_grad_()
    g = torch.Generator("cuda").manual_seed(1)
    order = t.sort_by_expert(torch.randint(0, 16, (tokens, k), device="cuda", generator=g), 16)
    rows = t.dispatch(x, order)
    places = order.position[-20:].long()
    assert torch.equal(rows[places.flatten()], x[-20:].repeat_interleave(k, 0))
    assert int((rows != 0).any(1).sum()) == 20 * k
    y = t.combine(rows, order)
    ref.close(y[-20:], x.detach()[-20:].cpu().double() * 2, torch.zeros(20, COLS, dtype=torch.float64), torch.bfloat16)
    dy = far(rows=tokens)
    dx, = torch.autograd.grad(y, x, dy)
    assert torch.equal(dx, dy * 2)


@pytest.mark.parametrize("cols,sizes", [(3, ((40000, 300), (9000001, 5000), (34000001, 300))), (8, ((600001, 70000), (5000001, 300), (17000001, 300))),
                                        (40, ((40000, 300), (900001, 70000), (3500001, 2000))), (100, ((600001, 1000), (1400001, 600000))),
                                        (300, ((200001, 1000), (600001, 270000)))])
def test_many_tokens(t, cols, sizes):
    """Chunks of 16, 64 and 256 tokens of every number of lanes, sorts of more tiles than count for themselves, and of three passes."""
    for n, vocab in sizes:
        table = torch.zeros(vocab, cols, device="cuda", requires_grad=True)
        ids = torch.randint(0, vocab, (n,), device="cuda", generator=torch.Generator("cuda").manual_seed(n)).square() // vocab
        dy = torch.randint(-8, 9, (n, cols), device="cuda").float()  # sums of whole numbers are exact, in any order
        d, = torch.autograd.grad(t.embedding(ids, table), table, dy)
        assert torch.equal(d, torch.zeros(vocab, cols, device="cuda").index_add_(0, ids, dy))


@pytest.mark.parametrize("experts", [7, 255, 300])
def test_many_choices(t, experts):
    chosen = torch.randint(-1, experts, (150001, 3), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    got = t.sort_by_expert(chosen, experts)
    key = torch.where(chosen < 0, experts, chosen).flatten()
    order = torch.sort(key, stable=True).indices
    assert torch.equal(got.order.long(), order)
    assert torch.equal(got.position.flatten()[order].cpu(), torch.arange(key.numel(), dtype=torch.int32))
    assert torch.equal(got.offsets.cpu(), torch.searchsorted(key[order].cpu(), torch.arange(experts + 1)).int())
