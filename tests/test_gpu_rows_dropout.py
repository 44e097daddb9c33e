"""Dropout on the GPU: the generator's numbers, the sums, gradients, seeds in memory."""

import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def t():
    import torchft_amd
    return torchft_amd


def want_of(x, p, seed, offset, residual=None):
    """(64-bit values, what stays, how far fp32 may be)."""
    threshold = round(p * 65536)
    keep = (ref.bits16(seed, offset, x.numel()) >= threshold).reshape(x.shape)
    factor = 65536 / (65536 - threshold) if threshold < 65536 else 0.0
    y = torch.where(keep, x.double() * factor, 0.0)
    error = y.abs() * 2 * ref.U
    if residual is not None:
        y = y + residual.double()
        error = error + y.abs() * ref.U + error * ref.U
    return y, keep, error


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 15, 511, 4096, 4097, 8200, 12345])
def test_dropout(t, n, dtype):
    g = torch.Generator().manual_seed(n)
    x, r, dy = (torch.randn(n, generator=g).to(dtype) for _ in range(3))
    for p, seed, offset in ((0.1, 5, 0), (0.5, 2 ** 63 - 1, 2 ** 40 + 3), (0.3, -2, -7)):
        leaf, res = x.cuda().requires_grad_(), r.cuda().requires_grad_()
        y = t.dropout(leaf, p, seed, offset)
        want, keep, error = want_of(x, p, seed % 2 ** 64, offset % 2 ** 64)
        ref.close(y, want, error, dtype)
        assert torch.equal(y.detach().cpu() != 0, keep & (x != 0))
        dx, = torch.autograd.grad(y, leaf, dy.cuda())
        want, _, error = want_of(dy, p, seed % 2 ** 64, offset % 2 ** 64)
        ref.close(dx, want, error, dtype)
        z = t.dropout(leaf, p, seed, offset, residual=res)
        want, _, error = want_of(x, p, seed % 2 ** 64, offset % 2 ** 64, r)
        ref.close(z, want, error, dtype)
        both = torch.autograd.grad(z, (leaf, res), dy.cuda())
        assert torch.equal(both[0], dx) and torch.equal(both[1].cpu(), dy)


def test_probability(t):
    """No element, every element, and as many as p says: 2^20 draws of variance p (1 - p), five deviations."""
    x = torch.ones(1 << 20, device="cuda")
    assert torch.equal(t.dropout(x, 0.0, 1), x)
    assert not t.dropout(x, 1.0, 1).any()
    assert not t.dropout(torch.full_like(x, float("inf")), 1.0, 1).any()
    for p in (0.01, 0.25, 0.9):
        lost = (t.dropout(x, p, 3) == 0).sum().item()
        assert abs(lost - p * x.numel()) <= 5 * (p * (1 - p) * x.numel()) ** 0.5 + x.numel() / 65536
    a, b = t.dropout(x, 0.5, 3, 0), t.dropout(x, 0.5, 3, 1)
    assert abs((a == b).float().mean().item() - 0.5) <= 5 * 0.5 / 1024


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_orders(t, dtype):
    """The mask goes by an element's place in row-major order, whatever the memory's; any dimensions, none, no elements."""
    big = torch.randn(40, 90).to(dtype)
    for view in (big.t(), big[3:9, 1:], big[:, ::4], big[:1].expand(5, -1), big.view(4, 10, 90).transpose(0, 2), big[0, 0], big[:0], big[7, 1:9]):
        on = view.cuda() if not view.numel() else big.cuda().as_strided(view.shape, view.stride(), view.storage_offset())
        y = t.dropout(on, 0.4, 9, residual=on)
        want, _, error = want_of(view.contiguous(), 0.4, 9, 0, view.contiguous())
        ref.close(y, want, error, dtype)


def test_seed_in_memory(t):
    """The same numbers as from the seed itself; another seed after a change; gradients of the forward pass's seed."""
    x = torch.randn(5000, device="cuda", requires_grad=True)
    seed = torch.tensor([77], device="cuda")
    y = t.dropout(x, 0.5, seed, 4)
    assert torch.equal(y, t.dropout(x, 0.5, 77, 4))
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0] != 0, y != 0)
    y = t.dropout(x, 0.5, seed, 4)
    seed += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    assert torch.equal(t.dropout(x, 0.5, seed, 4), t.dropout(x, 0.5, 78, 4))


def test_graph(t):
    """A captured step draws what the seed in memory says at every replay."""
    x = torch.randn(3000, device="cuda", requires_grad=True)
    seed, dy = torch.tensor([1], device="cuda"), torch.randn(3000, device="cuda")

    def step():
        y = t.dropout(x, 0.2, seed)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for s in (1, 8, 2 ** 50):
        seed.fill_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], t.dropout(x, 0.2, s).detach())
        assert torch.equal(out[1], t.dropout(dy, 0.2, s))
        torch.cuda.synchronize()
