"""The row operators under what programs put around their calls: hooks of saved tensors, checkpoints, two threads, gradients that are
expanded or strided, tensors kept in bits, a compiler that leaves them to run as they are."""

import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def t():
    import torchft_amd
    return torchft_amd


def inputs(seed, tokens=300, cols=136, k=2, experts=5, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g).to(dtype).cuda().requires_grad_()  # noqa: E731
    ids = torch.randint(0, 90, (tokens,), generator=g).cuda()
    chosen = torch.randint(-1, experts, (tokens, k), generator=g).cuda()
    mix = torch.rand(tokens, k, generator=g).cuda().requires_grad_()
    return ids, chosen, (normal(90, cols), normal(cols), normal(tokens, cols), mix)


def step(t, ids, chosen, table, weight, residual, mix):
    """All operators with a gradient, one behind the other."""
    x = t.embedding(ids, table, scale=2.0)
    y, h = t.rms_norm(x, weight, residual)
    order = t.sort_by_expert(chosen, 5)
    back = t.combine(t.dispatch(y, order) * 2, order, mix)
    return t.dropout(back, 0.25, 7, residual=h)


def want(t, ids, chosen, leaves, dy):
    z = step(t, ids, chosen, *leaves)
    return (z, *torch.autograd.grad(z, leaves, dy))


def same(got, expected):
    assert all(torch.equal(a, b) for a, b in zip(got, expected, strict=True))


def test_hooks(t):
    """Saved tensors kept on the host, as a list of numbers' bits, and given back."""
    ids, chosen, leaves = inputs(1)
    dy = torch.randn(300, 136, device="cuda").bfloat16()
    expected = want(t, ids, chosen, leaves, dy)
    packed = []

    def pack(v):
        packed.append(v.shape)
        return v.cpu()
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda v: v.cuda()):
        z = step(t, ids, chosen, *leaves)
    assert len(packed) >= 8
    same((z, *torch.autograd.grad(z, leaves, dy)), expected)
    with torch.autograd.graph.save_on_cpu():
        z = step(t, ids, chosen, *leaves)
    same((z, *torch.autograd.grad(z, leaves, dy)), expected)
    seen = []
    z = step(t, ids, chosen, *leaves)
    z.register_hook(lambda g: seen.append(g) or g * 2)
    half = torch.autograd.grad(z, leaves, dy / 2)
    same((z, *half), expected)
    assert len(seen) == 1


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpoint(t, reentrant):
    ids, chosen, leaves = inputs(2)
    dy = torch.randn(300, 136, device="cuda").bfloat16()
    expected = want(t, ids, chosen, leaves, dy)
    z = checkpoint(lambda *v: step(t, ids, chosen, *v), *leaves, use_reentrant=reentrant)
    z.backward(dy)
    same((z, *(v.grad for v in leaves)), expected)


def test_selective_checkpoint(t):
    """A mode that keeps some results and makes the others again, the operators' among them."""
    from torch.utils.checkpoint import create_selective_checkpoint_contexts
    ids, chosen, leaves = inputs(3)
    dy = torch.randn(300, 136, device="cuda").bfloat16()
    expected = want(t, ids, chosen, leaves, dy)
    z = checkpoint(lambda *v: step(t, ids, chosen, *v), *leaves, use_reentrant=False,
                   context_fn=lambda: create_selective_checkpoint_contexts([torch.ops.aten.mul.Tensor]))
    z.backward(dy)
    same((z, *(v.grad for v in leaves)), expected)


def test_threads(t):
    """Four threads, a stream each, on tensors of their own."""
    sets = []
    for seed in range(4):
        ids, chosen, leaves = inputs(10 + seed, tokens=200 + 3000 * seed)
        dy = torch.randn(200 + 3000 * seed, 136, device="cuda").bfloat16()
        sets.append((ids, chosen, leaves, dy, [v.detach().clone() for v in want(t, ids, chosen, leaves, dy)]))
    torch.cuda.synchronize()
    errors = []

    def body(ids, chosen, leaves, dy, expected):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got = want(t, ids, chosen, leaves, dy)
                stream.synchronize()
                same(got, expected)
        except BaseException as error:  # noqa: BLE001
            errors.append(error)
    threads = [threading.Thread(target=body, args=one) for one in sets]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    torch.cuda.synchronize()
    assert not errors, errors[0]


def test_gradients_in_any_order(t):
    ids, chosen, leaves = inputs(4)
    wide = torch.randn(136, 600, device="cuda").bfloat16()
    for dy in (wide.t()[::2], wide[:1, :1].expand(300, 136), wide[:, 0].expand(300, 136), torch.randn(300, 272, device="cuda").bfloat16()[:, ::2]):
        z = step(t, ids, chosen, *leaves)
        got = torch.autograd.grad(z, leaves, dy)
        same((z, *got), want(t, ids, chosen, leaves, dy.contiguous()))


def test_accumulated(t):
    """Gradients of two passes add up in the leaves, each its own memory."""
    ids, chosen, leaves = inputs(5, dtype=torch.float32)
    dy = torch.randn(300, 136, device="cuda")
    _, *once = want(t, ids, chosen, leaves, dy)
    for _ in range(2):
        step(t, ids, chosen, *leaves).backward(dy)
    same([v.grad for v in leaves], [2 * v for v in once])
    x, r = (torch.randn(40, 50, device="cuda", requires_grad=True) for _ in range(2))
    y, h = t.rms_norm(x, None, r)
    (y.sum() + h.sum()).backward()
    assert x.grad.data_ptr() != r.grad.data_ptr()
    kept = r.grad.clone()
    x.grad.zero_()
    assert torch.equal(r.grad, kept)


def test_compiled(t):
    """A compiler breaks its graph at the calls, and they run."""
    ids, chosen, leaves = inputs(6)
    dy = torch.randn(300, 136, device="cuda").bfloat16()
    expected = want(t, ids, chosen, leaves, dy)
    z = torch.compile(lambda *v: step(t, ids, chosen, *v), backend="eager")(*leaves)
    same((z, *torch.autograd.grad(z, leaves, dy)), expected)


def test_inference(t):
    ids, chosen, leaves = inputs(7)
    expected = step(t, ids, chosen, *leaves)
    with torch.inference_mode():
        z = step(t, ids, chosen, *leaves)
        assert torch.equal(z, expected) and not z.requires_grad
    with torch.no_grad():
        assert torch.equal(step(t, ids, chosen, *leaves), expected)
