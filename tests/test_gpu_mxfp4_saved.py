"""What a layer keeps for its backward pass is autograd's: released, seen by hooks, refused a second time."""

import gc

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from test_gpu_mxfp4 import values

pytestmark = pytest.mark.gpu

T, N, K = 130, 64, 300


@pytest.fixture(scope="module")
def mx():
    import torchft_amd
    return torchft_amd


def inputs():
    x, w, dy = (values(*s, torch.bfloat16, 130 + i).cuda() for i, s in enumerate(((T, K), (N, K), (T, N))))
    return x.requires_grad_(), w.requires_grad_(), dy


def gradients(mx):
    x, w, dy = inputs()
    mx.linear_mxfp4(x, w).backward(dy)
    return x.grad, w.grad


def test_released_after_backward(mx):
    """With the result still held."""
    mx.linear_mxfp4(*inputs()[:2])
    x = torch.randn(4096, 1024, device="cuda", requires_grad=True)
    w = torch.randn(512, 1024, device="cuda", requires_grad=True)
    gc.collect()
    before = torch.cuda.memory_allocated()
    y = mx.linear_mxfp4(x, w)
    held = torch.cuda.memory_allocated() - before - y.numel() * 4
    assert held >= (4096 + 512) * 1024 // 2  # both operands' codes
    y.backward(torch.ones_like(y))
    left = torch.cuda.memory_allocated() - before - y.numel() * 4 - (x.numel() + w.numel()) * 4
    assert left <= 4096, f"{left} bytes are still held"


def test_a_second_backward(mx):
    x, w, dy = inputs()
    y = mx.linear_mxfp4(x, w)
    y.backward(dy, retain_graph=True)
    once = x.grad.clone(), w.grad.clone()
    y.backward(dy)
    assert torch.equal(x.grad, 2 * once[0]) and torch.equal(w.grad, 2 * once[1])
    with pytest.raises(RuntimeError, match="a second time"):
        y.backward(dy)


def test_hooks(mx):
    """They see both matrices, may keep them elsewhere and bring them back."""
    want = gradients(mx)
    packed = []

    def pack(t):
        packed.append(t.numel())
        return t.cpu()
    x, w, dy = inputs()
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
        y = mx.linear_mxfp4(x, w)
    assert sorted(packed) == sorted((mx.quantize_mxfp4(x.detach(), 0).buffer.numel(), mx.quantize_mxfp4(w.detach(), 0).buffer.numel()))
    y.backward(dy)
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])
    x, w, dy = inputs()
    with torch.autograd.graph.save_on_cpu():
        y = mx.linear_mxfp4(x, w)
    y.backward(dy)
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointing(mx, reentrant):
    """The gradients of a layer that is computed again; nothing of it is kept meanwhile."""
    want = gradients(mx)
    x, w, dy = inputs()
    y = checkpoint(mx.linear_mxfp4, x, w, use_reentrant=reentrant)
    y.backward(dy)
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])
    x = torch.randn(4096, 1024, device="cuda", requires_grad=True)
    w = torch.randn(512, 1024, device="cuda", requires_grad=True)
    gc.collect()
    before = torch.cuda.memory_allocated()
    y = checkpoint(mx.linear_mxfp4, x, w, use_reentrant=reentrant)
    assert torch.cuda.memory_allocated() - before - y.numel() * 4 <= 4096


@pytest.mark.parametrize("wants", ["x", "w"])
def test_one_gradient(mx, wants):
    both = gradients(mx)
    x, w, dy = inputs()
    (w if wants == "x" else x).requires_grad_(False)
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t.shape) or t, lambda t: t):
        y = mx.linear_mxfp4(x, w)
    assert len(packed) == 1
    y.backward(dy)
    assert torch.equal(x.grad, both[0]) and w.grad is None if wants == "x" else torch.equal(w.grad, both[1]) and x.grad is None
