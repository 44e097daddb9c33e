"""Heads inside wider rows are normed where they lie: no copy of them is made, forward or backward."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pick", [lambda v: v[:, :, 1], lambda v: v[:, :, 2, :, :50], lambda v: v[:, :, 0].transpose(1, 2).transpose(1, 2)])
def test_no_copy(pick):
    import torchft_amd as t
    wide = torch.randn(8, 512, 3, 16, 64, device="cuda")
    x = pick(wide).detach().requires_grad_()
    w = torch.ones(x.shape[-1], device="cuda", requires_grad=True)
    dy = torch.randn(x.shape, device="cuda")
    size = x.numel() * 4

    def grown(call):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        result = call()
        torch.cuda.synchronize()
        return torch.cuda.max_memory_allocated() - before, result
    t.rms_norm(x, w)
    forward, y = grown(lambda: t.rms_norm(x, w))
    assert size <= forward < 1.5 * size
    torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    backward, _ = grown(lambda: torch.autograd.grad(y, (x, w), dy))
    assert size <= backward < 1.5 * size
