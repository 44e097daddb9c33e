"""Embedding: numbers outside the table under any scale, and runs of tokens beside the borders of the chunks that a size takes."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [float("inf"), float("-inf"), float("nan"), 3.4e38])
def test_zeros_outside(scale):
    import torchft_amd as t
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        for cols in (3, 40, 777):
            table = torch.ones(5, cols, device="cuda", dtype=dtype)
            y = t.embedding(torch.tensor([5, 2, -1, 2 ** 40, 0], device="cuda"), table, scale)
            assert not y[[0, 2, 3]].any()
            for row in y[[1, 4]]:
                assert row.isnan().all() if scale != scale else torch.equal(row, (table[0].float() * scale).to(dtype))


@pytest.mark.parametrize("chunk,n,cols", [(16, 32, 48), (16, 4096, 48), (16, 8193, 48), (16, 40000, 48), (64, 40000, 450), (64, 8192, 4100), (256, 270001, 512)])
def test_runs_of_chunks(chunk, n, cols):
    """Runs of exactly one chunk, half a chunk off, of three, of one less and one more; sums of small whole numbers are exact."""
    import torchft_amd as t
    rows = n // (chunk - 1) + 2
    table = torch.zeros(rows, cols, device="cuda", requires_grad=True)
    g = torch.Generator("cuda").manual_seed(n)
    dy = torch.randint(-2, 3, (n, cols), device="cuda", generator=g).float()
    at = torch.arange(n, device="cuda")
    for ids in (at // chunk, (at + chunk // 2) // chunk, at // (3 * chunk), at // (chunk - 1), at // (chunk + 1), at % 2):
        got, = torch.autograd.grad(t.embedding(ids, table), table, dy)
        assert torch.equal(got, torch.zeros(rows, cols, device="cuda").index_add_(0, ids, dy))
