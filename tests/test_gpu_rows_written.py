"""The gradient of a table is written whole and nowhere else: every number of it, of memory that held NaN, and none behind or before."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
GUARD = 4096


@pytest.mark.parametrize("dtype,vocab,cols,n", [
    (torch.bfloat16, 8193, 1, 9000), (torch.bfloat16, 1001, 1113, 9000), (torch.float16, 50257, 1201, 9000), (torch.bfloat16, 513, 7681, 9000),
    (torch.float32, 262145, 4097, 9000), (torch.float32, 300001, 4129, 140000), (torch.bfloat16, 700, 33, 9000), (torch.bfloat16, 700, 33, 8000),
    (torch.float16, 300, 7, 200), (torch.bfloat16, 300, 7, 9000), (torch.float32, 5, 1, 20000), (torch.bfloat16, 65537, 3, 0)])
def test_table(dtype, vocab, cols, n):
    from torchft_amd import _lib
    lib = _lib.load()
    whole = torch.full((vocab * cols + 2 * GUARD,), float("nan"), dtype=dtype, device="cuda")
    bits = whole.view(torch.int16 if dtype.itemsize == 2 else torch.int32)
    before = int(bits[0])
    table = whole[GUARD:GUARD + vocab * cols]
    g = torch.Generator().manual_seed(vocab)
    ids = torch.randint(0, max(1, vocab - 3), (n,), generator=g).cuda()  # the last rows have no token
    dy = torch.randint(-2, 3, (n, cols), generator=g).to(dtype).cuda()
    size = lib.tftq_embedding_backward_workspace(DTYPES[dtype], n, vocab, cols)
    workspace = torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert lib.tftq_embedding_backward(DTYPES[dtype], 8, ids.data_ptr(), n, -1, dy.data_ptr(), vocab, cols, 1.0, table.data_ptr(), workspace.data_ptr(), size,
                                       0, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert bool((bits[:GUARD] == before).all()) and bool((bits[GUARD + vocab * cols:] == before).all())
    assert not table.isnan().any(), f"{int(table.isnan().sum())} numbers were not written"
    names, where = ids.unique(return_inverse=True)
    sums = torch.zeros(names.numel(), cols, device="cuda").index_add_(0, where, dy.float())  # of small whole numbers: exact
    table = table.view(vocab, cols)
    assert torch.equal(table[names].float(), sums.to(dtype).float())
    assert int(table.count_nonzero()) == int(sums.count_nonzero())
