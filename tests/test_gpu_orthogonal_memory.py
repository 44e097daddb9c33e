"""Lists whose matrices together need more workspace than a call takes at once."""

import pytest
import torch

from test_gpu_orthogonal import DTYPES, HALF, PRECISE, ROUNDING, bound, check, gradient, reference, step_reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ta():
    import torchft_amd
    return torchft_amd


@pytest.mark.parametrize("precise", [False, True])
def test_workspace_of_a_large_list(ta, precise):
    """A model's widest matrices: beside inputs and results 9 GiB are used, whatever the number of matrices."""
    if torch.cuda.mem_get_info()[1] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    xs = [gradient(4096, 14336, torch.bfloat16, 150, device="cuda")] * 24
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ys = ta.orthogonalize(xs, precise=precise)
    used = torch.cuda.max_memory_allocated() - before - sum(y.numel() * 2 for y in ys)
    assert used <= 9 << 30, f"{used / 2 ** 30:.1f} GiB"
    want = ta.orthogonalize(xs[0], precise=precise).double()
    for y in ys:  # the order of the additions may be that of another size of tiles
        assert (y.double() - want).norm().item() <= bound(torch.bfloat16, precise) * want.norm().item()


SHAPES = [(70, 200), (200, 70), (0, 5), (64, 64), (33, 90), (300, 130), (5, 0), (130, 300), (1, 50)]


@pytest.mark.parametrize("limit", [1, 1 << 20, 2 << 20])
def test_orthogonalize_in_parts(ta, monkeypatch, limit):
    """A matrix at a time, or a few: each result in its place."""
    import torchft_amd.muon as muon
    xs = [gradient(*s, torch.float32, 151 + i) if s[0] and s[1] else torch.zeros(s) for i, s in enumerate(SHAPES)]
    monkeypatch.setattr(muon, "_WORKSPACE", limit)
    for x, y in zip(xs, ta.orthogonalize([x.cuda() for x in xs])):
        assert y.shape == x.shape
        if x.numel():
            check(y, reference(x), bound(torch.float32, True))


@pytest.mark.parametrize("dtype", DTYPES)
def test_step_in_parts(ta, monkeypatch, dtype):
    import torchft_amd.muon as muon
    monkeypatch.setattr(muon, "_WORKSPACE", 1 << 20)
    g = torch.Generator().manual_seed(160)
    ws = [(torch.randn(s, generator=g) * 0.02).to(dtype) for s in SHAPES]
    gs = [gradient(*s, dtype, 161 + i) if s[0] and s[1] else torch.zeros(s, dtype=dtype) for i, s in enumerate(SHAPES)]
    ms = [gradient(*s, torch.float32, 171 + i) if s[0] and s[1] else torch.zeros(s) for i, s in enumerate(SHAPES)]
    gw, gg, gm = ([t.cuda() for t in ts] for ts in (ws, gs, ms))
    gw[1] = gw[1].t().contiguous().t()  # stored in another order than its gradient
    ta.muon_(gw, gg, gm, lr=0.3, weight_decay=0.2, momentum=0.9)
    for w, gr, m, w2, m2 in zip(ws, gs, ms, gw, gm):
        if not w.numel():
            continue
        o, want_m = step_reference(w, gr, m, 0.3, 0.2, 0.9, True)
        assert (m2.cpu().double() - want_m).abs().le(want_m.abs() * 2.0 ** -22 + gr.double().abs() * 2.0 ** -22).all()
        want = (1 - 0.3 * 0.2) * w.double() - 0.3 * o
        off = (w2.cpu().double() - want).norm().item()
        assert off <= 0.3 * o.norm().item() * (PRECISE if dtype != torch.bfloat16 else HALF) + want.norm().item() * (ROUNDING[dtype] + 2.0 ** -22)
