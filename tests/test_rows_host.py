"""The row operators without a GPU: what they refuse, what the C entry points check, the cases' definitions."""

import ctypes
import os

import pytest
import torch

import rows_reference as ref
import torchft_amd as t
from torchft_amd import _lib

f = torch.zeros


def order(tokens=4, k=2, experts=3):
    return t.ExpertOrder(*(f(n, dtype=torch.int32) for n in (tokens * k, (tokens, k), experts + 1)))


@pytest.mark.parametrize("call,why", [
    (lambda: t.rms_norm(3), "A tensor is required"),
    (lambda: t.rms_norm(f(())), "at least one dimension"),
    (lambda: t.rms_norm(f(2, 3, dtype=torch.float64)), "Only fp32, fp16 and bf16"),
    (lambda: t.rms_norm(f(2, 3), f(4)), "one number for every column"),
    (lambda: t.rms_norm(f(2, 3), f(1, 3)), "one number for every column"),
    (lambda: t.rms_norm(f(2, 3), f(3).half()), "type of the rows or is fp32"),
    (lambda: t.rms_norm(f(2, 3), None, f(3, 2)), "another shape"),
    (lambda: t.rms_norm(f(2, 3), None, f(2, 3).half()), "another type"),
    (lambda: t.rms_norm(f(2, 3), eps=-1.0), "eps is negative"),
    (lambda: t.rms_norm(f(2, 3), eps=float("nan")), "eps is negative"),
    (lambda: t.rms_norm(f(2, 3)), "A GPU tensor is required"),
    (lambda: t.rms_norm(f(2, 3, device="meta")), "A GPU tensor is required"),
    (lambda: t.rms_norm(f(2, 3).to_sparse()), "Only plain tensors"),
    (lambda: t.rms_norm_fp8(f(2, 3).requires_grad_()), "in 8 bits has no gradient"),
    (lambda: t.FP8Rows(f(2, 3), f(2, 1)).dequantize(), "float8_e4m3fn"),
    (lambda: t.FP8Rows(f(2, 3).to(torch.float8_e4m3fn), f(3, 1)).dequantize(), "one fp32 number for every row"),
    (lambda: t.FP8Rows(f(2, 3).to(torch.float8_e4m3fn), f(2, 1)).dequantize(torch.float64), "Only fp32, fp16 and bf16"),
    (lambda: t.dropout(f(3), 1.5, 0), "p is between"),
    (lambda: t.dropout(f(3), float("nan"), 0), "p is between"),
    (lambda: t.dropout(f(3), 0.5, f(1)), "tensor of one int64"),
    (lambda: t.dropout(f(3), 0.5, f(2, dtype=torch.int64)), "tensor of one int64"),
    (lambda: t.dropout(f(3), 0.5, 0, residual=f(4)), "another shape"),
    (lambda: t.dropout(f(3).int(), 0.5, 0), "Only fp32, fp16 and bf16"),
    (lambda: t.dropout(f(3), 0.5, 0), "A GPU tensor is required"),
    (lambda: t.embedding(f(3), f(3, 3)), "int64 or int32"),
    (lambda: t.embedding(f(3).long(), f(3)), "Only 2D"),
    (lambda: t.embedding(f(3).long(), f(3, 3), padding_idx=3), "padding_idx"),
    (lambda: t.embedding(f(3).long(), f(3, 3), padding_idx=-1), "padding_idx"),
    (lambda: t.embedding(f(3).long(), f(3, 3).double()), "Only fp32, fp16 and bf16"),
    (lambda: t.embedding(f(3).long(), f(3, 3)), "A GPU tensor is required"),
    (lambda: t.sort_by_expert(f(3, 2), 3), "int64 or int32"),
    (lambda: t.sort_by_expert(f(3, 2, 1).int(), 3), r"\[tokens\] or \[tokens, k\]"),
    (lambda: t.sort_by_expert(f(3, 2).int(), 0), "At least one expert"),
    (lambda: t.sort_by_expert(f(3, 2).int(), 3), "A GPU tensor is required"),
    (lambda: t.dispatch(f(4), order()), "Only 2D"),
    (lambda: t.dispatch(f(5, 3), order()), "another number of tokens"),
    (lambda: t.dispatch(f(4, 3).double(), order()), "1, 2 and 4 bytes"),
    (lambda: t.dispatch(f(4, 3), t.ExpertOrder(f(8), f(4, 2), f(4))), "one of sort_by_expert"),
    (lambda: t.dispatch(f(4, 3), order()), "A GPU tensor is required"),
    (lambda: t.combine(f(7, 3), order()), "not as many rows as choices"),
    (lambda: t.combine(f(8, 3), order(), f(4, 3)), "one number for every choice"),
    (lambda: t.combine(f(8, 3), order(), f(2, 4)), "one number for every choice"),
    (lambda: t.combine(f(8, 3), order(), f(4, 2).half()), "type of the rows or are fp32"),
    (lambda: t.combine(f(8, 3), order()), "A GPU tensor is required"),
])
def test_refusals(call, why):
    with pytest.raises(AssertionError, match=why):
        call()


@pytest.mark.parametrize("call", [lambda: t.dropout(f(3), "a", 0), lambda: t.dropout(f(3), 0.5, 1.5), lambda: t.embedding(f(3).long(), f(3, 3), "x"),
                                  lambda: t.sort_by_expert(f(3).int(), 2.0), lambda: t.rms_norm(f(2, 3), eps=None)])
def test_types(call):
    with pytest.raises(TypeError):
        call()


def test_wrapped_tensors_are_refused():
    from torch.autograd import forward_ad
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(), pytest.raises(AssertionError, match="Only plain tensors"):
        t.rms_norm(torch.zeros(2, 3))
    with pytest.raises(AssertionError, match="Only plain tensors"):
        torch.func.vmap(t.rms_norm)(torch.zeros(2, 3))
    with forward_ad.dual_level(), pytest.raises(AssertionError, match="Forward-mode"):
        t.rms_norm(forward_ad.make_dual(torch.zeros(2, 3), torch.zeros(2, 3)))


def test_c_entries_check_before_they_launch():
    """Sizes, types, pointers, strides, workspaces: no device is touched."""
    lib = _lib.load()
    p = 4096  # an address that is never read
    norm = lambda **k: lib.tftq_rms_norm(*{**dict(dtype=2, wdtype=2, x=p, xs=8, xg=2, xgs=0, r=None, rs=0, w=p, rows=2, cols=8, eps=1e-6, h=None, y=p, c=None,  # noqa: E731
                                                    s=None, device=-1, stream=None), **k}.values())
    assert norm(dtype=3) == -2 and norm(wdtype=1) == -2 and norm(rows=-1) == -3 and norm(cols=2 ** 31) == -3
    assert norm(x=None) == -1 and norm(xs=7) == -1 and norm(xg=0) == -1 and norm(xg=1) == -1 and norm(xg=1, xgs=7) == -1 and norm(h=p) == -1 and norm(r=p, h=p, rs=7) == -1 and norm(c=p) == -1 and norm(y=None) == -1
    assert norm(y=None, c=p) == -1 and norm(eps=-1.0) == -1 and norm(rows=0, x=None) == 0 and norm(cols=0) == 0
    back = lambda **k: lib.tftq_rms_norm_backward(*{**dict(dtype=2, wdtype=2, dy=p, dh=None, h=p, hs=8, hg=2, hgs=0, w=p, rows=2, cols=8, eps=1e-6, dx=p, dw=p, ws=p,  # noqa: E731
                                                             n=1 << 20, device=-1, stream=None), **k}.values())
    assert back(n=16) == -4 and back(ws=p + 8) == -1 and back(w=None) == -1 and back(dy=None) == -1 and back(dx=None, dw=None) == -1 and back(hs=3) == -1 and back(hg=1) == -1
    assert lib.tftq_rms_norm_backward_workspace(2, -1, 3) == -3 and lib.tftq_rms_norm_backward_workspace(7, 1, 3) == -2
    drop = lambda **k: lib.tftq_dropout(*{**dict(dtype=0, x=p, r=None, n=8, p=0.5, seed=1, at=None, offset=0, out=p, device=-1, stream=None), **k}.values())  # noqa: E731
    assert drop(dtype=5) == -2 and drop(n=-1) == -3 and drop(p=1.01) == -1 and drop(p=float("nan")) == -1 and drop(out=None) == -1 and drop(at=p + 4) == -1
    assert drop(n=0) == 0
    emb = lambda **k: lib.tftq_embedding(*{**dict(dtype=0, size=8, ids=p, n=3, table=p, vocab=4, cols=8, stride=8, scale=1.0, out=p, device=-1,  # noqa: E731
                                                    stream=None), **k}.values())
    assert emb(dtype=-1) == -2 and emb(size=2) == -1 and emb(vocab=2 ** 31) == -3 and emb(stride=7) == -1 and emb(table=None) == -1 and emb(n=0) == 0
    emb = lambda **k: lib.tftq_embedding_backward(*{**dict(dtype=0, size=8, ids=p, n=3, skip=-1, dy=p, vocab=4, cols=8, scale=1.0, dt=p, ws=p,  # noqa: E731
                                                             bytes=1 << 20, device=-1, stream=None), **k}.values())
    assert emb(bytes=8) == -4 and emb(ws=None) == -1 and emb(dt=None) == -1 and emb(cols=-1) == -3 and emb(size=1) == -1 and emb(vocab=0) == 0
    sort = lambda **k: lib.tftq_expert_sort(*{**dict(size=8, chosen=p, n=3, experts=4, order=p, position=p, offsets=p, ws=p, bytes=1 << 20, device=-1,  # noqa: E731
                                                       stream=None), **k}.values())
    assert sort(size=3) == -1 and sort(n=-1) == -3 and sort(offsets=None) == -1 and sort(n=100000, bytes=0) == -4 and sort(n=100000, ws=p + 4) == -1
    send = lambda **k: lib.tftq_dispatch(*{**dict(size=2, x=p, xs=8, tokens=3, k=2, cols=8, position=p, used=p, out=p, device=-1, stream=None), **k}.values())  # noqa: E731
    assert send(size=8) == -2 and send(xs=7) == -1 and send(tokens=2 ** 30, k=4) == -3 and send(used=None) == -1 and send(k=0) == 0
    back = lambda **k: lib.tftq_combine(*{**dict(dtype=2, wdtype=0, rows=p, rs=8, w=p, tokens=3, k=2, cols=8, position=p, used=p, out=p, device=-1,  # noqa: E731
                                                   stream=None), **k}.values())
    assert back(wdtype=1) == -2 and back(rs=3) == -1 and back(rows=None) == -1 and back(tokens=0) == 0 and back(k=0, used=None) == -1
    back = lambda **k: lib.tftq_combine_backward(*{**dict(dtype=2, wdtype=0, dy=p, ds=8, rows=p, rs=8, w=p, tokens=3, k=2, cols=8, position=p, used=p,  # noqa: E731
                                                            dr=p, dw=p, device=-1, stream=None), **k}.values())
    assert back(w=None) == -1 and back(rows=None) == -1 and back(dr=None, dw=None) == -1 and back(ds=1) == -1 and back(wdtype=1) == -2
    assert lib.tftq_fp8_rows_dequantize(4, p, p, 1, 1, p, -1, None) == -2 and lib.tftq_fp8_rows_dequantize(0, None, p, 1, 1, p, -1, None) == -1


def test_workspaces_grow_with_their_sizes():
    lib = _lib.load()
    assert lib.tftq_expert_sort_workspace(100, 8) >= 0 and lib.tftq_expert_sort_workspace(0, 8) == 0
    n = 100000
    assert lib.tftq_embedding_backward_workspace(0, n, 128256, 64) >= 8 * n + 2 * 8 * n and lib.tftq_expert_sort_workspace(n, 1000) >= 12 * n
    assert lib.tftq_expert_sort_workspace(2 ** 31, 8) == -3
    assert lib.tftq_rms_norm_backward_workspace(2, 4, 100) >= 4 * 100


def test_the_generator():
    """Known numbers of the generator: counter and key all zeros, all ones (its authors' published test vectors)."""
    def words(bits):
        return [int(bits[2 * i]) | int(bits[2 * i + 1]) << 16 for i in range(4)]
    assert words(ref.bits16(0, 0, 8)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


def test_cases_are_what_they_say():
    """Sizes, names and work of the listed and drawn cases."""
    import random
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf"))
    import more_operators as m
    cases = m.listed()
    assert len({c["name"] for c in cases}) == len(cases) <= 12
    rng = random.Random(1)
    for case in cases + [m.draw(rng) for _ in range(300)]:
        work = m.work(case)
        assert work["bytes"] > 0 and work["flops"] > 0 and case["rows"] >= 1 and case["cols"] >= 1
        assert case["k"] <= case["experts"] or case["op"] != "experts"
