"""Coefficients that let the iterates, or the matrices they are multiplied by, grow past what 16 bits hold at the usual scale."""

import pytest
import torch

from test_gpu_orthogonal import bound, check, gradient, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ta():
    import torchft_amd
    return torchft_amd


def rank_one(m, n, dtype, seed):
    """One singular value, which is the norm: every bound on the iterates is reached."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, 1, generator=g) @ torch.randn(1, n, generator=g) * 1e-3).to(dtype)


# Every map has a relative condition of at most 5 (a term alone, or terms of one sign): what rounding leaves of X is
# multiplied by 5 at most in an iteration, 2^-22 of it with three products and 2^-12 over many elements with one.
TABLES = [
    ((5.0, 0.0, 0.0), (5.0, 0.0, 0.0), (1.0, 0.0, 0.0)),            # X to 25
    ((1.0, 40.0, 0.0), (0.5, 0.0, 0.0)),                            # B to 40, X to 41
    ((2.0, 0.0, 100.0), (0.01, 0.0, 0.0)),                          # B to 100, X to 102
    ((1000.0, 0.0, 0.0), (1.0, 1e-6, 0.0), (0.001, 0.0, 0.0)),      # A to 10^6
    ((1e6, 0.0, 0.0), (1e-6, 0.0, 0.0)),
    ((0.5, 0.0, 0.0),) * 3,                                         # nothing grows
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 50), (70, 200), (200, 70), (130, 1000)])
@pytest.mark.parametrize("table", TABLES)
def test_growth(ta, table, shape, dtype):
    for x in (rank_one(*shape, dtype, 180), gradient(*shape, dtype, 181)):
        want = reference(x, table)
        got = ta.orthogonalize(x.cuda(), steps=len(table), coefficients=table)
        check(got, want, bound(dtype, dtype == torch.float32 or min(shape) < 64))


@pytest.mark.parametrize("table", TABLES)
def test_growth_of_a_step(ta, table):
    w, g = torch.randn(80, 120, generator=torch.Generator().manual_seed(182)), rank_one(80, 120, torch.float32, 183)
    gw, m = w.cuda(), torch.zeros(80, 120, device="cuda")
    ta.muon_([gw], [g.cuda()], [m], lr=0.1, momentum=0.0, steps=len(table), coefficients=table)
    want = 0.1 * reference(g, table)
    off = (gw.cpu().double() - (w.double() - want)).norm().item()
    assert off <= 1.2e-5 * want.norm().item() + w.double().norm().item() * 2.0 ** -22


def test_small_gradients_that_grow(ta):
    """A norm under eps, which divides it: X starts small."""
    x = rank_one(70, 90, torch.float32, 184)
    small = x * (1e-10 / x.norm())
    for table in TABLES[:1] + TABLES[-2:]:
        check(ta.orthogonalize(small.cuda(), steps=len(table), coefficients=table), reference(small, table), bound(torch.float32, True))


def test_coefficients_without_a_result(ta):
    """Not finite, or growing past every number: not finite, and no error."""
    x = rank_one(70, 90, torch.float32, 185)
    for table in (((float("nan"), 0.0, 0.0),) * 2, ((float("inf"), 1.0, 1.0),) * 2, ((1e30, 0.0, 1e30),) * 4):
        assert not torch.isfinite(ta.orthogonalize(x.cuda(), steps=len(table), coefficients=table)).all()
