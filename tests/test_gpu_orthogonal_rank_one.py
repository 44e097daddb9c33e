"""Matrices of nearly rank one: one direction holds the norm, and the iteration multiplies what rounding leaves in all
the others by up to 480.  bf16 results stay within the bound of one product, the others within that of float32 products."""

import pytest
import torch

from test_gpu_orthogonal import bound, gradient, reference

pytestmark = pytest.mark.gpu


def nearly_rank_one(m, n, noise, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(m, 1, device="cuda", generator=g) @ torch.randn(1, n, device="cuda", generator=g)
    return x + noise * torch.randn(m, n, device="cuda", generator=g)


def error(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


SHAPES = [(64, 64), (64, 512), (80, 2560), (512, 96), (127, 127), (128, 300), (300, 128), (160, 321), (191, 1528), (192, 192), (234, 261), (600, 256)]


@pytest.mark.parametrize("noise", [0.0, 1e-4, 1e-3, 1e-2])
@pytest.mark.parametrize("shape", SHAPES)
def test_bf16(shape, noise):
    import torchft_amd as ta
    xs = [nearly_rank_one(*shape, noise, 210 + i) for i in range(6)]
    for x, y in zip(xs, ta.orthogonalize(xs, out_dtype=torch.bfloat16)):
        assert error(y, reference(x)) <= bound(torch.bfloat16, False)
    x = xs[0].to(torch.bfloat16)
    assert error(ta.orthogonalize(x), reference(x)) <= bound(torch.bfloat16, False)


def test_beside_matrices_of_one_product():
    """In a list with larger ones, which go on taking one."""
    import torchft_amd as ta
    xs = [nearly_rank_one(70, 90, 1e-4, 220), gradient(600, 700, torch.float32, 221, device="cuda"), nearly_rank_one(150, 100, 1e-4, 222)]
    for x, y in zip(xs, ta.orthogonalize(xs, out_dtype=torch.bfloat16)):
        assert error(y, reference(x)) <= bound(torch.bfloat16, False)


@pytest.mark.parametrize("shape", SHAPES)
def test_three_products(shape):
    """No further off than the iteration in float32 is, twice over."""
    import torchft_amd as ta
    for noise in (0.0, 1e-4, 1e-2):
        x = nearly_rank_one(*shape, noise, 230)
        want = reference(x)
        y = x if x.shape[0] <= x.shape[1] else x.t()
        y = y / y.norm()
        for _ in range(5):
            a = y @ y.t()
            y = 3.4445 * y + (-4.7750 * a + 2.0315 * (a @ a)) @ y
        plain = error(y if x.shape[0] <= x.shape[1] else y.t(), want)
        assert error(ta.orthogonalize(x), want) <= 2 * plain
