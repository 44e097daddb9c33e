"""Forward-mode differentiation of layers on 4-bit matrices is refused, not left out; without a GPU."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from torchft_amd import MXFP4Tensor, _lib, linear_mxfp4


def kept(rows, cols):
    return MXFP4Tensor(torch.zeros(_lib.load().tftq_mx_bytes(rows, cols), dtype=torch.uint8), (rows, cols), torch.float32)


@pytest.mark.parametrize("shape", [(3, 64), (2, 3, 64), (64,), (0, 64)])
def test_a_kept_weight(shape):
    w = kept(5, 64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones(shape), torch.ones(shape))
        for enabled in (True, False):  # forward mode does not ask for grad mode
            with torch.set_grad_enabled(enabled), pytest.raises(AssertionError, match="no gradient product"):
                linear_mxfp4(dual, w)


def test_a_weight_that_is_a_tensor():
    with forward_ad.dual_level():
        x, w = torch.ones(3, 64), torch.ones(5, 64)
        for args in ((forward_ad.make_dual(x, x), w), (x, forward_ad.make_dual(w, w))):
            for enabled in (True, False):
                with torch.set_grad_enabled(enabled), pytest.raises((NotImplementedError, AssertionError)):
                    linear_mxfp4(*args)
