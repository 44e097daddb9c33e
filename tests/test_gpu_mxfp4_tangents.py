"""Forward-mode differentiation of layers on 4-bit matrices is refused, not left out."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from test_gpu_mxfp4 import values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 70])
def test_tangents(rows):
    import torchft_amd as mx
    x, w = values(rows, 300, torch.bfloat16, 110).cuda(), values(40, 300, torch.bfloat16, 111).cuda()
    kept = mx.quantize_mxfp4(w)
    want = mx.linear_mxfp4(x, kept)  # from here on whole calls go through the native helper
    with forward_ad.dual_level():
        dual, dual_w = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, torch.ones_like(w))
        for enabled in (True, False):
            with torch.set_grad_enabled(enabled):
                with pytest.raises(AssertionError, match="no gradient product"):
                    mx.linear_mxfp4(dual, kept)
                for args in ((dual, w), (x, dual_w)):
                    with pytest.raises(NotImplementedError):
                        mx.linear_mxfp4(*args)
        assert torch.equal(mx.linear_mxfp4(x, kept), want)
        assert torch.equal(mx.linear_mxfp4(forward_ad.unpack_dual(dual).primal, kept), want)
    assert torch.equal(mx.linear_mxfp4(x, kept), want)
