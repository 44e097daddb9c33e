"""Calls of the row operators while a trace is taken are refused: it would have the results' allocation and not the kernels.

The refusal comes before any look at the tensors, so that it shows without a GPU.
"""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import torchft_amd as t

f = torch.zeros
ORDER = t.ExpertOrder(*(f(n, dtype=torch.int32) for n in (8, (4, 2), 4)))
CALLS = {
    "norm": lambda x: t.rms_norm(x),
    "norm in 8 bits": lambda x: t.rms_norm_fp8(x).codes,
    "values": lambda x: t.FP8Rows(x, x).dequantize(),
    "dropout": lambda x: t.dropout(x, 0.5, 1),
    "embedding": lambda x: t.embedding(f(3).long(), x),
    "sort": lambda x: t.sort_by_expert(x, 4).order,
    "dispatch": lambda x: t.dispatch(x, ORDER),
    "combine": lambda x: t.combine(x, ORDER),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("before", [False, True])
def test_fx(name, before):
    with pytest.raises(AssertionError, match="trace of the call"):
        make_fx(CALLS[name], pre_dispatch=before)(f(4, 3))


@pytest.mark.parametrize("name", CALLS)
def test_jit(name):
    with pytest.raises(AssertionError, match="trace of the call"):
        torch.jit.trace(CALLS[name], (f(4, 3),), check_trace=False)


@pytest.mark.parametrize("name", CALLS)
def test_export(name):
    class Module(torch.nn.Module):
        def forward(self, x):
            return CALLS[name](x)
    with pytest.raises(Exception, match="trace of the call"):
        torch.export.export(Module(), (f(4, 3),), strict=False)


@pytest.mark.parametrize("name", CALLS)
def test_fake_mode_around_real_tensors(name):
    from torch._subclasses.fake_tensor import FakeTensorMode
    x = f(4, 3)
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(AssertionError, match="trace of the call"):
        CALLS[name](x)


def test_modes_that_look_on():
    """A mode that counts what is done is no trace: the call gets as far as its tensors."""
    from torch.utils.flop_counter import FlopCounterMode
    with FlopCounterMode(display=False), pytest.raises(AssertionError, match="A GPU tensor is required"):
        t.rms_norm(f(2, 3))
