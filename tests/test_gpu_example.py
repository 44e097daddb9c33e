"""The example that trains, averages, steps and serves on this package's operators."""

import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import feed_forward
    return feed_forward


def test_train_and_serve(example):
    results = example.run(replicas=2, steps=30, width=192, hidden=320, tokens=256)
    params = results[0][0]
    assert all(torch.equal(a, b) for a, b in zip(params, results[1][0]))  # every replica took the same steps
    for _, losses in results:
        assert sum(losses[-5:]) < 0.5 * sum(losses[:5])
    assert results[0][1] != results[1][1]  # on data of its own
    token = torch.randn(1, 192, generator=torch.Generator().manual_seed(3)).cuda().to(torch.bfloat16)
    with torch.no_grad():
        assert torch.equal(example.serve(params, token), example.block(token, *params))
