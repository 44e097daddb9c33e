"""An optimiser that is stopped, saved and resumed takes the steps of one that was not."""

import io

import pytest
import torch

from test_gpu_orthogonal import DTYPES, gradient

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
def test_resumed(dtype):
    from torchft_amd import Muon
    shapes = [(96, 130), (130, 70)]
    g = torch.Generator().manual_seed(90)
    start = [(torch.randn(s, generator=g) * 0.02).to(dtype) for s in shapes]

    def fresh(weights):
        ps = [torch.nn.Parameter(w.detach().clone().cuda()) for w in weights]
        return ps, Muon(ps, lr=0.1, weight_decay=0.1)

    def steps(ps, opt, first, last):
        for i in range(first, last):
            for k, p in enumerate(ps):
                p.grad = gradient(*p.shape, dtype, 91 + 10 * i + k).cuda()
            opt.step()
    ps, opt = fresh(start)
    steps(ps, opt, 0, 2)
    saved = io.BytesIO()
    torch.save(opt.state_dict(), saved)
    saved.seek(0)
    qs, again = fresh([p.cpu() for p in ps])
    again.load_state_dict(torch.load(saved, weights_only=True, map_location="cpu"))  # as from a peer's host memory
    for p, q in zip(ps, qs):
        m = again.state[q]["momentum"]
        assert m.dtype == torch.float32 and m.device == q.device and torch.equal(m, opt.state[p]["momentum"])
    steps(ps, opt, 2, 4)
    steps(qs, again, 2, 4)
    for p, q in zip(ps, qs):
        assert torch.equal(p, q) and torch.equal(again.state[q]["momentum"], opt.state[p]["momentum"])
