"""A feed-forward block that replicas train and one of them serves, on this package alone.

    python examples/feed_forward.py [--replicas 2] [--steps 40] [--width 2048] [--hidden 5632] [--tokens 2048]

Every replica computes its own gradients with :func:`linear_mxfp4` (three 4-bit products to a layer), averages
them in 8 bits with :func:`allreduce_quantized` and takes the same step of :class:`Muon`; then the weights are
kept in 4 bits and one token goes through them.  The replicas are threads on one GPU (``sim_pg``); ``train``
takes any process group, one GPU to a rank over RCCL in earnest.
"""

from __future__ import annotations

import argparse
import os
import sys
import threading

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402
from torch.distributed import ReduceOp  # noqa: E402

import sim_pg  # noqa: E402
from torchft_amd import Muon, allreduce_quantized, linear_mxfp4, quantize_mxfp4  # noqa: E402


def block(x, up, down):
    """``down silu(up x)``; the weights are tensors, or 4-bit matrices."""
    return linear_mxfp4(torch.nn.functional.silu(linear_mxfp4(x, up)), down)


def weights(width: int, hidden: int, seed: int, device) -> list:
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * s[1] ** -0.5).to(device) for s in ((hidden, width), (width, hidden))]


def train(group, steps: int, width: int, hidden: int, tokens: int, lr: float = 0.02):
    """The weights and the losses of one replica, which learns what another block computes."""
    device = torch.device("cuda", torch.cuda.current_device())
    params = [torch.nn.Parameter(w) for w in weights(width, hidden, 1, device)]  # the same on every replica
    up, down = weights(width, hidden, 2, device)
    optimizer = Muon(params, lr=lr)
    g = torch.Generator(device).manual_seed(100 + group.rank())
    losses = []
    for _ in range(steps):
        x = torch.randn(tokens, width, generator=g, device=device).to(torch.bfloat16)
        with torch.no_grad():
            want = torch.nn.functional.silu(x.float() @ up.t()) @ down.t()
        loss = (block(x, *params).float() - want).square().mean() / want.square().mean()
        loss.backward()
        allreduce_quantized([p.grad for p in params], ReduceOp.AVG, group, torch.cuda.current_stream()).wait()
        optimizer.step()
        optimizer.zero_grad(set_to_none=True)
        losses.append(loss.detach())
    return [p.detach() for p in params], torch.stack(losses).tolist()


def serve(params: list, token: torch.Tensor) -> torch.Tensor:
    """One token through weights that are kept in 4 bits."""
    return block(token, *(quantize_mxfp4(p) for p in params))


def run(replicas: int, **sizes) -> list:
    """``train`` on every replica, a thread each."""
    group, results = sim_pg.SimGroup(replicas), [None] * replicas

    def body(rank):
        try:
            torch.cuda.set_device(0)
            with torch.cuda.stream(torch.cuda.Stream()):
                results[rank] = train(group.rank(rank), **sizes)
            torch.cuda.synchronize()
        except BaseException as error:  # noqa: BLE001
            results[rank] = error
            group.barrier.abort()  # the others fail too instead of waiting
    threads = [threading.Thread(target=body, args=(rank,)) for rank in range(replicas)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    errors = [r for r in results if isinstance(r, BaseException)]
    if errors:
        raise next((e for e in errors if not isinstance(e, threading.BrokenBarrierError)), errors[0])
    return results


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("replicas", 2), ("steps", 40), ("width", 2048), ("hidden", 5632), ("tokens", 2048)):
        parser.add_argument("--" + name, type=int, default=default)
    args = parser.parse_args()
    results = run(**vars(args))
    for rank, (_, losses) in enumerate(results):
        print(f"replica {rank}: loss " + " ".join(f"{v:.3f}" for v in losses[:: max(1, args.steps // 8)]) + f" ... {losses[-1]:.3f}")
    params = results[0][0]
    same = all(torch.equal(a, b) for other, _ in results[1:] for a, b in zip(params, other))
    print("the replicas' weights are", "the same" if same else "DIFFERENT")
    token = torch.randn(1, args.width, device="cuda").to(torch.bfloat16)
    print("a token through 4-bit weights:", serve(params, token)[0, :4].tolist())


if __name__ == "__main__":
    main()
