"""A small language model of experts that replicas train and one of them serves, on this package alone.

    python examples/experts.py [--replicas 2] [--steps 20] [--width 512] [--hidden 1024] [--tokens 1024] [--vocab 4096]
                               [--layers 2] [--experts 8] [--choices 2] [--dropout 0.1]

Between its 4-bit linear layers (:func:`linear_mxfp4`) run the row operators: token numbers become rows (:func:`embedding`),
every layer norms the residual (:func:`rms_norm`), sorts its tokens by expert and takes their rows there and back
(:func:`sort_by_expert`, :func:`dispatch`, :func:`combine`), and adds what comes back to the residual behind
:func:`dropout`.  Gradients are averaged in 8 bits (:func:`allreduce_quantized`); matrices take a step of :class:`Muon`,
vectors and tables one of Adam.  The replicas are threads on one GPU (``sim_pg``).
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
from torchft_amd import (  # noqa: E402
    Muon, allreduce_quantized, combine, dispatch, dropout, embedding, linear_mxfp4, quantize_mxfp4, rms_norm, rms_norm_fp8,
    sort_by_expert,
)


def parameters(width: int, hidden: int, vocab: int, layers: int, experts: int, seed: int, device, dtype=torch.float32) -> dict:
    g = torch.Generator().manual_seed(seed)

    def matrix(rows, cols):
        return (torch.randn(rows, cols, generator=g) * cols ** -0.5).to(device, dtype)

    p = {"table": torch.randn(vocab, width, generator=g).mul(width ** -0.5).to(device, dtype), "head": matrix(vocab, width),
         "norm": torch.ones(width, device=device)}
    for i in range(layers):
        p[f"{i}.norm"] = torch.ones(width, device=device)
        p[f"{i}.router"] = matrix(experts, width)
        for e in range(experts):
            p[f"{i}.{e}.up"], p[f"{i}.{e}.down"] = matrix(hidden, width), matrix(width, hidden)
    return p


def route(y: torch.Tensor, router: torch.Tensor, choices: int):
    """The experts of every token and their weights."""
    best = (y.float() @ router.float().t()).topk(choices, dim=1)
    return best.indices, best.values.softmax(1)


def visit(rows: torch.Tensor, offsets: list, p: dict, layer: int, linear) -> torch.Tensor:
    """Every expert on its rows."""
    out = [linear(torch.nn.functional.silu(linear(rows[a:b], p[f"{layer}.{e}.up"])), p[f"{layer}.{e}.down"])
           for e, (a, b) in enumerate(zip(offsets, offsets[1:])) if a < b]
    return torch.cat(out)


def forward(p: dict, ids: torch.Tensor, layers: int, experts: int, choices: int, rate: float = 0.0, seed=0, linear=linear_mxfp4,
            dtype=torch.bfloat16) -> torch.Tensor:
    """The logits of every token."""
    h = embedding(ids, p["table"].to(dtype), scale=p["table"].shape[1] ** 0.5)
    for i in range(layers):
        y = rms_norm(h, p[f"{i}.norm"])
        chosen, weights = route(y, p[f"{i}.router"], choices)
        order = sort_by_expert(chosen, experts)
        answers = visit(dispatch(y, order), order.offsets.tolist(), p, i, linear)
        h = dropout(combine(answers, order, weights), rate, seed, offset=i, residual=h)
    return linear(rms_norm(h, p["norm"]), p["head"])


def serve(p: dict, ids: torch.Tensor, layers: int, experts: int, choices: int) -> torch.Tensor:
    """The same without gradients: weights kept in 4 bits, rows sent to the experts in 8."""
    kept = {name: quantize_mxfp4(w) if name.endswith(("up", "down", "head")) else w for name, w in p.items()}
    h, answer = embedding(ids, p["table"].to(torch.bfloat16), scale=p["table"].shape[1] ** 0.5), None
    for i in range(layers):
        if answer is not None:
            rows, h = rms_norm_fp8(answer, p[f"{i}.norm"], h)
        else:
            rows = rms_norm_fp8(h, p[f"{i}.norm"])
        chosen, weights = route(rows.dequantize(), p[f"{i}.router"], choices)
        order = sort_by_expert(chosen, experts)
        sent = dispatch(rows, order)
        answer = combine(visit(sent.dequantize(), order.offsets.tolist(), kept, i, linear_mxfp4), order, weights)
    return linear_mxfp4(rms_norm(answer, p["norm"], h)[0], kept["head"])


def train(group, steps: int, tokens: int, choices: int, rate: float, lr: float = 0.02, **sizes):
    """The parameters and the losses of one replica, which learns to continue an arithmetic text."""
    device = torch.device("cuda", torch.cuda.current_device())
    layers, experts, vocab = sizes["layers"], sizes["experts"], sizes["vocab"]
    p = {name: torch.nn.Parameter(w) for name, w in parameters(seed=1, device=device, **sizes).items()}  # the same on every replica
    matrices = [w for name, w in p.items() if name.endswith(("up", "down"))]
    others = [w for name, w in p.items() if not name.endswith(("up", "down"))]
    optimizers = [Muon(matrices, lr=lr), torch.optim.Adam(others, lr=1e-3)]
    g = torch.Generator(device).manual_seed(100 + group.rank())
    losses = []
    for step in range(steps):
        ids = torch.randint(0, vocab, (tokens,), generator=g, device=device)
        logits = forward(p, ids, layers, experts, choices, rate, seed=1000 * step + group.rank())
        loss = torch.nn.functional.cross_entropy(logits.float(), (3 * ids + 1) % vocab)
        loss.backward()
        for w in p.values():  # an expert that no token chose has no gradient yet
            if w.grad is None:
                w.grad = torch.zeros_like(w)
        allreduce_quantized([w.grad for w in p.values()], ReduceOp.AVG, group, torch.cuda.current_stream()).wait()
        for optimizer in optimizers:
            optimizer.step()
            optimizer.zero_grad(set_to_none=True)
        losses.append(loss.detach())
    return {name: w.detach() for name, w in p.items()}, torch.stack(losses).tolist()


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
    for name, default in (("replicas", 2), ("steps", 20), ("width", 512), ("hidden", 1024), ("tokens", 1024), ("vocab", 4096), ("layers", 2),
                          ("experts", 8), ("choices", 2)):
        parser.add_argument("--" + name, type=int, default=default)
    parser.add_argument("--dropout", dest="rate", type=float, default=0.1)
    args = parser.parse_args()
    results = run(**vars(args))
    for rank, (_, losses) in enumerate(results):
        print(f"replica {rank}: loss " + " ".join(f"{v:.3f}" for v in losses[:: max(1, args.steps // 8)]) + f" ... {losses[-1]:.3f}")
    p = results[0][0]
    same = all(torch.equal(a, b) for other, _ in results[1:] for a, b in zip(p.values(), other.values()))
    print("the replicas' weights are", "the same" if same else "DIFFERENT")
    logits = serve(p, torch.arange(3, device="cuda"), args.layers, args.experts, args.choices)
    print("three tokens, served:", logits.argmax(1).tolist())


if __name__ == "__main__":
    main()
