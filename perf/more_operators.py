"""The row operators of a training step around its linear layers, as measurable cases.

``op`` is the operator, ``train`` whether the pass takes the gradients too:

    norm       root-mean-square norm of rows behind the residual's addition, with the new residual
    norm8      the same with an output in 8 bits (e4m3, one scale a row), and the values that it stands for
    dropout    dropout from a counter-based generator, added to the residual where there is one
    embedding  rows of a table, scaled; their gradient is a whole table
    experts    tokens sorted by expert, their rows there, and the experts' rows back with weights

Other keys of a case: ``dtype`` of the rows (norm weights have it too, the experts' weights are float32);
``rows`` and ``cols``, with ``residual``; ``p`` of ``dropout``; ``vocab`` of ``embedding`` (whose rows are
tokens); ``experts``, ``k`` of them to a token, and ``dropped``, the share of choices that name no expert.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_EPS = 1e-6
_MOST = 8192 * 4096        # elements of a drawn case
_MOST_TABLE = 128256 * 4096


def _case(name, op, dtype, rows, cols, train=True, residual=False, p=0.0, vocab=0, experts=0, k=0, dropped=0.0):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "cols": cols, "train": train, "residual": residual,
            "p": p, "vocab": vocab, "experts": experts, "k": k, "dropped": dropped}


def listed():
    return [
        # A decoding step of an 8B model: the smallest call, all of it latency.
        _case("one token, norm in 8 bits", "norm8", "bfloat16", 1, 4096, train=False, residual=True),
        # A prompt of 8192 tokens whose normed rows go to other GPUs in 8 bits.
        _case("prompt, norm in 8 bits", "norm8", "bfloat16", 8192, 4096, train=False, residual=True),
        # A layer's norm in a replica's training step (configuration 3's width).
        _case("layer, norm", "norm", "bfloat16", 8192, 4096, residual=True),
        # Queries and keys of 40 heads, normed head by head: very short rows, many of them.
        _case("heads, norm", "norm", "float16", 163840, 128),
        # A small head of odd sizes in single precision.
        _case("odd rows, dropout", "dropout", "float32", 33, 1001, p=0.5),
        # Dropout behind a layer's output projection, added to the residual.
        _case("layer, dropout", "dropout", "bfloat16", 8192, 4096, residual=True, p=0.1),
        # A decoding step of the 1.1B model (configuration 4's table).
        _case("one token, embedding", "embedding", "float32", 1, 2048, train=False, vocab=32000),
        # A replica's batch of the 1.1B model.
        _case("1.1B model, embedding", "embedding", "bfloat16", 4096, 2048, vocab=32000),
        # A large vocabulary: the gradient's empty rows are most of the work.
        _case("large vocabulary, embedding", "embedding", "bfloat16", 8192, 4096, vocab=128256),
        # A decoding step through two of eight experts.
        _case("one token, experts", "experts", "bfloat16", 1, 4096, train=False, experts=8, k=2),
        # A replica's batch through two of eight experts.
        _case("layer, experts", "experts", "bfloat16", 8192, 4096, experts=8, k=2),
        # Many small experts, odd sizes, with padding tokens that go to none.
        _case("many experts, odd rows", "experts", "float32", 4099, 777, experts=61, k=6, dropped=0.05),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm8", "dropout", "embedding", "embedding", "experts", "experts"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32", "float16"])
    cols = _spread(rng, 16, 16384)
    if rng.random() < 0.6:  # a model's own sizes
        cols = -(-cols // 64) * 64
    case = _case("", op, dtype, 1, cols, train=op != "norm8" and rng.random() < 0.75, residual=op in ("norm", "norm8", "dropout") and rng.random() < 0.6)
    del case["name"]
    most = _MOST // cols // (2 if dtype == "float32" else 1)
    if op == "dropout":
        case["p"] = rng.choice([0.05, 0.1, 0.2, 0.3, 0.5])
    if op == "embedding":
        case["vocab"] = _spread(rng, 100, max(100, min(131072, _MOST_TABLE // cols // (2 if dtype == "float32" else 1))))
    if op == "experts":
        case["experts"] = _spread(rng, 2, 256)
        case["k"] = rng.randint(1, min(8, case["experts"]))
        case["dropped"] = rng.choice([0.0, 0.0, 0.1])
        most = 2 * most // case["k"]
    case["rows"] = _spread(rng, 1, max(1, min(65536, most)))
    return case


# ---- inputs ------------------------------------------------------------------------------------


def _activations(rows, cols, dtype, generator):
    """Normal, with channels of up to 30 times the usual size and rows of differing size."""
    x = torch.randn(rows, cols, device="cuda", generator=generator)
    x *= torch.where(torch.rand(cols, device="cuda", generator=generator) < 0.01, 30.0, 1.0)
    x *= 10.0 ** (torch.rand(rows, 1, device="cuda", generator=generator) - 0.5)
    return x.to(dtype)


def _gradient(rows, cols, dtype, generator):
    return (torch.randn(rows, cols, device="cuda", generator=generator) * 1e-2).to(dtype)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    op, dtype, rows, cols, train = case["op"], _DTYPES[case["dtype"]], case["rows"], case["cols"], case["train"]
    state = {"op": op, "dtype": dtype, "train": train, "residual": None}
    if op in ("norm", "norm8"):
        state["x"] = _activations(rows, cols, dtype, g).requires_grad_(train)
        state["weight"] = (1 + 0.2 * torch.randn(cols, device="cuda", generator=g)).to(dtype).requires_grad_(train)
    elif op == "dropout":
        state["x"] = _activations(rows, cols, dtype, g).requires_grad_(train)
        state["p"] = case["p"]
        state["seed"], state["offset"] = seed * 0x9E3779B97F4A7C15 % 2**62, seed % 1000
    elif op == "embedding":
        # the frequent tokens of a text have the small numbers, and come about as often as 1 / number
        u = torch.rand(rows, device="cuda", generator=g, dtype=torch.float64)
        state["ids"] = (case["vocab"] ** u - 1).long().clamp(0, case["vocab"] - 1)
        state["table"] = (torch.randn(case["vocab"], cols, device="cuda", generator=g) * 0.02).to(dtype).requires_grad_(train)
        state["scale"] = math.sqrt(cols)
    else:
        experts, k = case["experts"], case["k"]
        logits = torch.randn(rows, experts, device="cuda", generator=g) + torch.randn(experts, device="cuda", generator=g)
        best = logits.topk(k, dim=1)
        none = torch.rand(rows, k, device="cuda", generator=g) < case["dropped"]
        state["chosen"] = torch.where(none, -1, best.indices)
        state["weights"] = best.values.softmax(1).requires_grad_(train)
        state["experts"] = experts
        state["x"] = _activations(rows, cols, dtype, g).requires_grad_(train)
        state["answers"] = _activations(rows * k, cols, dtype, g).requires_grad_(train)
    if case["residual"]:
        state["residual"] = _activations(rows, cols, dtype, g).requires_grad_(train)
    if train:
        state["dy"] = _gradient(rows, cols, dtype, g)
        if op == "norm" and case["residual"]:
            state["dresidual"] = _gradient(rows, cols, dtype, g)
        if op == "experts":
            state["dsorted"] = _gradient(rows * case["k"], cols, dtype, g)
    return state


# ---- the plain form ----------------------------------------------------------------------------


def _random16(seed, offset, count, device):
    """``count`` whole numbers of 16 bits: the ten rounds of the Philox generator of four 32-bit words, a word two numbers."""
    low = 0xFFFFFFFF
    block = torch.arange(-(-count // 8), device=device)
    c0, c1 = block & low, block >> 32
    c2, c3 = torch.full_like(block, offset & low), torch.full_like(block, offset >> 32 & low)
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the sign bit is the product's highest
        c0, c1, c2, c3 = (p1 >> 32 & low) ^ c1 ^ k0, p1 & low, (p0 >> 32 & low) ^ c3 ^ k1, p0 & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    words = torch.stack([c0, c1, c2, c3], 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).flatten()[:count]


def _plain_norm(state):
    x, weight, dtype = state["x"].detach(), state["weight"].detach().float(), state["dtype"]
    h = x if state["residual"] is None else (x.float() + state["residual"].detach().float()).to(dtype)
    f = h.float()
    r = (f.square().mean(1, keepdim=True) + _EPS).rsqrt()
    y = f * r * weight
    if state["op"] == "norm8":
        amax = y.abs().amax(1, keepdim=True)
        scales = torch.where(amax > 0, amax / 448, 1.0)
        out = {"values": ((y / scales).to(torch.float8_e4m3fn).float() * scales).to(dtype), "scales": scales}
    else:
        out = {"y": y.to(dtype)}
    if state["residual"] is not None:
        out["residual"] = h
    if state["train"]:
        dy = state["dy"].float()
        g = dy * weight
        dx = r * (g - f * (r * r * (g * f).mean(1, keepdim=True)))
        if state["residual"] is not None:
            dx = dx + state["dresidual"].float()
        out |= {"dx": dx.to(dtype), "dweight": (dy * f * r).sum(0).to(dtype)}
    return out


def _plain_dropout(state):
    x, dtype = state["x"].detach(), state["dtype"]
    threshold = round(state["p"] * 65536)
    keep = _random16(state["seed"], state["offset"], x.numel(), x.device).view(x.shape) >= threshold
    factor = 65536 / (65536 - threshold)
    y = torch.where(keep, x.float() * factor, 0.0)
    if state["residual"] is not None:
        y = y + state["residual"].detach().float()
    out = {"y": y.to(dtype)}
    if state["train"]:
        out["dx"] = torch.where(keep, state["dy"].float() * factor, 0.0).to(dtype)
    return out


def _plain_embedding(state):
    ids, table, scale, dtype = state["ids"], state["table"].detach(), state["scale"], state["dtype"]
    out = {"y": (table[ids].float() * scale).to(dtype)}
    if state["train"]:
        out["dtable"] = torch.zeros(table.shape, device=table.device).index_add_(0, ids, state["dy"].float() * scale).to(dtype)
    return out


def _plain_experts(state):
    chosen, dtype, k = state["chosen"], state["dtype"], state["chosen"].shape[1]
    x, answers, weights = state["x"].detach(), state["answers"].detach(), state["weights"].detach()
    flat = chosen.flatten()
    key = torch.where((flat >= 0) & (flat < state["experts"]), flat, state["experts"])
    order = key.argsort(stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=order.device)
    offsets = (key[order][None] < torch.arange(state["experts"] + 1, device=key.device)[:, None]).sum(1)
    live = (torch.arange(order.numel(), device=order.device) < offsets[-1])[:, None]
    slot = order.argsort()  # of every choice, its place
    taken = (key < state["experts"]).view(-1, k, 1)
    out = {"position": position.view_as(chosen).int(), "offsets": offsets.int(), "sorted": torch.where(live, x[order // k], 0)}
    rows = torch.where(taken, answers[slot].view(-1, k, x.shape[1]).float(), 0.0)
    out["y"] = (rows * weights[:, :, None]).sum(1).to(dtype)
    if state["train"]:
        dy = state["dy"].float()
        out["dx"] = torch.where(taken, state["dsorted"][slot].view(-1, k, x.shape[1]).float(), 0.0).sum(1).to(dtype)
        each = (dy[:, None, :] * weights[:, :, None]).flatten(0, 1)[order]
        out["danswers"] = torch.where(live, each, 0.0).to(dtype)
        out["dweights"] = (rows * dy[:, None, :]).sum(2)
    return out


# ---- the framework's operators -----------------------------------------------------------------


def _own_norm(state, lib):
    x, weight, residual = state["x"], state["weight"], state["residual"]
    if state["op"] == "norm8":
        got = lib.rms_norm_fp8(x, weight, residual, eps=_EPS)
        rows, h = (got, None) if residual is None else got
        out = {"values": rows.dequantize(), "scales": rows.scales}
    else:
        got = lib.rms_norm(x, weight, residual, eps=_EPS)
        y, h = (got, None) if residual is None else got
        out = {"y": y.detach()}
    if h is not None:
        out["residual"] = h.detach()
    if state["train"]:
        if h is None:
            grads = torch.autograd.grad(y, (x, weight), state["dy"])
        else:
            grads = torch.autograd.grad((y, h), (x, weight, residual), (state["dy"], state["dresidual"]))
        out |= {"dx": grads[0], "dweight": grads[1]}
    return out


def run(state):
    op = state["op"]
    if not own:
        return {"norm": _plain_norm, "norm8": _plain_norm, "dropout": _plain_dropout, "embedding": _plain_embedding,
                "experts": _plain_experts}[op](state)
    import torchft_amd

    if op in ("norm", "norm8"):
        return _own_norm(state, torchft_amd)
    train = state["train"]
    if op == "dropout":
        x, residual = state["x"], state["residual"]
        y = torchft_amd.dropout(x, state["p"], state["seed"], state["offset"], residual=residual)
        out = {"y": y.detach()}
        if train:
            out["dx"] = torch.autograd.grad(y, (x,) if residual is None else (x, residual), state["dy"])[0]
        return out
    if op == "embedding":
        y = torchft_amd.embedding(state["ids"], state["table"], scale=state["scale"])
        out = {"y": y.detach()}
        if train:
            out["dtable"], = torch.autograd.grad(y, state["table"], state["dy"])
        return out
    order = torchft_amd.sort_by_expert(state["chosen"], state["experts"])
    sorted_rows = torchft_amd.dispatch(state["x"], order)
    y = torchft_amd.combine(state["answers"], order, state["weights"])
    out = {"position": order.position, "offsets": order.offsets, "sorted": sorted_rows.detach(), "y": y.detach()}
    if train:
        out["dx"], = torch.autograd.grad(sorted_rows, state["x"], state["dsorted"])
        out["danswers"], out["dweights"] = torch.autograd.grad(y, (state["answers"], state["weights"]), state["dy"])
    return out


# ---- what a pass cannot do without -------------------------------------------------------------


def work(case):
    op, size, rows, cols, train = case["op"], _DTYPES[case["dtype"]].itemsize, case["rows"], case["cols"], case["train"]
    row = cols * size
    if op == "norm8":
        return {"bytes": rows * (2 * row + cols + 4) + row + (2 * rows * row if case["residual"] else 0), "flops": 6 * rows * cols}
    if op == "norm":
        passes = 2 + (2 if case["residual"] else 0) + (2 + (1 if case["residual"] else 0) if train else 0)
        return {"bytes": passes * rows * row + (2 if train else 1) * row, "flops": (16 if train else 5) * rows * cols}
    if op == "dropout":
        passes = 2 + (1 if case["residual"] else 0) + (2 if train else 0)
        return {"bytes": passes * rows * row, "flops": (4 if train else 2) * rows * cols}
    if op == "embedding":
        table = case["vocab"] * row + rows * row if train else 0  # the gradient, and the rows that it sums
        return {"bytes": 2 * rows * row + 8 * rows + table, "flops": (2 if train else 1) * rows * cols}
    k = case["k"]
    numbers = rows * k * 16 + 4 * case["experts"]
    forward = rows * row * (1 + k + k + 1)
    backward = rows * row * (k + 1 + 1 + k) + 4 * rows * k if train else 0
    return {"bytes": forward + backward + numbers, "flops": rows * k * cols * (6 if train else 2)}


# ---- in 64 bits --------------------------------------------------------------------------------


def _bits16(seed, offset, count, device):
    """The same numbers as ``_random16``, with products of 16-bit halves."""
    def product(a, m):
        m_low, m_high = m & 0xFFFF, m >> 16
        bottom = a * m_low                   # below 2^48
        top = a * m_high + (bottom >> 16)    # the product without its lowest 16 bits
        return top >> 16, (top & 0xFFFF) << 16 | bottom & 0xFFFF
    ctr = [torch.arange((count + 7) // 8, device=device) % 2**32, torch.arange((count + 7) // 8, device=device) // 2**32]
    ctr += [torch.zeros_like(ctr[0]) + offset % 2**32, torch.zeros_like(ctr[0]) + offset // 2**32]
    key = [seed % 2**32, seed // 2**32]
    for _ in range(10):
        (h0, l0), (h1, l1) = product(ctr[0], 0xD2511F53), product(ctr[2], 0xCD9E8D57)
        ctr = [h1 ^ ctr[1] ^ key[0], l1, h0 ^ ctr[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
    return torch.stack([half for word in ctr for half in (word % 65536, word // 65536)], 1).reshape(-1)[:count]


def _e4m3(v):
    """The nearest number of four significant bits, steps of 2^-9 at least, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0**-6))) - 3)
    return torch.round(v / step) * step


def _rows64(rows, cols, numbers):
    """``numbers[..., None]`` times one, as a matrix."""
    return numbers.reshape(rows, 1).expand(rows, cols)


def exact(case, seed):
    state = prepare(case, seed)
    op, dtype, train = case["op"], state["dtype"], case["train"]
    wide = {name: t.detach().double() for name, t in state.items() if isinstance(t, torch.Tensor) and t.is_floating_point()}
    dy = wide.get("dy")
    if op in ("norm", "norm8"):
        x, w, n = wide["x"], wide["weight"], case["cols"]
        total = x + wide["residual"] if case["residual"] else x
        h = total.to(dtype).double()  # the norm is that of the residual as it is kept
        root = torch.sqrt((h * h).sum(1) / n + _EPS)
        unit = h / _rows64(case["rows"], n, root)
        y = unit * w
        out = {"y": y}
        if op == "norm8":
            scales = y.abs().max(1).values / 448
            scales = torch.where(scales == 0, torch.ones_like(scales), scales)[:, None]
            out = {"values": _e4m3(y / scales) * scales, "scales": scales}
        if case["residual"]:
            out["residual"] = total
        if train:
            out["dweight"] = torch.einsum("rc,rc->c", dy, unit)
            along = ((dy * w) * unit).sum(1) / n
            out["dx"] = (dy * w - unit * _rows64(case["rows"], n, along)) / _rows64(case["rows"], n, root)
            if case["residual"]:
                out["dx"] = out["dx"] + wide["dresidual"]
        return out
    if op == "dropout":
        border = round(case["p"] * 65536)
        lost = (_bits16(state["seed"], state["offset"], case["rows"] * case["cols"], "cuda") < border).reshape(case["rows"], -1)
        scale = 1 / (1 - border / 65536)
        y = (wide["x"] * scale).masked_fill(lost, 0)
        out = {"y": y + wide["residual"] if case["residual"] else y}
        if train:
            out["dx"] = (dy * scale).masked_fill(lost, 0)
        return out
    if op == "embedding":
        ids = state["ids"]
        out = {"y": wide["table"].index_select(0, ids) * state["scale"]}
        if train:
            names, where = ids.unique(return_inverse=True)
            sums = torch.zeros(names.numel(), case["cols"], dtype=torch.float64, device="cuda").index_add_(0, where, dy)
            out["dtable"] = torch.zeros_like(wide["table"]).index_copy_(0, names, sums * state["scale"])
        return out
    k, cols, chosen = case["k"], case["cols"], state["chosen"].cpu()
    lists = [[] for _ in range(case["experts"] + 1)]
    for choice, expert in enumerate(chosen.flatten().tolist()):
        lists[expert if 0 <= expert < case["experts"] else -1].append(choice)
    by_expert = torch.tensor([c for one in lists for c in one])
    starts = [0]
    for one in lists[:-1]:
        starts.append(starts[-1] + len(one))
    place = torch.zeros_like(by_expert).scatter_(0, by_expert, torch.arange(by_expert.numel())).cuda()
    by_expert, used = by_expert.cuda()[: starts[-1]], starts[-1]
    token = by_expert // k
    weight = wide["weights"].flatten()[by_expert][:, None]
    zeros = torch.zeros(case["rows"], cols, dtype=torch.float64, device="cuda")
    rest = torch.zeros(case["rows"] * k - used, cols, dtype=torch.float64, device="cuda")
    out = {"position": place.reshape(case["rows"], k).int(), "offsets": torch.tensor(starts, dtype=torch.int32, device="cuda"),
           "sorted": torch.cat([wide["x"][token], rest]), "y": zeros.index_add(0, token, wide["answers"][:used] * weight)}
    if train:
        out["dx"] = zeros.index_add(0, token, wide["dsorted"][:used])
        out["danswers"] = torch.cat([dy[token] * weight, rest])
        dots = torch.zeros(case["rows"] * k, dtype=torch.float64, device="cuda")
        dots[by_expert] = (dy[token] * wide["answers"][:used]).sum(1)
        out["dweights"] = dots.reshape(case["rows"], k)
    return out
