"""The operators of a low-precision data-parallel training step, as measurable cases.

``op`` is the operator:

    roundtrip    4-bit microscaled codes of a matrix along its rows and along its columns, and the values
                 that they stand for (what quantisation-aware training and a check of a checkpoint do)
    serve        ``x @ w.T`` with 4-bit microscaled weights that the program keeps; x is quantised in the call
    train        a linear layer's training step: ``y = x @ w.T`` and both gradients, every product of
                 4-bit microscaled matrices whose blocks lie along the contracted axis
    orthogonal   the Newton-Schulz orthogonalisation of one matrix
    muon         the Muon optimiser's step on a list of matrices: momentum, orthogonalisation, update

Other keys of a case: ``dtype``, the type of the matrices (``muon``: of weights and gradients; the momentum
is float32); ``rows`` and ``cols`` of the matrix (``serve`` and ``train``: of the weight, so ``cols`` is the
contracted size of the forward product) with ``tokens``; ``shapes`` for ``muon``, ``2*256x2048, 512x512``
for two matrices and a third.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_STEPS, _A, _B, _C, _EPS = 5, 3.4445, -4.7750, 2.0315, 1e-7
_LR, _DECAY, _MOMENTUM = 0.02, 0.1, 0.95
_MOST_FLOPS = 4 * 2 * 4096 * 4096 * 14336  # no drawn case has more


def _matrix(name, op, dtype, rows, cols, tokens=0):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "cols": cols, "tokens": tokens}


def _muon(name, dtype, shapes):
    return {"name": name, "op": "muon", "dtype": dtype, "shapes": shapes}


def listed():
    return [
        # A layer of a small model (benchmark configuration 1): the smallest call, all of it latency.
        _matrix("small layer, codes", "roundtrip", "float32", 256, 512),
        # The widest weight of an 8B model (configuration 3), both ways as a training step needs it.
        _matrix("wide weight, codes", "roundtrip", "bfloat16", 14336, 4096),
        # One token through that weight: a decoding step's largest product.
        _matrix("one token", "serve", "bfloat16", 14336, 4096, 1),
        # A few dozen requests decoded together, of a model whose sizes are no whole blocks.
        _matrix("odd batch", "serve", "float16", 5003, 1001, 33),
        # A prompt of 8192 tokens through the same weight.
        _matrix("prompt", "serve", "bfloat16", 14336, 4096, 8192),
        # A replica's batch through a layer of the 1.1B model (configuration 4).
        _matrix("training, 1.1B", "train", "bfloat16", 5632, 2048, 4096),
        # A replica's batch through the widest weight of the 8B model: the largest work.
        _matrix("training, 8B", "train", "bfloat16", 14336, 4096, 8192),
        # A head of odd sizes in single precision, on a ragged number of tokens.
        _matrix("odd training", "train", "float32", 333, 257, 1001),
        # The pseudo-gradient of a small layer before an outer step (configuration 1).
        _matrix("small layer, orthogonal", "orthogonal", "float32", 256, 512),
        # The averaged gradient of an 8B model's down projection.
        _matrix("wide weight, orthogonal", "orthogonal", "bfloat16", 4096, 14336),
        # One fragment of the 1.1B model, as one optimiser step takes it.
        _muon("1.1B fragment", "bfloat16", "2*2048x2048, 2*256x2048, 2*5632x2048, 2048x5632"),
        # Matrices of odd sizes, taller and wider, with a vector kept as a matrix, in single precision.
        _muon("odd matrices", "float32", "3*333x1001, 1001x130, 1x777, 2*517x517"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    op = rng.choice(["roundtrip", "serve", "serve", "train", "train", "orthogonal", "muon"])
    case = {"op": op, "dtype": rng.choice(["bfloat16", "bfloat16", "float32", "float16"])}
    if op == "muon":
        width, items, left = _spread(rng, 64, 2048), [], _MOST_FLOPS // 4
        for _ in range(rng.randint(1, 5)):
            count, other = rng.randint(1, 4), rng.choice([width, 2 * width + 1, max(1, width // 3), 4 * width, 1])
            shape = rng.choice([(width, other), (other, width)])
            cost = count * _newton_schulz_flops(*shape)
            if cost <= left:
                left -= cost
                items.append(f"{count}*{shape[0]}x{shape[1]}")
        case["shapes"] = ", ".join(items) or "64x64"
        return case
    if op == "orthogonal":
        while True:
            rows, cols = _spread(rng, 16, 8192), _spread(rng, 16, 16384)
            if _newton_schulz_flops(rows, cols) <= _MOST_FLOPS:
                break
    else:
        rows, cols = _spread(rng, 32, 16384), _spread(rng, 32, 16384)
    if rng.random() < 0.6:  # a model's own sizes: whole blocks
        rows, cols = -(-rows // 64) * 64, -(-cols // 64) * 64
    case |= {"rows": rows, "cols": cols, "tokens": 0}
    if op in ("serve", "train"):
        most = max(1, min(16384, _MOST_FLOPS // (6 * rows * cols)))
        case["tokens"] = _spread(rng, 1, most) if op == "serve" else _spread(rng, min(64, most), most)
    return case


def _shapes(case):
    out = []
    for item in case["shapes"].split(","):
        times, _, shape = item.strip().rpartition("*")
        out += [tuple(int(x) for x in shape.split("x"))] * int(times or 1)
    return out


# ---- inputs ------------------------------------------------------------------------------------


def _activations(rows, cols, dtype, generator):
    """Normal, with channels of up to 30 times the usual size and tokens of differing size."""
    x = torch.randn(rows, cols, device="cuda", generator=generator)
    channel = torch.rand(cols, device="cuda", generator=generator)
    x *= torch.where(channel < 0.01, 30.0, 1.0)
    x *= 10.0 ** (torch.rand(rows, 1, device="cuda", generator=generator) - 0.5)
    return x.to(dtype)


def _weight(rows, cols, dtype, generator):
    return (torch.randn(rows, cols, device="cuda", generator=generator) * 0.02).to(dtype)


def _gradient(rows, cols, dtype, generator):
    """A few strong directions over noise, as the gradient of a weight matrix has, at a gradient's size."""
    rank = max(1, min(rows, cols) // 8)
    g = torch.randn(rows, rank, device="cuda", generator=generator) @ torch.randn(rank, cols, device="cuda", generator=generator)
    g *= 1.0 / math.sqrt(rank)
    g += 0.3 * torch.randn(rows, cols, device="cuda", generator=generator)
    return (g * 1e-3).to(dtype)


def prepare(case, seed):
    generator = torch.Generator("cuda").manual_seed(seed)
    op, dtype = case["op"], _DTYPES[case["dtype"]]
    state = {"op": op, "dtype": dtype}
    if op == "muon":
        shapes = _shapes(case)
        state["weights"] = [_weight(*s, dtype, generator) for s in shapes]
        state["grads"] = [_gradient(*s, dtype, generator) for s in shapes]
        state["momenta"] = [_gradient(*s, torch.float32, generator) for s in shapes]
        return state
    rows, cols, tokens = case["rows"], case["cols"], case["tokens"]
    if op == "orthogonal":
        state["x"] = _gradient(rows, cols, dtype, generator)
    elif op == "roundtrip":
        state["x"] = _activations(rows, cols, dtype, generator)
    elif op == "serve":
        state["x"] = _activations(tokens, cols, dtype, generator)
        # what a checkpoint of 4-bit microscaled weights holds: two codes a byte, a scale for 32 elements
        state["codes"], state["scales"] = _encode(_weight(rows, cols, torch.float32, generator))
        state["cols"] = cols
        if own:
            import torchft_amd

            state["weight"] = torchft_amd.MXFP4Tensor.from_blocks(state["codes"], state["scales"], cols)
    else:
        state["x"] = _activations(tokens, cols, dtype, generator).requires_grad_()
        state["w"] = _weight(rows, cols, dtype, generator).requires_grad_()
        state["dy"] = _gradient(tokens, rows, dtype, generator)
    return state


# ---- the plain form ----------------------------------------------------------------------------


def _blocks(x):
    """x's rows in blocks of 32, filled up with zeros: [rows, blocks, 32] in float32."""
    x = x.float()
    return torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).unflatten(1, (-1, 32))


def _scale_exponent(blocks):
    """floor(log2 of the block's largest magnitude) - 2; that of an empty block is the smallest."""
    amax = blocks.abs().amax(-1, keepdim=True)
    exponent = torch.frexp(amax).exponent - 3
    return torch.where(amax == 0, -127, exponent).clamp(-127, 127)


def _to_e2m1(v):
    """The index of the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties to the even index."""
    a = v.abs()
    return ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))


def _encode(x):
    """(codes, scales) of x's rows: [rows, blocks, 16] and [rows, blocks] bytes."""
    blocks = _blocks(x)
    exponent = _scale_exponent(blocks)
    code = _to_e2m1(torch.ldexp(blocks, -exponent)) | ((blocks < 0).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4), (exponent[..., 0] + 127).to(torch.uint8)


def _values(device):
    half = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=device)
    return torch.cat([half, -half])


def _decode(codes, scales, cols):
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(2)
    v = torch.ldexp(_values(codes.device)[code.int()], scales.int().unsqueeze(-1) - 127)
    return v.flatten(1)[:, :cols]


def _quantized(x):
    """The values that the 4-bit form of x's rows stands for, and its scales."""
    codes, scales = _encode(x)
    return _decode(codes, scales, x.shape[1]), scales


def _newton_schulz(u):
    x = u.float()
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t()
    x = x / x.norm().clamp(min=_EPS)
    for _ in range(_STEPS):
        a = x @ x.t()
        x = _A * x + (_B * a + _C * (a @ a)) @ x
    return x.t() if tall else x


def _plain(state):
    op, dtype = state["op"], state["dtype"]
    if op == "roundtrip":
        x = state["x"]
        by_rows, row_scales = _quantized(x)
        by_cols, col_scales = _quantized(x.t())
        return {"rows": by_rows.to(dtype), "row_scales": row_scales, "columns": by_cols.to(dtype), "column_scales": col_scales}
    if op == "serve":
        weight = _decode(state["codes"], state["scales"], state["cols"])
        return (_quantized(state["x"])[0] @ weight.t()).to(dtype)
    if op == "train":
        x, w, dy = state["x"].detach(), state["w"].detach(), state["dy"]
        y = _quantized(x)[0] @ _quantized(w)[0].t()
        dx = _quantized(dy)[0] @ _quantized(w.t())[0].t()
        dw = _quantized(dy.t())[0] @ _quantized(x.t())[0].t()
        return {"y": y.to(dtype), "dx": dx.to(dtype), "dw": dw.to(dtype)}
    if op == "orthogonal":
        return _newton_schulz(state["x"]).to(dtype)
    for w, g, m in zip(state["weights"], state["grads"], state["momenta"]):
        g = g.float()
        m.mul_(_MOMENTUM).add_((1 - _MOMENTUM) * g)
        update = _newton_schulz(g + _MOMENTUM * (m - g))
        scale = math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
        w.copy_((1 - _LR * _DECAY) * w.float() - _LR * scale * update)
    return {"weights": state["weights"], "momenta": state["momenta"]}


# ---- the framework's operators -----------------------------------------------------------------


def run(state):
    if not own:
        return _plain(state)
    import torchft_amd

    op = state["op"]
    if op == "roundtrip":
        rows, cols = torchft_amd.quantize_mxfp4_both(state["x"])
        return {"rows": rows.dequantize(), "row_scales": rows.scales, "columns": cols.dequantize(), "column_scales": cols.scales}
    if op == "serve":
        return torchft_amd.linear_mxfp4(state["x"], state["weight"])
    if op == "train":
        x, w = state["x"], state["w"]
        y = torchft_amd.linear_mxfp4(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), state["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    if op == "orthogonal":
        return torchft_amd.orthogonalize(state["x"])
    torchft_amd.muon_(state["weights"], state["grads"], state["momenta"], lr=_LR, weight_decay=_DECAY, momentum=_MOMENTUM)
    return {"weights": state["weights"], "momenta": state["momenta"]}


# ---- what a pass cannot do without -------------------------------------------------------------


def _newton_schulz_flops(rows, cols):
    """A and A A are symmetric: half of each is enough."""
    r, k = min(rows, cols), max(rows, cols)
    return _STEPS * (r * r * k + r * r * r + 2 * r * r * k)


def work(case):
    op, size = case["op"], _DTYPES[case["dtype"]].itemsize
    if op == "muon":
        elements = sum(r * c for r, c in _shapes(case))
        return {"bytes": elements * (3 * size + 8), "flops": sum(_newton_schulz_flops(*s) for s in _shapes(case))}
    rows, cols, tokens = case["rows"], case["cols"], case["tokens"]
    if op == "roundtrip":
        scales = rows * -(-cols // 32) + cols * -(-rows // 32)
        return {"bytes": 3 * rows * cols * size + scales, "flops": 4 * rows * cols}
    if op == "orthogonal":
        return {"bytes": 2 * rows * cols * size, "flops": _newton_schulz_flops(rows, cols)}
    product = 2 * tokens * rows * cols
    if op == "serve":
        weight = rows * -(-cols // 32) * 17
        return {"bytes": weight + tokens * (rows + cols) * size, "flops": product}
    return {"bytes": 2 * (tokens * cols + rows * cols + tokens * rows) * size, "flops": 3 * product}


# ---- in 64 bits --------------------------------------------------------------------------------


def _nearest(x):
    """x's rows in blocks of 32, each element at the nearest value of its block's grid, and the scales."""
    n = x.shape[1]
    x = x.detach().double()
    x = torch.cat([x, x.new_zeros(x.shape[0], -n % 32)], 1).reshape(x.shape[0], -1, 32)
    power = torch.floor(torch.log2(x.abs().max(-1).values)) - 2
    power = power.clamp(min=-127, max=127)
    scale = torch.exp2(power)[..., None]
    v = x / scale
    grid = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=1))) - 1)
    v = (torch.round(v / grid) * grid).clamp(-6, 6) * scale
    return v.reshape(x.shape[0], -1)[:, :n], (power + 127).to(torch.uint8)


def _orthogonal64(u):
    x = u.double()
    if x.shape[0] > x.shape[1]:
        return _orthogonal64(u.t()).t()
    x = x / max(float(torch.linalg.matrix_norm(x)), _EPS)
    eye = torch.eye(x.shape[0], dtype=x.dtype, device=x.device)
    for _ in range(_STEPS):
        a = x @ x.t()
        x = (_A * eye + _B * a + _C * a @ a) @ x
    return x


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "roundtrip":
        (rows, row_scales), (cols, col_scales) = _nearest(state["x"]), _nearest(state["x"].t())
        return {"rows": rows, "row_scales": row_scales, "columns": cols, "column_scales": col_scales}
    if op == "serve":
        low, high = state["codes"] & 15, state["codes"] >> 4
        code = torch.stack([low, high], -1).reshape(low.shape[0], -1, 32).long()
        magnitude = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=code.device)[code % 8]
        weight = torch.where(code > 7, -magnitude, magnitude) * torch.exp2(state["scales"].double() - 127)[..., None]
        return _nearest(state["x"])[0] @ weight.reshape(low.shape[0], -1)[:, :case["cols"]].t()
    if op == "train":
        x, w, dy = state["x"], state["w"], state["dy"]
        return {"y": _nearest(x)[0] @ _nearest(w)[0].t(), "dx": _nearest(dy)[0] @ _nearest(w.t())[0].t(),
                "dw": _nearest(dy.t())[0] @ _nearest(x.t())[0].t()}
    if op == "orthogonal":
        return _orthogonal64(state["x"])
    weights, momenta = [], []
    for w, g, m in zip(state["weights"], state["grads"], state["momenta"]):
        g = g.double()
        m = _MOMENTUM * m.double() + (1 - _MOMENTUM) * g
        scale = math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
        weights.append((1 - _LR * _DECAY) * w.double() - _LR * scale * _orthogonal64((1 - _MOMENTUM) * g + _MOMENTUM * m))
        momenta.append(m)
    return {"weights": weights, "momenta": momenta}
