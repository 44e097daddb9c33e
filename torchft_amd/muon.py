"""Orthogonalised updates: the Muon optimiser's step on averaged gradients (no counterpart in the reference).

A replica that has its averaged gradients (or DiLoCo's averaged pseudo-gradients) replaces the
momentum ``u`` of a weight matrix by the nearest orthogonal matrix, up to singular values between
about 0.7 and 1.2, with a few Newton-Schulz iterations

    X = u / max(|u|, eps);   X <- a X + (b A + c A A) X   with A = X X^T

and takes that as the step:

* :func:`orthogonalize`: the orthogonalisation of one matrix or of a list;
* :func:`muon_`: the whole step of a list of weights, in place;
* :class:`Muon`: the same as a ``torch.optim.Optimizer``.

Products run on the 16-bit matrix cores with float32 sums.  bfloat16 results take one product each,
with the diagonals and the remainders of the iterates kept apart, so that the result is off by less than
its own rounding; float32 and float16 results, and matrices with a side of fewer than 192 (with the
small ones beside them in a list), take three, of high and low parts, with the accuracy of float32 products.
The whole list is worked on at once, 24 matrices to a launch: about 17 launches whatever their number.
The workspace comes from torch's allocator for the length of the call: 8 to 12 bytes an element, 12 to 20 with
three products, and 8 GiB at most for matrices that do not need more each (larger lists are taken in runs).
"""

from __future__ import annotations

import ctypes
import math
from typing import Iterable, Sequence

import torch

from . import _lib
from .quantization import _DTYPE_CODE, _check, _stream_of

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _coefficients(coefficients, steps: int):
    rows = list(coefficients)
    assert steps >= 1, "At least one iteration is required"
    if len(rows) == 3 and all(isinstance(c, (int, float)) for c in rows):
        rows = [rows] * steps
    assert len(rows) == steps and all(len(r) == 3 for r in rows), "coefficients are three numbers, or three for every iteration"
    return (ctypes.c_float * (3 * steps))(*[c for r in rows for c in r])


def _by_rows(t: torch.Tensor) -> bool:
    return (t.shape[1] <= 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= max(1, t.shape[1])) and not t.is_neg()


def _same_order(tensors: tuple) -> "tuple | None":
    """The tensors of one matrix, all stored by rows: as they are, or all transposed (orthogonalisation
    and transposition commute); None if they are stored in different orders."""
    if all(map(_by_rows, tensors)):
        return tensors
    flipped = tuple(t.t() for t in tensors)
    return flipped if all(map(_by_rows, flipped)) else None


def _check_list(name: str, tensors: list, device: torch.device, dtype: torch.dtype, shapes: "list | None") -> None:
    assert all(t.dim() == 2 for t in tensors), "Only 2D tensors are supported"
    assert all(t.device == device for t in tensors), "All inputs must be on the same device"
    assert all(t.dtype == dtype for t in tensors), f"All {name} must be of the same dtype"
    assert dtype in _DTYPE_CODE, "Only fp32, fp16 and bf16 are supported"
    if shapes is not None:
        assert [tuple(t.shape) for t in tensors] == shapes, f"The {name} have other shapes than the first list"


def _check_options(lr: float, weight_decay: float, momentum: float) -> None:
    assert lr >= 0 and weight_decay >= 0 and 0 <= momentum < 1, "lr, weight_decay or momentum is out of range"


# Bytes of workspace that a call takes for several matrices together; what needs more by itself is taken alone.
# So many fill the GPU many times over: 24 of 4096x14336 in bf16, 12.9 GB in one call, take 94.8 ms so, 94.7 in runs of
# 8 GiB, 96.0 of 4, 102.6 of 1; 48 of 2048x5632 24.0, 24.0, 24.0, 27.0.
_WORKSPACE = 8 << 30


def _parts(lib, n: int, shapes, precise: bool) -> "list[tuple[int, int]]":
    """The list in runs of matrices whose workspaces, one beside the other, stay within ``_WORKSPACE``."""
    parts, first, held = [], 0, 0
    for i in range(n):
        size = lib.tftq_newton_schulz_workspace(1, _from(shapes, 2 * i), precise)
        if size < 0:
            _check(size, "tftq_newton_schulz_workspace")
        if i > first and held + size > _WORKSPACE:
            parts.append((first, i))
            first, held = i, 0
        held += size
    return parts + [(first, n)]


def _from(array, first: int):
    """A C array from its element ``first`` on."""
    if first == 0:
        return array
    return ctypes.cast(ctypes.addressof(array) + first * ctypes.sizeof(array._type_), ctypes.POINTER(array._type_))


def _run(outs: list, ins: list, momenta: "list | None", steps_sizes: "list | None", keep: float, momentum: float,
         nesterov: bool, iterations: int, coefficients, eps: float, precise: "bool | None") -> None:
    """out = X, or keep * out - step * X, for every matrix; all lists checked."""
    assert eps >= 0, "eps is negative"
    coefficients = _coefficients(coefficients, iterations)
    device, out_dtype = outs[0].device, outs[0].dtype
    assert device.type == "cuda", "A GPU tensor is required"
    _lib.check_device(device.index)
    if precise is None:
        precise = out_dtype != torch.bfloat16
    after = []  # (the caller's tensor, the one that took its place)

    def in_place(t):
        copy = t.resolve_neg().contiguous() if steps_sizes is not None or momenta is not None else torch.empty_like(t, memory_format=torch.contiguous_format)
        after.append((t, copy))
        return copy

    n = len(outs)
    shapes, strides = (ctypes.c_int64 * (2 * n))(), [(ctypes.c_int64 * n)() for _ in range(3)]
    pointers = [(ctypes.c_void_p * n)() for _ in range(3)]
    held = []
    for i in range(n):
        group = (outs[i], ins[i]) if momenta is None else (outs[i], ins[i], momenta[i])
        ordered = _same_order(group)
        if ordered is None:
            ordered = tuple(t if _by_rows(t) else t.resolve_neg().contiguous() if k == 1 else in_place(t) for k, t in enumerate(group))
        held.append(ordered)
        shapes[2 * i], shapes[2 * i + 1] = ordered[0].shape
        for k, t in enumerate(ordered):
            pointers[k][i] = t.data_ptr()
            strides[k][i] = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    lib = _lib.load()
    size = lib.tftq_newton_schulz_workspace(n, shapes, precise)
    parts = [(0, n)] if size <= _WORKSPACE else _parts(lib, n, shapes, precise)
    for first, last in parts:
        if len(parts) > 1:
            size = lib.tftq_newton_schulz_workspace(last - first, _from(shapes, 2 * first), precise)
        if size < 0:
            _check(size, "tftq_newton_schulz_workspace")
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        what = _lib.NewtonSchulz(
            n=last - first, shapes=_from(shapes, 2 * first), inputs=_from(pointers[1], first), in_stride=_from(strides[1], first),
            in_dtype=_DTYPE_CODE[ins[0].dtype], momenta=_from(pointers[2], first) if momenta is not None else None,
            momenta_stride=_from(strides[2], first) if momenta is not None else None, momentum=momentum, nesterov=nesterov,
            out=_from(pointers[0], first), out_stride=_from(strides[0], first), out_dtype=_DTYPE_CODE[out_dtype],
            steps=(ctypes.c_float * (last - first))(*steps_sizes[first:last]) if steps_sizes is not None else None, keep=keep,
            iterations=iterations, coefficients=coefficients, eps=eps, precise=precise)
        _check(lib.tftq_newton_schulz(ctypes.byref(what), workspace.data_ptr(), size, device.index, _stream_of(device)),
               "tftq_newton_schulz")
        del workspace  # the next part's may take its place: the stream runs them one after the other
    for t, copy in after:
        t.copy_(copy)


@torch.no_grad()
def orthogonalize(matrices: "torch.Tensor | Sequence[torch.Tensor]", steps: int = 5, coefficients=COEFFICIENTS,
                  eps: float = 1e-7, out_dtype: "torch.dtype | None" = None, precise: "bool | None" = None):
    """The Newton-Schulz orthogonalisation of a matrix, or a list with that of each.

    ``coefficients``: ``(a, b, c)``, or one such triple for every one of the ``steps`` iterations; the numbers
    that they make of X are held in 16 bits, scaled by what they can be at most (up to 4e9).
    ``out_dtype``: of the results, the input's by default.  ``precise``: whether products are exact to
    22 bits and not to 11; by default only bfloat16 results do without."""
    single = isinstance(matrices, torch.Tensor)
    ins = [matrices] if single else list(matrices)
    if not ins:
        return []
    _check_list("matrices", ins, ins[0].device, ins[0].dtype, None)
    out_dtype = ins[0].dtype if out_dtype is None else out_dtype
    assert out_dtype in _DTYPE_CODE, "Only fp32, fp16 and bf16 are supported"
    outs = [torch.empty_like(t, dtype=out_dtype) for t in ins]
    _run(outs, ins, None, None, 1.0, 0.0, False, steps, coefficients, eps, precise)
    return outs[0] if single else outs


@torch.no_grad()
def muon_(weights: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], momenta: Sequence[torch.Tensor], lr: float,
          weight_decay: float = 0.0, momentum: float = 0.95, nesterov: bool = True, steps: int = 5,
          coefficients=COEFFICIENTS, eps: float = 1e-7, precise: "bool | None" = None) -> None:
    """One step of Muon on a list of weight matrices, in place:

        m = momentum m + (1 - momentum) g;   u = g + momentum (m - g) with ``nesterov``, else m
        w = (1 - lr weight_decay) w - lr sqrt(max(1, rows / columns)) orthogonalize(u)

    The momenta are float32; weights and gradients are of one type each.  ``precise`` as in
    :func:`orthogonalize`, by the type of the weights."""
    weights, grads, momenta = list(weights), list(grads), list(momenta)
    assert len(weights) == len(grads) == len(momenta), "The lists are of different lengths"
    _check_options(lr, weight_decay, momentum)
    if not weights:
        return
    first = weights[0]
    _check_list("weights", weights, first.device, first.dtype, None)
    shapes = [tuple(w.shape) for w in weights]
    _check_list("grads", grads, first.device, grads[0].dtype, shapes)
    _check_list("momenta", momenta, first.device, torch.float32, shapes)
    sizes = [lr * math.sqrt(max(1.0, r / c)) if r and c else 0.0 for r, c in shapes]
    _run(weights, grads, momenta, sizes, 1.0 - lr * weight_decay, momentum, nesterov, steps, coefficients, eps, precise)
    torch.autograd.graph.increment_version(weights + momenta)  # autograd learns of the writes as of any in place


class Muon(torch.optim.Optimizer):
    """:func:`muon_` as an optimiser, for the matrices of a model (its vectors and its embeddings go to
    another one).  The momentum is float32 whatever the type of the weights.  All weights of a parameter
    group that share device, type and type of gradient are taken in one call."""

    def __init__(self, params: Iterable, lr: float = 0.02, weight_decay: float = 0.0, momentum: float = 0.95,
                 nesterov: bool = True, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7,
                 precise: "bool | None" = None) -> None:
        _check_options(lr, weight_decay, momentum)
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov, steps=steps,
                                      coefficients=coefficients, eps=eps, precise=precise))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            assert all(p.dim() == 2 for p in group["params"]), "Only 2D tensors are supported"
            _check_options(group["lr"], group["weight_decay"], group["momentum"])
        except AssertionError:
            self.param_groups.pop()
            raise

    def load_state_dict(self, state_dict) -> None:
        """As ``torch.optim.Optimizer.load_state_dict``, which brings floating-point state to the type of its
        weight; the momenta stay the float32 numbers that were saved."""
        saved: dict = {}

        def before(_, state):  # after the caller's own hooks, which may have replaced the state
            saved.update(state)

        def after(_):  # before the caller's own
            ids = (i for group in saved["param_groups"] for i in group["params"])
            params = (p for group in self.param_groups for p in group["params"])
            for i, p in zip(ids, params):
                if "momentum" in saved["state"].get(i, ()):
                    self.state[p]["momentum"] = saved["state"][i]["momentum"].to(device=p.device, dtype=torch.float32)

        hooks = self.register_load_state_dict_pre_hook(before), self.register_load_state_dict_post_hook(after, prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            lists: dict = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    state["momentum"] = torch.zeros_like(p, dtype=torch.float32)
                entry = lists.setdefault((p.device, p.dtype, p.grad.dtype), ([], [], []))
                entry[0].append(p)
                entry[1].append(p.grad)
                entry[2].append(state["momentum"])
            options = {k: v for k, v in group.items() if k != "params"}
            for weights, grads, momenta in lists.values():
                muon_(weights, grads, momenta, **{k: options[k] for k in (
                    "lr", "weight_decay", "momentum", "nesterov", "steps", "coefficients", "eps", "precise")})
        return loss
