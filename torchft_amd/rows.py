"""Row operators of a training step, between its linear layers (no counterpart in the reference).

* :func:`rms_norm` / :func:`rms_norm_fp8`: root-mean-square norm behind the residual's addition, in the rows' type
  with gradients, or in 8 bits with a scale a row (:func:`dispatch` moves such rows to their experts' places on the same GPU; no
  collective here takes them, and products take their values);
* :func:`dropout`: with a mask that a counter-based generator makes again in the backward pass, added to the residual;
* :func:`embedding`: rows of a table, scaled; its gradient is summed over sorted tokens;
* :func:`sort_by_expert`, :func:`dispatch`, :func:`combine`: tokens by expert, their rows there, and the experts' rows
  back with weights.

All take fp32, fp16 and bf16 tensors in any order (what is not stored in rows is copied first), sum in fp32 in
an order that the arguments alone decide, and round each result once; gradients are computed once (no second
derivatives, no forward mode).  Kernels are enqueued on the current stream of the tensors' device; nothing synchronises the
host, no function keeps anything from one call for the next, and all can be captured into graphs (a backward pass once no
graph of the same leaves is left that was made on the default stream; it is refused until then).  A call while a trace is taken (``make_fx``,
``torch.jit.trace``, ``torch.export``) is refused: the trace would not have its kernels.  There is no CPU or eager fallback.
"""

from __future__ import annotations

import ctypes
import threading

import torch

from . import _build, _lib
from .quantization import _DTYPE_CODE

_FUNCTIONS = ("strerror", "check_device", "rms_norm", "rms_norm_backward_workspace", "rms_norm_backward", "dropout", "embedding",
              "embedding_backward_workspace", "embedding_backward", "expert_sort_workspace", "expert_sort", "dispatch", "combine",
              "combine_backward", "fp8_rows_dequantize")
_native = None
_load_lock = threading.Lock()


def _module():
    """The module that makes the calls, once it knows the library's functions."""
    global _native
    with _load_lock:
        if _native is None:
            lib, module = _lib.load(), _build.load_rows()
            for name in _FUNCTIONS:
                module.bind(name, ctypes.cast(getattr(lib, "tftq_" + name), ctypes.c_void_p).value)
            _native = module
    return _native


class FP8Rows:
    """Rows in 8 bits: ``codes`` (``float8_e4m3fn``) and ``scales`` (float32, ``[..., 1]``) that multiply them, a row's
    largest magnitude / 448 (1 where that is below 2^-126).  ``dtype`` is the type of what they were made of.  It is
    no ``torch.Tensor`` and has no gradient."""

    __slots__ = ("codes", "scales", "dtype")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> None:
        self.codes = codes
        self.scales = scales
        self.dtype = dtype

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dequantize(self, dtype: "torch.dtype | None" = None) -> torch.Tensor:
        """The values that the rows stand for, rounded once to ``dtype``."""
        dtype = self.dtype if dtype is None else dtype
        assert dtype in _DTYPE_CODE, "Only fp32, fp16 and bf16 are supported"
        return (_native or _module()).fp8_rows(self.codes, self.scales, _DTYPE_CODE[dtype])

    def record_stream(self, stream: torch.cuda.Stream) -> None:
        """As ``torch.Tensor.record_stream``: the memory is used on another stream than the one it was made on."""
        self.codes.record_stream(stream)
        self.scales.record_stream(stream)

    def __repr__(self) -> str:
        return f"FP8Rows({'x'.join(map(str, self.shape))}, of {self.dtype}, on {self.device})"


def rms_norm(x: torch.Tensor, weight: "torch.Tensor | None" = None, residual: "torch.Tensor | None" = None, eps: float = 1e-6):
    """``y = h weight / sqrt(mean(h^2) + eps)`` over the last dimension, with ``h = x``, or ``(y, h)`` with
    ``h = x + residual`` rounded to their type: y is the norm of the h that is returned.

    ``weight`` has the type of ``x`` or is float32.  The sum of squares is float32: rows of magnitudes beyond 1e18
    pass its range."""
    return (_native or _module()).rms_norm(x, weight, residual, eps, False)


def rms_norm_fp8(x: torch.Tensor, weight: "torch.Tensor | None" = None, residual: "torch.Tensor | None" = None, eps: float = 1e-6):
    """:func:`rms_norm` with y as :class:`FP8Rows`: the codes are the nearest to ``448 h weight / max |h weight|``, the even one of two that
    are as near.  It has no gradient and refuses one."""
    got = (_native or _module()).rms_norm(x, weight, residual, eps, True)
    rows = FP8Rows(got[0], got[1], x.dtype)
    return rows if residual is None else (rows, got[2])


def dropout(x: torch.Tensor, p: float, seed: "int | torch.Tensor", offset: int = 0, residual: "torch.Tensor | None" = None) -> torch.Tensor:
    """``x`` with every element zero with probability ``p`` and divided by ``1 - p`` otherwise; with ``residual``, its sum with that.

    ``p`` is rounded to a multiple of 2^-16.  Which elements stay depends on ``seed``, ``offset`` and an element's place in
    row-major order alone (``tftq_dropout`` of ``include/tftq.h`` has the generator); the mask is made again in the
    backward pass, not kept.  Calls of one step take one seed and an offset each.  A seed on the GPU (a tensor
    of one int64) is read when the kernel runs: a captured graph draws other numbers after it has changed, which it may
    not between a forward and its backward pass."""
    return (_native or _module()).dropout(x, p, seed, offset, residual)


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, padding_idx: "int | None" = None) -> torch.Tensor:
    """``scale table[ids]``; ``ids`` int64 or int32 of any shape, ``table`` ``[vocabulary, columns]``.

    Numbers outside the table have a row of zeros and no gradient: a rank that holds a part of a vocabulary takes
    ``ids - first`` and adds up the ranks' rows.  ``padding_idx`` has its row and no gradient.  The gradient is a
    whole table of the table's type; a row's sum is float32, in the order of the tokens."""
    return (_native or _module()).embedding(ids, table, scale, padding_idx)


class ExpertOrder:
    """Where the choices of tokens go, by :func:`sort_by_expert`: ``position`` ``[tokens, k]``, the place of a choice; ``order``
    ``[tokens k]``, the choice (token times k plus its number) at a place; ``offsets`` ``[experts + 1]``, where an expert's
    places begin; all int32 on the GPU.  Expert e has the rows ``offsets[e]`` to ``offsets[e + 1]`` of what :func:`dispatch`
    returns; the last offset is the number of places with an expert."""

    __slots__ = ("order", "position", "offsets")

    def __init__(self, order: torch.Tensor, position: torch.Tensor, offsets: torch.Tensor) -> None:
        self.order = order
        self.position = position
        self.offsets = offsets

    @property
    def counts(self) -> torch.Tensor:
        """``[experts]`` numbers of choices."""
        return self.offsets[1:] - self.offsets[:-1]

    def record_stream(self, stream: torch.cuda.Stream) -> None:
        """As ``torch.Tensor.record_stream``: the memory is used on another stream than the one it was made on."""
        for t in (self.order, self.position, self.offsets):
            t.record_stream(stream)

    def __repr__(self) -> str:
        tokens, k = self.position.shape
        return f"ExpertOrder({tokens} tokens, {k} of {self.offsets.numel() - 1} experts, on {self.position.device})"


def sort_by_expert(experts: torch.Tensor, num_experts: int) -> ExpertOrder:
    """The places of the tokens' choices, sorted by expert, those of an expert in the order of their tokens.

    ``experts`` ``[tokens, k]`` (or ``[tokens]``), int64 or int32.  A choice outside ``0 ... num_experts - 1`` (a token that
    is padding, or was dropped) names no expert and has a place behind all others."""
    return ExpertOrder(*(_native or _module()).sort_by_expert(experts, num_experts))


def dispatch(x: "torch.Tensor | FP8Rows", order: ExpertOrder) -> "torch.Tensor | FP8Rows":
    """The rows of the tokens at the places of their choices, ``[tokens k, columns]``; zeros in places without an
    expert.  Gradients sum over a token's choices.  Rows of any elements of 1, 2 or 4 bytes can be sent without one;
    rows in 8 bits take their scales along."""
    native = _native or _module()
    if isinstance(x, FP8Rows):
        return FP8Rows(native.dispatch(x.codes, order.position, order.offsets), native.dispatch(x.scales, order.position, order.offsets), x.dtype)
    return native.dispatch(x, order.position, order.offsets)


def combine(rows: torch.Tensor, order: ExpertOrder, weights: "torch.Tensor | None" = None) -> torch.Tensor:
    """``y[t] = sum over s of weights[t, s] rows[position[t, s]]``, ``[tokens, columns]``: the way back from the
    experts.  Choices without an expert are left out.  ``weights`` ``[tokens, k]`` have the type of the rows or are
    float32, and are 1 by default.  Rows and weights have gradients."""
    return (_native or _module()).combine(rows, order.position, order.offsets, weights)
