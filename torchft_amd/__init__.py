"""MI355X-native FP8 quantized-collective kernels, a drop-in for torchft's
``torchft.quantization`` (and its callers in ``torchft.collectives``); and, with no counterpart there,
operators of the training step around them: 4-bit matrices and linear layers on them, Muon's update."""

from .quantization import (  # noqa: F401
    PreparedBucket,
    fused_dequantize_from_fp8,
    fused_quantize_into_fp8,
    fused_reduce_fp8,
    prepare,
)

from .mxfp4 import (  # noqa: F401
    MXFP4Tensor,
    linear_mxfp4,
    matmul_mxfp4,
    quantize_mxfp4,
    quantize_mxfp4_both,
)

from .muon import Muon, muon_, orthogonalize  # noqa: F401

from .collectives import (  # noqa: F401
    allocate_reduce_scatter_output,
    allreduce_quantized,
    get_padded_sizes,
    reduce_scatter_quantized,
)

__all__ = [
    "allocate_reduce_scatter_output",
    "allreduce_quantized",
    "get_padded_sizes",
    "reduce_scatter_quantized",
    "fused_dequantize_from_fp8",
    "fused_quantize_into_fp8",
    "fused_reduce_fp8",
    "prepare",
    "PreparedBucket",
    "MXFP4Tensor",
    "linear_mxfp4",
    "matmul_mxfp4",
    "quantize_mxfp4",
    "quantize_mxfp4_both",
    "Muon",
    "muon_",
    "orthogonalize",
]
