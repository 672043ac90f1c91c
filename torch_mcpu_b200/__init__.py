"""torch_mcpu on B200: the mcpu device hot path as sm_100a CUDA.

The product is the C-ABI library libtorch_mcpu_b200.so (include/openreg.h,
include/mcpu_ops.h); this package builds it in-tree and exposes the ops with
the reference's Python signatures.
"""

from . import _lib  # noqa: F401
from .ops import (  # noqa: F401
    device_error,
    gather_cache,
    gemm_swiglu,
    grouped_topk,
    grouped_topk_exact_rows,
    grouped_topk_moe_align,
    interleave_gate_up,
    mm_nt,
    reshape_and_cache,
    rms_norm,
    rotary_cos_sin_cache,
    rotary_embedding,
    rotary_reshape_and_cache,
    sigmoid,
    silu,
    silu_and_mul,
    tree_attention,
)

__all__ = ["grouped_topk", "grouped_topk_exact_rows", "grouped_topk_moe_align", "silu_and_mul", "rms_norm", "mm_nt",
           "gemm_swiglu", "interleave_gate_up", "device_error", "sigmoid", "silu",
           "rotary_cos_sin_cache", "rotary_embedding", "reshape_and_cache", "rotary_reshape_and_cache", "gather_cache",
           "tree_attention"]
