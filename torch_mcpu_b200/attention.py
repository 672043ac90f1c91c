"""The attention path of a serving step, with vLLM's signatures: rotary
positions, the paged key / value cache, quantised as it is written, its
read-back, and attention over it for single tokens and drafted trees.

Like torch_mcpu_b200.ops (which re-exports every function here), each call
checks its arguments, enqueues on torch's current stream of the tensors'
device and returns; there is no CPU fallback.  The operators have no
gradients: tensors that require one are refused while gradients are recorded.
"""

from __future__ import annotations

import ctypes
import importlib.util
import math
import os

import torch

from . import _lib

_ops = None


def _native():
    """The module behind the calls (csrc_torch/cuda/attention_module.cpp),
    bound to the loaded device library."""
    global _ops
    if _ops is None:
        from . import build_ext

        lib = _lib.load()
        path = build_ext.OPS_SO
        if not os.path.exists(path) or (os.environ.get("MCPU_AUTOBUILD") == "1" and not build_ext.ops_up_to_date()):
            path = build_ext.build_ops()
        spec = importlib.util.spec_from_file_location(build_ext.OPS_NAME, path)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        mod.bind(*(ctypes.cast(getattr(lib, f), ctypes.c_void_p).value for f in (
            "mcpu_rotary_embedding", "mcpu_rotary_reshape_and_cache", "mcpu_gather_cache", "mcpu_tree_attention",
            "mcpu_tree_attention_workspace_bytes", "mcpuGetLastErrorString")))
        _ops = mod
    return _ops


def _fail(op: str, why: str):
    raise RuntimeError(f"{op}: {why}")


# Keys of a configuration's scaling that each kind reads, beside its name; those of _SAID say what the call says already, or
# nothing about the table
_SCALINGS = {
    "default": (),
    "linear": ("factor", "original_max_position_embeddings"),
    "dynamic": ("factor", "original_max_position_embeddings"),
    "llama3": ("factor", "original_max_position_embeddings", "low_freq_factor", "high_freq_factor"),
    "yarn": ("factor", "original_max_position_embeddings", "beta_fast", "beta_slow", "attention_factor", "mscale",
             "mscale_all_dim", "truncate"),
}
_SAID = ("rope_type", "type", "rope_theta", "partial_rotary_factor", "finetuned")


def rotary_cos_sin_cache(max_position: int, rotary_dim: int, base: float = 10000.0, scaling: dict | None = None,
                         device=None) -> torch.Tensor:
    """The float32 [max_position, rotary_dim] table of rotary_embedding: row p
    holds cos then sin of p * f_i for f_i = base^(-2i / rotary_dim), made once
    when a model is loaded.  Angles are taken in 64 bits: in 32 the angle of
    position 100000 is off by up to 2^-8.

    scaling stretches the positions for longer contexts, in the form model
    configurations use: {"rope_type": ..., "factor": s, ...} with rope_type
      "linear"   f_i / s
      "dynamic"  base * (s m / o - (s - 1))^(d / (d - 2)) for m =
                 max_position beyond o = "original_max_position_embeddings"
      "llama3"   f_i where its wavelength is below o / "high_freq_factor",
                 f_i / s above o / "low_freq_factor", blended between
      "yarn"     blended over the dimensions that turn between "beta_fast"
                 (32) and "beta_slow" (1) times in o positions, from whole
                 dimensions unless "truncate" is false; cos and sin times
                 "attention_factor", else, with m(c) = 0.1 c ln s + 1 for
                 s > 1, m("mscale") / m("mscale_all_dim") where both are
                 given, else m(1)
    Keys whose value is None count as not given; "rope_theta" must be base, and
    "partial_rotary_factor" is what rotary_dim says.  Other keys are refused:
    they would make another table."""
    op = "rotary_cos_sin_cache"
    if rotary_dim <= 0 or rotary_dim % 2 or max_position <= 0 or base <= 0:
        _fail(op, "max_position and base must be positive, rotary_dim even and positive")
    scaling = {k: v for k, v in (scaling or {}).items() if v is not None}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in _SCALINGS:
        _fail(op, f"unknown rope_type {kind!r}")
    if scaling.get("type", kind) != kind:
        _fail(op, f"rope_type is {kind!r}, type {scaling['type']!r}")
    unknown = [k for k in scaling if k not in _SCALINGS[kind] and k not in _SAID]
    if unknown:
        _fail(op, f"{kind} scaling does not know {', '.join(map(str, unknown))}")
    if float(scaling.get("rope_theta", base)) != float(base):
        _fail(op, f"rope_theta is {scaling['rope_theta']}, base {base}")
    if ("mscale" in scaling) != ("mscale_all_dim" in scaling):
        _fail(op, "mscale and mscale_all_dim are given together: what one alone means differs between models")
    factor = float(scaling.get("factor", 1.0))
    if factor <= 0:
        _fail(op, "factor must be positive")
    if kind in ("dynamic", "llama3", "yarn"):
        needed = ["original_max_position_embeddings"] + (["low_freq_factor", "high_freq_factor"] if kind == "llama3" else [])
        missing = [k for k in needed if k not in scaling]
        if missing:
            _fail(op, f"{kind} scaling needs {', '.join(missing)}")
        original = float(scaling["original_max_position_embeddings"])
    if kind == "dynamic" and max_position > original:
        if rotary_dim <= 2:
            _fail(op, "dynamic scaling needs rotary_dim > 2")
        base = base * (factor * max_position / original - (factor - 1)) ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    inv = float(base) ** (-i / rotary_dim)
    amp = 1.0
    if kind == "linear":
        inv = inv / factor
    elif kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not high > low > 0:
            _fail(op, "high_freq_factor must be above low_freq_factor, both positive")
        turns = original * inv / (2 * math.pi)  # original length in wavelengths
        blend = ((turns - low) / (high - low)).clamp(0, 1)
        inv = (1 - blend) * inv / factor + blend * inv
    elif kind == "yarn":
        def dim_of(turns: float) -> float:
            return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = dim_of(float(scaling.get("beta_fast", 32))), dim_of(float(scaling.get("beta_slow", 1)))
        if scaling.get("truncate", True):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, rotary_dim - 1)
        ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        inv = inv / factor * ramp + inv * (1 - ramp)
        def grown(c: float) -> float:
            return 0.1 * c * math.log(factor) + 1.0 if factor > 1 else 1.0

        amp = float(scaling.get("attention_factor", 0)) or grown(float(scaling.get("mscale", 1))) / grown(
            float(scaling.get("mscale_all_dim", 0)))
    angle = torch.arange(max_position, dtype=torch.float64)[:, None] * inv[None]
    table = torch.cat([angle.cos() * amp, angle.sin() * amp], dim=1).float()
    return table if device is None else table.to(device)


def rotary_embedding(positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor | None, head_size: int,
                     cos_sin_cache: torch.Tensor, is_neox: bool = True) -> None:
    """Rotary positions with vLLM's argument order, in place: the first rotary_dim = cos_sin_cache.size(1) dimensions of every
    head of query and key ([tokens, heads * head_size] or [tokens, heads,
    head_size], float32, bfloat16 or float16; views of a larger tensor are
    fine) are rotated by their position's angles.  is_neox: pairs (i, i +
    rotary_dim / 2), else (2i, 2i + 1).  bfloat16 and float16 results are
    64-bit ones rounded once; float32 ones, a cos - b sin, are off by at most
    2^-24 (|b sin| + |result|)."""
    (_ops or _native()).rotary_embedding(positions, query, key, head_size, cos_sin_cache, is_neox)


def reshape_and_cache(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                      slot_mapping: torch.Tensor, k_scale: torch.Tensor | None = None,
                      v_scale: torch.Tensor | None = None) -> None:
    """Writes the rows of key and value [tokens, kv_heads, head_size] into
    their slots (slot_mapping[t] = block * block_size + place; negative: not
    written; no slot twice) of a paged cache [num_blocks, block_size,
    kv_heads, head_size] (vLLM's layout; strided views
    such as a [num_blocks, kv_heads, block_size, head_size] tensor permuted
    are fine).

    The cache holds the rows' own type, or float8_e4m3fn / int8 with float32
    scales: k_scale, v_scale of [num_blocks, block_size, kv_heads] are written
    with the rows (max|x| / 448 or / 127), those of one element or [kv_heads]
    are given by the caller.  Values are rn(x / scale), correctly rounded."""
    (_ops or _native()).write(None, None, key, value, None, True, key_cache, value_cache, slot_mapping, k_scale, v_scale)


def rotary_reshape_and_cache(positions: torch.Tensor, query: torch.Tensor | None, key: torch.Tensor,
                             value: torch.Tensor, cos_sin_cache: torch.Tensor, is_neox: bool, key_cache: torch.Tensor,
                             value_cache: torch.Tensor, slot_mapping: torch.Tensor,
                             k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> None:
    """rotary_embedding and reshape_and_cache in one launch: query is rotated
    in place, the rotated key goes to the cache only (key is left as it is).
    rotary_dim is a multiple of 16 here.  Results are those of the two calls,
    bit for bit."""
    if cos_sin_cache is None:
        _fail("rotary_reshape_and_cache", "cos_sin_cache is needed")
    (_ops or _native()).write(positions, query, key, value, cos_sin_cache, is_neox, key_cache, value_cache, slot_mapping,
                              k_scale, v_scale)


def gather_cache(key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor,
                 cu_seq_lens: torch.Tensor, key_out: torch.Tensor, value_out: torch.Tensor,
                 k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                 seq_starts: torch.Tensor | None = None) -> None:
    """Reads sequences back from their pages into the contiguous key_out and
    value_out [tokens, kv_heads, head_size] (bfloat16 or float16),
    dequantising an 8-bit cache: rows cu_seq_lens[b] .. cu_seq_lens[b + 1]
    hold sequence b from its token seq_starts[b] (0 where not given) on.
    Rows behind cu_seq_lens[-1] are left as they are."""
    (_ops or _native()).gather_cache(key_cache, value_cache, block_table, cu_seq_lens, key_out, value_out, k_scale, v_scale,
                                     seq_starts)


def tree_attention(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor,
                   seq_lens: torch.Tensor, cu_query_lens: torch.Tensor, max_query_len: int, scale: float,
                   tree_mask: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
                   v_scale: torch.Tensor | None = None, out: torch.Tensor | None = None, return_lse: bool = False):
    """Attention of a decoding step's new tokens over the paged cache that
    already holds their own keys and values.

    query [tokens, heads, head_size] (bfloat16 / float16, head_size 64 or
    128): request b's tokens are cu_query_lens[b] .. cu_query_lens[b + 1]
    (int32), at most max_query_len (up to 256) each; seq_lens[b] (int32) keys
    are in its pages, its new tokens last.  A token sees all of its request's
    context and, of the new tokens, those whose bits are set in its row of
    tree_mask (int64 [tokens, words], bit d of the row for new token d: itself
    and its ancestors in a tree of drafts); without a mask, the ones up to
    itself.  heads is a multiple of kv_heads; scales as in reshape_and_cache.

    Returns the output (`out` where given), with return_lse also the float32
    [tokens, heads] logarithms of the softmax sums.  A token that sees nothing
    gives zeros and -inf; tokens outside every request are left as they are
    (undefined in an output made by the call).  out may be query itself and
    overlaps no other tensor of the call."""
    return (_ops or _native()).tree_attention(query, key_cache, value_cache, block_table, seq_lens, cu_query_lens,
                                              max_query_len, scale, tree_mask, k_scale, v_scale, out, return_lse)
