"""The attention path of a serving step, with vLLM's signatures: rotary
positions, the paged key / value cache, quantised as it is written, its
read-back, and attention over it for single tokens and drafted trees.

Like torch_mcpu_b200.ops (which re-exports every function here), each call
checks its arguments, enqueues on torch's current stream of the tensors'
device and returns; there is no CPU fallback.
"""

from __future__ import annotations

import ctypes
import math
import struct

import torch

from . import _lib

_FLOAT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_HALF = {torch.bfloat16: 1, torch.float16: 2}
_SMALL = {torch.float8_e4m3fn: 10, torch.int8: 8}
_CACHE = struct.Struct("=4Q13q6i")  # mcpuKvCache of include/mcpu_ops.h
_ZEROS = (0, 0, 0)


class _on:
    """The tensors' device as the current one while a call is enqueued."""

    __slots__ = ("index", "before")

    def __init__(self, device: torch.device):
        self.index = device.index

    def __enter__(self):
        self.before = torch._C._cuda_getDevice()
        if self.before != self.index:
            torch._C._cuda_setDevice(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch._C._cuda_setDevice(self.before)


def _fail(op: str, why: str):
    raise RuntimeError(f"{op}: {why}")


def _same_device(op: str, device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            _fail(op, f"{name} is on {t.device}, expected {device}")


def _device_of(op: str, t: torch.Tensor, name: str) -> torch.device:
    if not t.is_cuda:
        _fail(op, f"{name} must be a device tensor (got device {t.device}); the mcpu B200 ops have no CPU fallback")
    return t.device


def _heads(op: str, t: torch.Tensor, name: str, head_size: int):
    """(heads, token stride, head stride) of [tokens, heads * head_size] or
    [tokens, heads, head_size] with contiguous heads."""
    if t.dim() == 2:
        if t.shape[1] % head_size or (t.stride(1) != 1 and t.shape[1] > 1):
            _fail(op, f"{name} must be [tokens, heads * {head_size}] with contiguous rows")
        return t.shape[1] // head_size, t.stride(0), head_size
    if t.dim() != 3 or t.shape[2] != head_size or (t.stride(2) != 1 and head_size > 1):
        _fail(op, f"{name} must be [tokens, heads, {head_size}] with contiguous heads")
    return t.shape[1], t.stride(0), t.stride(1)


def _writable(op: str, name: str, tokens: int, heads: int, size: int, tok: int, head: int) -> None:
    """In-place tensors: no two of their elements at the same place."""
    inner = size if heads <= 1 else (heads - 1) * head + size
    disjoint = (heads <= 1 or head >= size) and (tokens <= 1 or tok >= inner)
    if not disjoint and tokens > 1 and heads > 1 and tok >= size and head >= (tokens - 1) * tok + size:
        disjoint = True  # heads outside, tokens inside
    if not disjoint:
        _fail(op, f"{name} is written in place and must not overlap itself")


def _positions(op: str, positions: torch.Tensor, tokens: int, table: torch.Tensor) -> None:
    if positions.dtype != torch.int64 or positions.dim() != 1 or positions.shape[0] != tokens or (
            tokens > 1 and positions.stride(0) != 1):
        _fail(op, f"positions must be a contiguous int64 [{tokens}] tensor")
    if table.dtype != torch.float32 or table.dim() != 2 or not table.is_contiguous():
        _fail(op, "cos_sin_cache must be a contiguous float32 [max_position, rotary_dim] tensor")


def _cache(op: str, key_cache: torch.Tensor, value_cache: torch.Tensor, k_scale, v_scale, dtype, writes: bool):
    """mcpuKvCache as bytes, after the checks that need the tensors."""
    if key_cache.dim() != 4 or value_cache.shape != key_cache.shape:
        _fail(op, "key_cache and value_cache must both be [num_blocks, block_size, kv_heads, head_size]")
    if dtype not in _HALF:
        _fail(op, f"bfloat16 or float16 tensors expected, got {dtype}")
    kind = key_cache.dtype
    if value_cache.dtype != kind or (kind != dtype and kind not in _SMALL):
        _fail(op, f"the caches must hold {dtype}, float8_e4m3fn or int8 (got {kind}, {value_cache.dtype})")
    blocks, block, kv, head = key_cache.shape
    ks, vs = key_cache.stride(), value_cache.stride()
    if ks[3] != 1 or vs[3] != 1:
        _fail(op, "cache rows must be contiguous")
    if writes:
        for name, st in (("key_cache", ks), ("value_cache", vs)):
            reach = head
            for st_i, n in sorted(((st[0], blocks), (st[1], block), (st[2], kv))):
                if n > 1:
                    if st_i < reach:
                        _fail(op, f"{name} must not overlap itself")
                    reach = (n - 1) * st_i + reach
    if kind == dtype:
        if k_scale is not None or v_scale is not None:
            _fail(op, f"a {kind} cache has no scales")
        return _CACHE.pack(key_cache.data_ptr(), value_cache.data_ptr(), 0, 0, blocks, *ks[:3], *vs[:3], *_ZEROS,
                           *_ZEROS, block, kv, head, _HALF[dtype], 0, 0)
    if k_scale is None or v_scale is None:
        _fail(op, f"a {kind} cache needs k_scale and v_scale")
    if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32 or k_scale.shape != v_scale.shape:
        _fail(op, "k_scale and v_scale must be float32 tensors of one shape")
    if tuple(k_scale.shape) == (blocks, block, kv):
        mode, k3, v3 = 2, k_scale.stride(), v_scale.stride()
        if writes and any(n > 1 and s == 0 for st in (k3, v3) for n, s in zip(k_scale.shape, st)):
            _fail(op, "scales that are written must not overlap themselves")
    elif k_scale.numel() == 1:
        mode, k3, v3 = 1, _ZEROS, _ZEROS
    elif tuple(k_scale.shape) == (kv,):
        mode, k3, v3 = 1, (0, 0, k_scale.stride(0)), (0, 0, v_scale.stride(0))
    else:
        _fail(op, f"scales must have 1, [{kv}] or [{blocks}, {block}, {kv}] elements, got {tuple(k_scale.shape)}")
    return _CACHE.pack(key_cache.data_ptr(), value_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), blocks,
                       *ks[:3], *vs[:3], *k3, *v3, block, kv, head, _SMALL[kind], mode, 0)


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
                 (32) and "beta_slow" (1) times in o positions; cos and sin
                 times "attention_factor" (0.1 ln s + 1)."""
    op = "rotary_cos_sin_cache"
    if rotary_dim <= 0 or rotary_dim % 2 or max_position <= 0 or base <= 0:
        _fail(op, "max_position and base must be positive, rotary_dim even and positive")
    scaling = dict(scaling or {})
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in ("default", "linear", "dynamic", "llama3", "yarn"):
        _fail(op, f"unknown rope_type {kind!r}")
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

        lo = max(math.floor(dim_of(float(scaling.get("beta_fast", 32)))), 0)
        hi = min(math.ceil(dim_of(float(scaling.get("beta_slow", 1)))), rotary_dim - 1)
        ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        inv = inv / factor * ramp + inv * (1 - ramp)
        amp = float(scaling.get("attention_factor") or (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0))
    angle = torch.arange(max_position, dtype=torch.float64)[:, None] * inv[None]
    table = torch.cat([angle.cos() * amp, angle.sin() * amp], dim=1).float()
    return table if device is None else table.to(device)


def rotary_embedding(positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor | None, head_size: int,
                     cos_sin_cache: torch.Tensor, is_neox: bool = True) -> None:
    """vLLM's rotary_embedding (vllm/_custom_ops.py, rotary_embedding), in
    place: the first rotary_dim = cos_sin_cache.size(1) dimensions of every
    head of query and key ([tokens, heads * head_size] or [tokens, heads,
    head_size], float32, bfloat16 or float16; views of a larger tensor are
    fine) are rotated by their position's angles.  is_neox: pairs (i, i +
    rotary_dim / 2), else (2i, 2i + 1).  Results are rounded once."""
    op = "rotary_embedding"
    device = _device_of(op, query, "query")
    _same_device(op, device, positions=positions, key=key, cos_sin_cache=cos_sin_cache)
    if query.dtype not in _FLOAT or (key is not None and key.dtype != query.dtype):
        _fail(op, "query and key must both be float32, bfloat16 or float16")
    tokens = query.shape[0]
    _positions(op, positions, tokens, cos_sin_cache)
    part = cos_sin_cache.shape[1]
    if part > head_size:
        _fail(op, f"rotary_dim {part} exceeds head_size {head_size}")
    heads, qt, qh = _heads(op, query, "query", head_size)
    _writable(op, "query", tokens, heads, part, qt, qh)
    kv, kt, kh, kptr = 0, 0, 0, 0
    if key is not None:
        kv, kt, kh = _heads(op, key, "key", head_size)
        if key.shape[0] != tokens:
            _fail(op, f"key has {key.shape[0]} tokens, query {tokens}")
        _writable(op, "key", tokens, kv, part, kt, kh)
        kptr = key.data_ptr()
    with _on(device) as stream:
        _lib.check(_lib.load().mcpu_rotary_embedding(
            positions.data_ptr(), tokens, query.data_ptr(), heads, qt, qh, kptr, kv, kt, kh, part,
            cos_sin_cache.data_ptr(), cos_sin_cache.shape[0], int(bool(is_neox)), _FLOAT[query.dtype], stream), op)


def _write(op, positions, query, key, value, table, is_neox, key_cache, value_cache, slot_mapping, k_scale, v_scale):
    device = _device_of(op, key, "key")
    _same_device(op, device, positions=positions, query=query, value=value, cos_sin_cache=table, key_cache=key_cache,
                 value_cache=value_cache, slot_mapping=slot_mapping, k_scale=k_scale, v_scale=v_scale)
    if value.dtype != key.dtype or (query is not None and query.dtype != key.dtype):
        _fail(op, "query, key and value must have one type")
    cache = _cache(op, key_cache, value_cache, k_scale, v_scale, key.dtype, True)
    _, _, kv_heads, head_size = key_cache.shape
    tokens = key.shape[0]
    kv, kt, kh = _heads(op, key, "key", head_size)
    kv2, vt, vh = _heads(op, value, "value", head_size)
    if kv != kv_heads or kv2 != kv_heads or value.shape[0] != tokens:
        _fail(op, f"key and value must be [{tokens}, {kv_heads}, {head_size}], as the cache is")
    if slot_mapping.dtype != torch.int64 or tuple(slot_mapping.shape) != (tokens,) or (
            tokens > 1 and slot_mapping.stride(0) != 1):
        _fail(op, f"slot_mapping must be a contiguous int64 [{tokens}] tensor")
    heads = qt = qh = qptr = part = reach = pptr = tptr = 0
    if table is not None:
        _positions(op, positions, tokens, table)
        reach, part = table.shape
        if part == 0 or part > head_size:
            _fail(op, f"rotary_dim {part} must be in 1..head_size ({head_size})")
        pptr, tptr = positions.data_ptr(), table.data_ptr()
        if query is not None:
            heads, qt, qh = _heads(op, query, "query", head_size)
            if query.shape[0] != tokens:
                _fail(op, f"query has {query.shape[0]} tokens, key {tokens}")
            _writable(op, "query", tokens, heads, part, qt, qh)
            qptr = query.data_ptr()
    with _on(device) as stream:
        _lib.check(_lib.load().mcpu_rotary_reshape_and_cache(
            pptr, tokens, qptr, heads, qt, qh, key.data_ptr(), kt, kh, value.data_ptr(), vt, vh, part, tptr, reach,
            int(bool(is_neox)), _HALF[key.dtype], slot_mapping.data_ptr(), cache, stream), op)


def reshape_and_cache(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                      slot_mapping: torch.Tensor, k_scale: torch.Tensor | None = None,
                      v_scale: torch.Tensor | None = None) -> None:
    """Writes the rows of key and value [tokens, kv_heads, head_size] into
    their slots (slot_mapping[t] = block * block_size + place; negative: not
    written; no slot twice) of a paged cache [num_blocks, block_size,
    kv_heads, head_size] (vLLM's reshape_and_cache_flash layout; strided views
    such as a [num_blocks, kv_heads, block_size, head_size] tensor permuted
    are fine).

    The cache holds the rows' own type, or float8_e4m3fn / int8 with float32
    scales: k_scale, v_scale of [num_blocks, block_size, kv_heads] are written
    with the rows (max|x| / 448 or / 127), those of one element or [kv_heads]
    are given by the caller.  Values are rn(x / scale), correctly rounded."""
    _write("reshape_and_cache", None, None, key, value, None, True, key_cache, value_cache, slot_mapping, k_scale,
           v_scale)


def rotary_reshape_and_cache(positions: torch.Tensor, query: torch.Tensor | None, key: torch.Tensor,
                             value: torch.Tensor, cos_sin_cache: torch.Tensor, is_neox: bool, key_cache: torch.Tensor,
                             value_cache: torch.Tensor, slot_mapping: torch.Tensor,
                             k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> None:
    """rotary_embedding and reshape_and_cache in one launch: query is rotated
    in place, the rotated key goes to the cache only (key is left as it is).
    Results are those of the two calls, bit for bit."""
    _write("rotary_reshape_and_cache", positions, query, key, value, cos_sin_cache, is_neox, key_cache, value_cache,
           slot_mapping, k_scale, v_scale)


def _table(op: str, block_table: torch.Tensor, batch: int) -> None:
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != batch or (
            block_table.shape[1] > 1 and block_table.stride(1) != 1):
        _fail(op, f"block_table must be an int32 [{batch}, blocks] tensor with contiguous rows")
    if batch > 1 and block_table.stride(0) < block_table.shape[1]:
        _fail(op, "block_table rows must not overlap")


def _int32(op: str, t: torch.Tensor, name: str, n: int) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != (n,) or (n > 1 and t.stride(0) != 1):
        _fail(op, f"{name} must be a contiguous int32 [{n}] tensor")


def gather_cache(key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor,
                 cu_seq_lens: torch.Tensor, key_out: torch.Tensor, value_out: torch.Tensor,
                 k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                 seq_starts: torch.Tensor | None = None) -> None:
    """Reads sequences back from their pages into the contiguous key_out and
    value_out [tokens, kv_heads, head_size] (bfloat16 or float16),
    dequantising an 8-bit cache: rows cu_seq_lens[b] .. cu_seq_lens[b + 1]
    hold sequence b from its token seq_starts[b] (0 where not given) on.
    Rows behind cu_seq_lens[-1] are left as they are."""
    op = "gather_cache"
    device = _device_of(op, key_cache, "key_cache")
    _same_device(op, device, value_cache=value_cache, block_table=block_table, cu_seq_lens=cu_seq_lens,
                 key_out=key_out, value_out=value_out, k_scale=k_scale, v_scale=v_scale, seq_starts=seq_starts)
    if value_out.dtype != key_out.dtype or key_out.shape != value_out.shape:
        _fail(op, "key_out and value_out must have one shape and type")
    cache = _cache(op, key_cache, value_cache, k_scale, v_scale, key_out.dtype, False)
    if key_out.dim() != 3 or key_out.shape[1:] != key_cache.shape[2:] or not (
            key_out.is_contiguous() and value_out.is_contiguous()):
        _fail(op, f"outputs must be contiguous [tokens, {key_cache.shape[2]}, {key_cache.shape[3]}] tensors")
    batch = block_table.shape[0]
    _table(op, block_table, batch)
    _int32(op, cu_seq_lens, "cu_seq_lens", batch + 1)
    if seq_starts is not None:
        _int32(op, seq_starts, "seq_starts", batch)
    with _on(device) as stream:
        _lib.check(_lib.load().mcpu_gather_cache(
            cache, block_table.data_ptr(), max(block_table.stride(0), block_table.shape[1]), block_table.shape[1], batch,
            cu_seq_lens.data_ptr(), 0 if seq_starts is None else seq_starts.data_ptr(), key_out.data_ptr(),
            value_out.data_ptr(), key_out.shape[0], _HALF[key_out.dtype], stream), op)


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
    (undefined in an output made by the call)."""
    op = "tree_attention"
    device = _device_of(op, query, "query")
    _same_device(op, device, key_cache=key_cache, value_cache=value_cache, block_table=block_table, seq_lens=seq_lens,
                 cu_query_lens=cu_query_lens, tree_mask=tree_mask, k_scale=k_scale, v_scale=v_scale, out=out)
    cache = _cache(op, key_cache, value_cache, k_scale, v_scale, query.dtype, False)
    if query.dim() != 3:
        _fail(op, "query must be [tokens, heads, head_size]")
    tokens, heads, head_size = query.shape
    _, _, kv, head2 = key_cache.shape
    if head2 != head_size or query.stride(2) != 1:
        _fail(op, f"query must have contiguous heads of the cache's size {head2}")
    if kv == 0 or heads % kv:
        _fail(op, f"{heads} query heads cannot share {kv} key / value heads evenly")
    batch = block_table.shape[0]
    _table(op, block_table, batch)
    _int32(op, seq_lens, "seq_lens", batch)
    _int32(op, cu_query_lens, "cu_query_lens", batch + 1)
    words = mstride = mptr = 0
    if tree_mask is not None:
        if tree_mask.dtype != torch.int64 or tree_mask.dim() != 2 or tree_mask.shape[0] != tokens or (
                tree_mask.shape[1] > 1 and tree_mask.stride(1) != 1):
            _fail(op, f"tree_mask must be an int64 [{tokens}, words] tensor with contiguous rows")
        words, mptr = tree_mask.shape[1], tree_mask.data_ptr()
        mstride = tree_mask.stride(0) if tokens > 1 else words
        if words < 1 or (tokens > 1 and mstride < words):
            _fail(op, "tree_mask rows must hold at least one word and not overlap")
    if out is None:
        out = torch.empty((tokens, heads, head_size), dtype=query.dtype, device=device)
    else:
        if out.shape != query.shape or out.dtype != query.dtype or out.stride(2) != 1:
            _fail(op, f"out must be a {query.dtype} {tuple(query.shape)} tensor with contiguous heads")
        _writable(op, "out", tokens, heads, head_size, out.stride(0), out.stride(1))
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=device) if return_lse else None
    lib = _lib.load()
    with _on(device) as stream:
        need = ctypes.c_uint64()
        _lib.check(lib.mcpu_tree_attention_workspace_bytes(max_query_len, heads, kv, head_size, ctypes.byref(need)), op)
        work = torch.empty(need.value, dtype=torch.uint8, device=device)
        _lib.check(lib.mcpu_tree_attention(
            query.data_ptr(), query.stride(0), query.stride(1), tokens, heads, out.data_ptr(), out.stride(0),
            out.stride(1), 0 if lse is None else lse.data_ptr(), _HALF[query.dtype], cache, block_table.data_ptr(),
            max(block_table.stride(0), block_table.shape[1]), block_table.shape[1], batch, seq_lens.data_ptr(),
            cu_query_lens.data_ptr(), max_query_len, mptr, mstride, words, scale, work.data_ptr(), need.value, stream),
            op)
    return (out, lse) if return_lse else out
