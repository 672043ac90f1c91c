"""Plain 64-bit forms of the attention path's operators, for its tests."""

import math

import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
# bits of the significand (with the leading one) and the exponent of the least subnormal
FORMAT = {torch.bfloat16: (8, -133), torch.float16: (11, -24), torch.float8_e4m3fn: (4, -9)}


def nearest(x, dtype):
    """64-bit values rounded once to dtype (ties to even), still in 64 bits."""
    bits, low = FORMAT[dtype]
    e = torch.frexp(x)[1].clamp(min=low + bits)
    step = torch.ldexp(torch.ones_like(x), e - bits)
    return torch.round(x / step) * step


def rotated(x, positions, table, neox):
    """x [tokens, heads, size] rotated in 64 bits, not rounded."""
    part = table.shape[1]
    row = table[positions].double()[:, None]
    c, s = row[..., : part // 2], row[..., part // 2:]
    y = x.double().clone()
    a, b = (slice(0, part // 2), slice(part // 2, part)) if neox else (slice(0, part, 2), slice(1, part, 2))
    xa, xb = x.double()[..., a], x.double()[..., b]
    y[..., a] = xa * c - xb * s
    y[..., b] = xb * c + xa * s
    return y


def quantised(x, dtype, scale=None):
    """(values held, scales) of rows x [..., size] in 64 bits: token scales, or given ones broadcastable to x."""
    top = LARGEST[dtype]
    if scale is None:
        scale = (x.abs().amax(-1) / top).float()
        by = scale.double()[..., None]
    else:
        by = scale.double()
    q = torch.where(by == 0, torch.zeros_like(x), x / by)
    q = torch.round(q).clamp(-127, 127) if dtype == torch.int8 else nearest(q.clamp(-448, 448), dtype)
    return q, scale


def scale_view(scale, shape):
    """Any accepted form of scales as [blocks, block, kv_heads, 1]."""
    blocks, block, kv, _ = shape
    if scale.numel() == 1 and scale.dim() != 3:
        return scale.double().reshape(1, 1, 1, 1).expand(blocks, block, kv, 1)
    if scale.dim() == 1:
        return scale.double().view(1, 1, kv, 1).expand(blocks, block, kv, 1)
    return scale.double()[..., None]


def values_of(cache, scale):
    v = cache.double()
    return v if scale is None else v * scale_view(scale, cache.shape)


def rows_of(values, table_row, block, n, start=0):
    at = torch.arange(start, start + n, device=values.device)
    return values[table_row[at // block].long(), at % block]


def attention(query, keys, values, block_table, seq_lens, cu, scale, mask=None, absolute=False):
    """(out, lse, tolerance parts) per token in 64 bits; keys, values are 64-bit caches.  Tokens outside requests: None.
    The last result holds, per token and head, A = sum p |v| / sum p, sum |v| and the largest scale * sum |q k|."""
    T, H, D = query.shape
    block, kv = keys.shape[1], keys.shape[2]
    dev = query.device
    out = torch.zeros(T, H, D, dtype=torch.float64, device=dev)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64, device=dev)
    spread = torch.zeros(T, H, D, dtype=torch.float64, device=dev)
    total_v = torch.zeros(T, H, D, dtype=torch.float64, device=dev)
    reach = torch.zeros(T, H, dtype=torch.float64, device=dev)
    cu, lens = cu.tolist(), seq_lens.tolist()
    for b, L in enumerate(lens):
        t0, n = cu[b], cu[b + 1] - cu[b]
        if n == 0 or L == 0:
            continue
        k = rows_of(keys, block_table[b], block, L)
        v = rows_of(values, block_table[b], block, L)
        for i in range(n):
            t = t0 + i
            seen = torch.ones(L, dtype=torch.bool)
            for d in range(n):
                seen[L - n + d] = d <= i if mask is None else bool((int(mask[t, d // 64]) >> (d % 64)) & 1)
            seen = seen.to(dev)
            if not seen.any():
                continue
            for h in range(H):
                kk, vv, q = k[seen][:, h * kv // H], v[seen][:, h * kv // H], query[t, h].double()
                s = kk @ q * scale
                m = s.max()
                if m == -math.inf:
                    continue
                p = torch.exp(s - m)
                out[t, h] = p @ vv / p.sum()
                lse[t, h] = m + torch.log(p.sum())
                spread[t, h] = p @ vv.abs() / p.sum()
                total_v[t, h] = vv.abs().sum(0)
                reach[t, h] = ((kk.abs() @ q.abs()) * abs(scale)).max()
    return out, lse, (spread, total_v, reach)
