"""What is measured of the attention path's operators: rotary positions, the paged key / value cache that is quantised as
it is written, its read-back, and attention over it for single tokens and trees of drafted tokens.

`run` computes them in elementary torch operations, or, where `own` is true, with this repository's kernels.  A state holds
what a serving loop has in hand before the call: the step's projections, the cache with its scales, the block table and
lengths on the device, and the rotary table.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CACHES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {"e4m3": 448.0, "int8": 127.0}


def listed():
    return [
        # one user's decoding step: launch latency is all there is
        dict(name="rotary, one token", op="rotary", tokens=1, heads=32, kv_heads=8, head=128, part=128, layout="half",
             dtype="bf16", reach=8192),
        # a long prefill whose heads rotate only their last 64 of 192 dimensions, in pairs, at far positions
        dict(name="rotary, prefill of a part", op="rotary", tokens=16111, heads=128, kv_heads=1, head=192, part=64,
             layout="interleaved", dtype="bf16", reach=163840),
        # a decoding batch: query and key rotated, key and value quantised into their slots
        dict(name="write, decoding batch", op="write", tokens=256, heads=32, kv_heads=8, head=128, part=128, layout="half",
             dtype="bf16", cache="e4m3", scales="token", block=16, reach=32768, back=False),
        # a prefill chunk of many prompts into a cache with one calibrated scale
        dict(name="write, prefill chunk", op="write", tokens=16383, heads=32, kv_heads=8, head=128, part=64, layout="half",
             dtype="bf16", cache="e4m3", scales="tensor", block=32, reach=131072, back=False),
        # keys without positions, whole numbers in the cache, and the prefix read back for the next chunk's attention
        dict(name="write and read back", op="write", tokens=4099, heads=0, kv_heads=8, head=128, part=0, layout="none",
             dtype="fp16", cache="int8", scales="token", block=16, reach=4099, back=True),
        # one short prefix read back
        dict(name="read back, one prefix", op="read", batch=1, context=777, kv_heads=8, head=128, dtype="bf16", cache="int8",
             scales="token", block=16),
        # the prefixes of a batch read back before a chunk's attention
        dict(name="read back, many prefixes", op="read", batch=24, context=8192, kv_heads=8, head=128, dtype="bf16",
             cache="e4m3", scales="tensor", block=64),
        # one user's decoding step over a short context
        dict(name="attend, one token", op="attend", batch=1, drafts=1, context=1000, heads=32, kv_heads=8, head=128,
             dtype="bf16", cache="same", scales="none", block=16),
        # the decoding batch of a server, requests of all lengths, cache in 8 bits
        dict(name="attend, decoding batch", op="attend", batch=128, drafts=1, context=8192, heads=32, kv_heads=8, head=128,
             dtype="bf16", cache="e4m3", scales="token", block=16),
        # a few users' trees of drafted tokens over long contexts
        dict(name="attend, small trees", op="attend", batch=6, drafts=13, context=32768, heads=32, kv_heads=8, head=128,
             dtype="fp16", cache="int8", scales="token", block=32),
        # a batch of full trees
        dict(name="attend, full trees", op="attend", batch=16, drafts=61, context=8192, heads=64, kv_heads=8, head=128,
             dtype="bf16", cache="same", scales="none", block=64),
        # trees over heads of 64, shared by all query heads of a rank
        dict(name="attend, narrow heads", op="attend", batch=31, drafts=29, context=4096, heads=12, kv_heads=2, head=64,
             dtype="bf16", cache="e4m3", scales="tensor", block=16),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotary", "write", "read", "attend", "attend"])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    head = rng.choice([64, 128])
    dtype = rng.choice(["bf16", "fp16"])
    cache = rng.choice(["e4m3", "int8", "same"])
    scales = "none" if cache == "same" else rng.choice(["token", "token", "tensor", "head"])
    block = rng.choice([8, 16, 32, 48, 64, 128])
    if op == "rotary":
        return dict(op=op, tokens=_spread(rng, 1, 8191), heads=heads, kv_heads=kv_heads, head=head,
                    part=rng.choice([head, head // 2]), layout=rng.choice(["half", "interleaved"]),
                    dtype=rng.choice([dtype, "fp32"]), reach=_spread(rng, 8192, 200000))
    if op == "write":
        part = rng.choice([0, head // 2, head])
        back = part == 0 or cache == "int8"
        return dict(op=op, tokens=_spread(rng, 1, 8191), heads=heads if part else 0, kv_heads=kv_heads, head=head, part=part,
                    layout=rng.choice(["half", "interleaved"]) if part else "none", dtype=dtype, cache=cache, scales=scales,
                    block=block, reach=_spread(rng, 8192, 200000), back=back)
    if op == "read":
        batch = _spread(rng, 1, 24)
        return dict(op=op, batch=batch, context=_spread(rng, 30, 8192), kv_heads=kv_heads, head=head, dtype=dtype, cache=cache,
                    scales=scales, block=block)
    batch = _spread(rng, 1, 128)
    drafts = rng.choice([1, 1, _spread(rng, 2, 64)])
    most = min(32768, 2000000 // (batch * drafts), 1000000 // batch)
    return dict(op=op, batch=batch, drafts=drafts, context=max(drafts, _spread(rng, 30, max(40, most))), heads=heads,
                kv_heads=kv_heads, head=head, dtype=dtype, cache=cache, scales=scales, block=block)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Each request's length and its drafted tokens: spread over the range, the first at its end."""
    batch, context, drafts = case["batch"], case["context"], case.get("drafts", 0)
    parts = [(i * 0.6180339887) % 1.0 for i in range(batch)]
    lengths = [max(1, context - int(p * 0.875 * context)) for p in parts]
    counts = [max(1, drafts - int(p * 0.5 * drafts)) if drafts > 1 else drafts for p in parts]
    lengths = [max(a, b) for a, b in zip(lengths, counts)]
    return lengths, counts


def _table(reach, part):
    """cos and sin of every position, long contexts scaled by 8 as a linear scaling does; angles in 64 bits."""
    if not part:
        return None
    inv = 10000.0 ** (-torch.arange(0, part, 2, dtype=torch.float64, device="cuda") / part)
    angle = (torch.arange(reach, dtype=torch.float64, device="cuda") / (8.0 if reach > 32768 else 1.0))[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _random(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _fresh_cache(gen, blocks, case):
    """Key and value caches [blocks, block, kv_heads, head] with values in them, and their scales."""
    kind, shape = case["cache"], (blocks, case["block"], case["kv_heads"], case["head"])
    if kind == "same":
        return [_random(gen, shape, DTYPES[case["dtype"]]) for _ in range(2)] + [None, None]
    caches, scales = [], []
    for k in range(2):
        x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * (LARGEST[kind] / 4)
        caches.append(x.clamp_(-LARGEST[kind], LARGEST[kind]).to(CACHES[kind]))
        of = {"token": shape[:3], "head": shape[2:3], "tensor": (1,)}[case["scales"]]
        s = torch.rand(of, generator=gen, device="cuda", dtype=torch.float32) * 0.5 + 0.75
        scales.append(s * (4.0 / LARGEST[kind]))
    return caches + scales


def _tree(gen, counts):
    """One 64-bit word of visible drafted tokens for each drafted token: every token hangs on an earlier one of its request."""
    total, longest = sum(counts), max(counts)
    r = torch.rand(len(counts), longest, generator=gen, device="cuda").cpu().numpy()
    words = np.zeros(total, dtype=np.uint64)
    t = 0
    for b, n in enumerate(counts):
        own_words = []
        for i in range(n):
            up = own_words[int(r[b, i] * i)] if i else 0
            own_words.append(up | (1 << i))
        words[t:t + n] = np.array(own_words, dtype=np.uint64)
        t += n
    return torch.from_numpy(words.view(np.int64)).to("cuda").view(total, 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    op, dev = case["op"], "cuda"
    if op in ("rotary", "write"):
        tokens = case["tokens"]
        s["positions"] = torch.randint(0, case["reach"], (tokens,), generator=gen, device=dev)
        s["table"] = _table(case["reach"], case["part"])
    if op == "rotary":
        dtype, part, head = DTYPES[case["dtype"]], case["part"], case["head"]
        # the rotated part comes last in its head where it is taken in pairs: the call gets a view
        s["query"] = _random(gen, (case["tokens"], case["heads"], head), dtype)
        s["key"] = _random(gen, (case["tokens"], case["kv_heads"], head), dtype)
        if case["layout"] == "interleaved":
            s["query"], s["key"] = s["query"][..., head - part:], s["key"][..., head - part:]
        return s
    if op == "write":
        dtype, head, kv = DTYPES[case["dtype"]], case["head"], case["kv_heads"]
        # the three projections of one matrix product, as views of its result
        packed = _random(gen, (tokens, case["heads"] + 2 * kv, head), dtype)
        s["query"] = packed[:, :case["heads"]]
        s["key"] = packed[:, case["heads"]:case["heads"] + kv]
        s["value"] = packed[:, case["heads"] + kv:]
        blocks = -(-tokens // case["block"]) + 3
        s["key_cache"], s["value_cache"], s["k_scale"], s["v_scale"] = _fresh_cache(gen, blocks, case)
        order = torch.randperm(blocks, generator=gen, device=dev)
        at = torch.arange(tokens, device=dev)
        s["slots"] = order[at // case["block"]] * case["block"] + at % case["block"]
        padded = tokens // 100  # the last tokens of a padded batch have no slot
        if padded and not case["back"]:
            s["slots"][tokens - padded:] = -1
        s["written"] = torch.arange(tokens - (padded if not case["back"] else 0), device=dev)
        if case["back"]:
            s["block_table"] = order.to(torch.int32)[None]
            s["cu_seq_lens"] = torch.tensor([0, tokens], dtype=torch.int32, device=dev)
            s["seq_of"] = torch.zeros(tokens, dtype=torch.int64, device=dev)
            s["key_out"], s["value_out"] = torch.empty_like(s["key"].contiguous()), torch.empty_like(s["key"].contiguous())
        return s
    lengths, counts = _lengths(case)
    needs = [-(-n // case["block"]) for n in lengths]
    width, blocks = max(needs), sum(needs) + 5
    s["key_cache"], s["value_cache"], s["k_scale"], s["v_scale"] = _fresh_cache(gen, blocks, case)
    order = torch.randperm(blocks, generator=gen, device=dev).to(torch.int32)
    need = torch.tensor(needs, device=dev)
    start = torch.cumsum(need, 0) - need
    j = torch.arange(width, device=dev)
    s["block_table"] = torch.where(j[None] < need[:, None], order[(start[:, None] + j[None]).clamp(max=blocks - 1)], 0).contiguous()
    s["longest"] = max(lengths)
    if op == "read":
        total = sum(lengths)
        s["cu_seq_lens"] = torch.tensor([0] + list(np.cumsum(lengths)), dtype=torch.int32, device=dev)
        shape = (total, case["kv_heads"], case["head"])
        s["key_out"], s["value_out"] = (torch.empty(shape, dtype=DTYPES[case["dtype"]], device=dev) for _ in range(2))
        return s
    s["seq_lens"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
    s["cu_query_lens"] = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=dev)
    s["most"] = max(counts)
    s["query"] = _random(gen, (sum(counts), case["heads"], case["head"]), DTYPES[case["dtype"]]) * 1.5
    s["mask"] = _tree(gen, counts) if s["most"] > 1 else None
    s["scale"] = case["head"] ** -0.5
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms
def _rounded(x, dtype):
    """64-bit values rounded once to a type of fewer bits: to 32 bits with the last bit set where that was inexact, which
    lies on no border of the shorter types, then to the nearest."""
    if dtype == torch.float32:
        return x.float()
    r = x.float()
    far = x - r.double()
    even = (r.view(torch.int32) & 1) == 0
    to = torch.where(far > 0, torch.full_like(r, math.inf), torch.full_like(r, -math.inf))
    r = torch.where(even & (far != 0) & torch.isfinite(r), torch.nextafter(r, to), r)
    return r.to(dtype)


def _rotated(x, positions, table, part, layout):
    """x [tokens, heads, head] with its first `part` dimensions turned by its position's angles, in 64 bits."""
    row = table[positions].double()[:, None]
    cos, sin = row[..., :part // 2], row[..., part // 2:]
    x = x.double()
    turn, rest = x[..., :part], x[..., part:]
    if layout == "half":
        a, b = turn[..., :part // 2], turn[..., part // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = turn[..., 0::2], turn[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _put(cache, slots, rows):
    """rows into their slots of a cache [blocks, block, ...]; 8-bit floats as their bytes, which indexing knows."""
    bits = (lambda t: t.view(torch.int8)) if cache.dtype == torch.float8_e4m3fn else (lambda t: t)
    bits(cache).flatten(0, 1).index_copy_(0, slots, bits(rows))


def _store(x, cache, scale, slots, kind, how):
    """Rows x [tokens, kv_heads, head] written to a cache, in its type."""
    if kind == "same":
        _put(cache, slots, x)
        return
    x = x.double()
    if how == "token":
        s = (x.abs().amax(-1).float().double() / LARGEST[kind]).float()
        _put(scale, slots, s)
    else:
        s = scale
    s = s.double()[..., None] if how != "tensor" else s.double()
    q = torch.where(s == 0, torch.zeros_like(x), x / s)
    if kind == "int8":
        _put(cache, slots, q.round().clamp(-127, 127).to(torch.int8))
    else:
        _put(cache, slots, _rounded(q.clamp(-448, 448), torch.float8_e4m3fn))


def _values(cache, scale, table):
    """The pages of a block table [batch, width] as 32-bit values [batch, width * block, kv_heads, head]."""
    x = cache.view(torch.int8)[table].view(cache.dtype) if cache.dtype == torch.float8_e4m3fn else cache[table]
    x = x.float()
    if scale is not None:
        x = x * (scale[table][..., None] if scale.dim() == 3 else scale[:, None] if scale.numel() > 1 else scale)
    return x.flatten(1, 2)


def _read_back(s):
    case = s["case"]
    cu = s["cu_seq_lens"]
    t = torch.arange(s["key_out"].shape[0], device=cu.device)
    b = torch.searchsorted(cu, t, right=True, out_int32=False) - 1
    at = t - cu[b]
    page = s["block_table"][b, at // case["block"]].long()
    for cache, scale, out in ((s["key_cache"], s["k_scale"], s["key_out"]), (s["value_cache"], s["v_scale"], s["value_out"])):
        inside = at % case["block"]
        x = cache.view(torch.int8)[page, inside].view(cache.dtype) if cache.dtype == torch.float8_e4m3fn else cache[page, inside]
        x = x.float()
        if scale is not None:
            x = x * (scale[page, inside][..., None] if scale.dim() == 3 else scale[:, None] if scale.numel() > 1 else scale)
        out.copy_(x)
    return [s["key_out"], s["value_out"]]


def _attend(s):
    case = s["case"]
    heads, kv, head, most = case["heads"], case["kv_heads"], case["head"], s["most"]
    group, cu = heads // kv, s["cu_query_lens"].long()
    count, length = cu[1:] - cu[:-1], s["seq_lens"].long()
    batch, dev = length.shape[0], length.device
    k = _values(s["key_cache"], s["k_scale"], s["block_table"])
    v = _values(s["value_cache"], s["v_scale"], s["block_table"])
    i = torch.arange(most, device=dev)
    token = (cu[:-1, None] + i).clamp(max=s["query"].shape[0] - 1)                       # [batch, most]
    q = s["query"][token].float().view(batch, most, kv, group, head).permute(0, 2, 3, 1, 4).reshape(batch, kv, group * most, head)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)).view(batch, kv, group, most, -1) * s["scale"]
    j = torch.arange(k.shape[1], device=dev)
    draft = j[None] - (length - count)[:, None]                                            # [batch, keys]
    if s["mask"] is None:
        seen = draft[:, None] <= i[None, :, None]
    else:
        bit = (s["mask"][token, 0][..., None] >> draft[:, None].clamp(0, 63)) & 1
        seen = (draft[:, None] < 0) | (bit == 1)
    seen = (seen & (j[None] < length[:, None])[:, None])[:, None, None]                    # [batch, 1, 1, most, keys]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    v = torch.where((j[None] < length[:, None])[..., None, None], v, 0.0)
    o = torch.matmul(p.view(batch, kv, group * most, -1), v.permute(0, 2, 1, 3)).view(batch, kv, group, most, head)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(batch, most, heads, head)
    lse = (top + torch.log(total))[..., 0].permute(0, 3, 1, 2).reshape(batch, most, heads)
    t = torch.arange(s["query"].shape[0], device=dev)
    b = torch.searchsorted(cu, t, right=True) - 1
    return o[b, t - cu[b]].to(s["query"].dtype), lse[b, t - cu[b]]


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "rotary":
        for x in (s["query"], s["key"]):
            part = case["part"]
            x.copy_(_rounded(_rotated(x, s["positions"], s["table"], part, case["layout"]), x.dtype))
        return [s["query"], s["key"]]
    if op == "write":
        key, out = s["key"], []
        if case["part"]:
            query = _rotated(s["query"], s["positions"], s["table"], case["part"], case["layout"])
            s["query"].copy_(_rounded(query, s["query"].dtype))
            key = _rounded(_rotated(key, s["positions"], s["table"], case["part"], case["layout"]), key.dtype)
            out = [s["query"]]
        rows, slots = s["written"], s["slots"][s["written"]]
        _store(key[rows], s["key_cache"], s["k_scale"], slots, case["cache"], case["scales"])
        _store(s["value"][rows], s["value_cache"], s["v_scale"], slots, case["cache"], case["scales"])
        if case["back"]:
            out += _read_back(s)
        else:
            out += [s["key_cache"], s["value_cache"]]
        return out + ([s["k_scale"], s["v_scale"]] if case["scales"] == "token" else [])
    return _read_back(s) if op == "read" else _attend(s)


# ------------------------------------------------------------------------------------------------------------------- run
def run(state):
    if not own:
        return _plain(state)
    from torch_mcpu_b200 import ops

    s, case = state, state["case"]
    op, neox = case["op"], case.get("layout") == "half"
    if op == "rotary":
        ops.rotary_embedding(s["positions"], s["query"], s["key"], s["query"].shape[-1], s["table"], neox)
        return [s["query"], s["key"]]
    if op == "attend":
        return ops.tree_attention(s["query"], s["key_cache"], s["value_cache"], s["block_table"], s["seq_lens"],
                                  s["cu_query_lens"], s["most"], s["scale"], tree_mask=s["mask"], k_scale=s["k_scale"],
                                  v_scale=s["v_scale"], return_lse=True)
    out = []
    if op == "write":
        if case["part"]:
            ops.rotary_reshape_and_cache(s["positions"], s["query"], s["key"], s["value"], s["table"], neox, s["key_cache"],
                                         s["value_cache"], s["slots"], s["k_scale"], s["v_scale"])
            out = [s["query"]]
        else:
            ops.reshape_and_cache(s["key"], s["value"], s["key_cache"], s["value_cache"], s["slots"], s["k_scale"],
                                  s["v_scale"])
        if not case["back"]:
            out += [s["key_cache"], s["value_cache"]]
    if op == "read" or case["back"]:
        ops.gather_cache(s["key_cache"], s["value_cache"], s["block_table"], s["cu_seq_lens"], s["key_out"], s["value_out"],
                         s["k_scale"], s["v_scale"])
        out += [s["key_out"], s["value_out"]]
    return out + ([s["k_scale"], s["v_scale"]] if op == "write" and case["scales"] == "token" else [])


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    op, size = case["op"], {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    held = {"same": size}.get(case.get("cache"), 1)
    per_row = 4 if case.get("scales") == "token" else 0  # a scale for each token and head
    if op == "rotary":
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["part"]
        return {"bytes": 2 * size * values + case["tokens"] * (8 + 4 * case["part"]),
                "flops": 3 * values}
    if op == "write":
        t, kv, head = case["tokens"], case["kv_heads"], case["head"]
        turned = t * case["heads"] * case["part"]
        row = 2 * t * kv
        total = 2 * size * turned + row * (head * size + head * held + per_row) + t * (8 + (8 + 4 * case["part"] if case["part"] else 0))
        if case["back"]:
            total += row * (head * held + per_row + head * size)
        return {"bytes": total, "flops": 3 * (turned + t * kv * case["part"]) + 2 * row * head}
    lengths, counts = _lengths(case)
    if op == "read":
        row = 2 * sum(lengths) * case["kv_heads"]
        return {"bytes": row * (case["head"] * (held + size) + per_row), "flops": row * case["head"]}
    row = 2 * sum(lengths) * case["kv_heads"]
    asked = sum(counts) * case["heads"]
    return {"bytes": row * (case["head"] * held + per_row) + asked * (2 * case["head"] * size + 4),
            "flops": 4 * case["heads"] * case["head"] * sum(n * (a - n) + n for a, n in zip(lengths, counts))}


# ----------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The operators' definitions in 64 bits, one head or request at a time."""
    s = prepare(case, seed)
    op = case["op"]

    def turn(x):
        part = case["part"]
        first, second = (slice(0, part // 2), slice(part // 2, part)) if case["layout"] == "half" else (slice(0, part, 2), slice(1, part, 2))
        cos, sin = (h.double() for h in s["table"][s["positions"]].split(part // 2, 1))
        y = x.double()
        for h in range(x.shape[1]):
            a, b = x[:, h, first].double(), x[:, h, second].double()
            y[:, h, first], y[:, h, second] = a * cos - b * sin, a * sin + b * cos
        return y

    def shorter(x, dtype):  # to the nearest value with so many bits, ties to even
        bits, low = {torch.bfloat16: (8, -133), torch.float16: (11, -24), torch.float8_e4m3fn: (4, -9)}[dtype]
        e = torch.frexp(x)[1].clamp(min=low + bits)
        step = torch.ldexp(torch.ones_like(x), e - bits)
        return torch.round(x / step) * step

    if op == "rotary":
        return [turn(s["query"]), turn(s["key"])]
    if op == "write":
        kind, out, scales = case["cache"], [], []
        key = s["key"].double()
        if case["part"]:
            out = [turn(s["query"])]
            key = shorter(turn(s["key"]), s["key"].dtype)
        held = []
        for x, cache, scale in ((key, s["key_cache"], s["k_scale"]), (s["value"].double(), s["value_cache"], s["v_scale"])):
            x, slots = x[s["written"]], s["slots"][s["written"]]
            now = cache.double().flatten(0, 1)
            if kind == "same":
                now[slots] = x
            else:
                if case["scales"] == "token":
                    fresh = (x.abs().max(-1).values / LARGEST[kind]).float()
                    scale = scale.clone()
                    scale.view(-1, case["kv_heads"])[slots] = fresh
                    by = fresh.double()[..., None]
                else:
                    by = scale.double().view(-1, 1)
                y = x / by
                y = torch.round(y).clamp(-127, 127) if kind == "int8" else shorter(y.clamp(-448, 448), torch.float8_e4m3fn)
                now[slots] = torch.where(by == 0, 0.0, y)
                scales.append(scale)
            held.append(now.view(cache.shape))
        if case["back"]:
            at = s["slots"]
            for k in range(2):
                y = held[k].flatten(0, 1)[at]
                if kind != "same":
                    y = y * {"token": lambda c: c.view(-1, case["kv_heads"])[at][..., None], "head": lambda c: c[:, None],
                             "tensor": lambda c: c}[case["scales"]](scales[k].double())
                out.append(y)
        else:
            out += held
        return out + (scales if case["scales"] == "token" else [])
    block, table = case["block"], s["block_table"].cpu().tolist()
    lengths, counts = _lengths(case)

    def pages(cache, scale, b, n):
        ids = torch.tensor(table[b][:-(-n // block)], device="cuda")
        x = torch.stack([cache[p] for p in ids.tolist()]).double() if cache.dtype == torch.float8_e4m3fn else cache[ids].double()
        if scale is not None:
            x = x * (scale[ids].double()[..., None] if scale.dim() == 3 else scale.double().view(-1, 1))
        return x.flatten(0, 1)[:n]

    if op == "read":
        return [torch.cat([pages(c, f, b, n) for b, n in enumerate(lengths)])
                for c, f in ((s["key_cache"], s["k_scale"]), (s["value_cache"], s["v_scale"]))]
    out, lse, t = [], [], 0
    for b, (n, m) in enumerate(zip(lengths, counts)):
        k, v = (pages(c, f, b, n) for c, f in ((s["key_cache"], s["k_scale"]), (s["value_cache"], s["v_scale"])))
        q = s["query"][t:t + m].double()
        seen = torch.ones(m, n, dtype=torch.bool, device="cuda")
        if s["mask"] is None:
            seen[:, n - m:] = torch.ones(m, m, dtype=torch.bool, device="cuda").tril()
        else:
            words = s["mask"][t:t + m, 0].cpu().tolist()
            seen[:, n - m:] = torch.tensor([[(w >> d) & 1 for d in range(m)] for w in words], dtype=torch.bool, device="cuda")
        group = case["heads"] // case["kv_heads"]
        o, z = [], []
        for h in range(case["heads"]):
            score = (q[:, h] @ k[:, h // group].T) * s["scale"]
            score = score.masked_fill(~seen, -math.inf)
            z.append(torch.logsumexp(score, -1))
            o.append(torch.exp(score - z[-1][:, None]) @ v[:, h // group])
        out.append(torch.stack(o, 1))
        lse.append(torch.stack(z, 1))
        t += m
    return [torch.cat(out), torch.cat(lse)]
