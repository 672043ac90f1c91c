"""Rotary positions, the paged key / value cache, its read-back and tree
attention on the B200 against 64-bit forms (tests/attention_reference.py).

Rotations of 16-bit tensors, cache contents and scales are the correctly
rounded values: compared for equality.  Read-back values carry one fp32 product
before their rounding.  For attention the tolerance per output is derived from
the arithmetic (h: half a step of the output's type, eps / 2):
  h |o|                       the output's rounding
  (hp + 2 es) sum p|v|/sum p  probabilities rounded to the products' type (hp)
                              and the error es of the exponents: (D + 4)
                              2^-24 max(scale sum|qk|) for the fp32 sums, 2^-20
                              for exp2 and its argument's products, n 2^-24
                              for the sum of n probabilities
  2^-25 r sum|v|              fp16 probabilities below the normal range; r is
                              the ratio of the largest to the smallest scale
"""

import math

import pytest
import torch

import attention_reference as ref
from torch_mcpu_b200 import ops

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def table(reach, part, **kw):
    return ops.rotary_cos_sin_cache(reach, part, device="cuda", **kw)


# ------------------------------------------------------------------ rotary
@pytest.mark.parametrize("dtype", HALF + [torch.float32])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("tokens,heads,kv,size,part", [
    (1, 4, 1, 128, 128), (7, 3, 2, 128, 64), (33, 5, 5, 64, 16), (2, 1, 0, 192, 192), (5, 2, 1, 80, 20),
    (300, 9, 3, 64, 64), (3, 2, 1, 512, 512), (4, 2, 1, 16, 2), (2500, 2, 1, 128, 128)])
def test_rotary(dtype, neox, tokens, heads, kv, size, part):
    g = gen(tokens + size + part)
    q, k = randn(g, tokens, heads, size, dtype=dtype), randn(g, tokens, kv, size, dtype=dtype)
    pos = torch.randint(0, 4000, (tokens,), generator=g, device="cuda")
    pos[-1] = 3999
    tab = table(4000, part)
    want = [ref.rotated(x, pos, tab, neox) for x in (q, k)]
    mag = [x.double().abs().amax(-1, keepdim=True) * 2 for x in (q, k)] if kv else None
    ops.rotary_embedding(pos, q, k if kv else None, size, tab, neox)
    for i, x in enumerate((q, k)[: 2 if kv else 1]):
        if dtype == torch.float32:
            # two fp32 roundings of products of at most mag / 2 each
            bound = (mag[i] if mag else 20.0) * 2.0 ** -23
            assert ((x.double() - want[i]).abs() <= bound).all()
        else:
            assert torch.equal(x.double(), ref.nearest(want[i], dtype))


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("form", ["flat", "packed", "tail", "odd offset", "heads first"])
def test_rotary_strides(neox, form):
    g = gen(5)
    tokens, heads, size = 19, 6, 64
    part = 32
    if form == "flat":
        big = randn(g, tokens, heads * size, dtype=torch.bfloat16)
        q = big
    elif form == "packed":
        big = randn(g, tokens, heads + 3, size, dtype=torch.bfloat16)
        q = big[:, 2:2 + heads]
    elif form == "tail":
        big = randn(g, tokens, heads, 96, dtype=torch.bfloat16)
        q = big[..., 32:]
    elif form == "odd offset":
        big = randn(g, tokens * heads * size + 3, dtype=torch.bfloat16)
        q = big[3:].view(tokens, heads, size)
    else:
        big = randn(g, heads, tokens, size, dtype=torch.bfloat16)
        q = big.transpose(0, 1)
    pos = torch.randint(0, 100, (tokens,), generator=g, device="cuda")
    tab = table(100, part)
    want_all = big.clone()
    want = ref.nearest(ref.rotated(q.reshape(tokens, heads, size), pos, tab, neox), torch.bfloat16).to(torch.bfloat16)
    view = {"flat": lambda b: b.view(tokens, heads, size), "packed": lambda b: b[:, 2:2 + heads], "tail": lambda b: b[..., 32:],
            "odd offset": lambda b: b[3:].view(tokens, heads, size), "heads first": lambda b: b.transpose(0, 1)}[form]
    view(want_all).copy_(want)
    ops.rotary_embedding(pos, q, None, size, tab, neox)
    assert torch.equal(big, want_all)  # what lies around it is untouched


def test_rotary_scaled_table_far_positions():
    g = gen(9)
    tab = table(150000, 64, base=500000.0, scaling={"rope_type": "yarn", "factor": 16.0,
                                                    "original_max_position_embeddings": 8192})
    q = randn(g, 50, 4, 64, dtype=torch.bfloat16)
    pos = torch.arange(149950, 150000, device="cuda")
    want = ref.nearest(ref.rotated(q, pos, tab, True), torch.bfloat16)
    ops.rotary_embedding(pos, q, None, 64, tab, True)
    assert torch.equal(q.double(), want)


def test_rotary_position_outside_leaves_the_token_and_sets_the_flag():
    g = gen(11)
    ops.device_error(reset=True)
    for size, part in ((64, 64), (20, 10)):
        q = randn(g, 4, 2, size, dtype=torch.bfloat16)
        before = q.clone()
        pos = torch.tensor([0, -1, 10, 5], device="cuda")
        tab = table(10, part)
        ops.rotary_embedding(pos, q, None, size, tab, True)
        assert torch.equal(q[1:3], before[1:3]) and not torch.equal(q[3], before[3])
        assert ops.device_error(reset=True) == 1
    assert ops.device_error() == 0


# ------------------------------------------------------------------ write and read back
def new_cache(blocks, block, kv, size, kind, dtype, scales, g, layout="NHD"):
    held = dtype if kind == "same" else kind
    shape = (blocks, block, kv, size) if layout == "NHD" else (blocks, kv, block, size)
    caches = [randn(g, *shape).to(held) for _ in range(2)]
    if layout == "HND":
        caches = [c.permute(0, 2, 1, 3) for c in caches]
    if kind == "same":
        return caches + [None, None]
    of = {"token": (blocks, block, kv), "head": (kv,), "tensor": (1,)}[scales]
    return caches + [torch.rand(of, generator=g, device="cuda") * 0.01 + 0.008 for _ in range(2)]


CACHES = [("same", "none"), (torch.float8_e4m3fn, "token"), (torch.float8_e4m3fn, "tensor"), (torch.float8_e4m3fn, "head"),
          (torch.int8, "token"), (torch.int8, "head")]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("kind,scales", CACHES)
@pytest.mark.parametrize("tokens,heads,kv,size,part,block,layout", [
    (1, 4, 1, 128, 128, 16, "NHD"), (37, 6, 3, 64, 32, 8, "HND"), (130, 2, 2, 128, 0, 48, "NHD"), (9, 5, 5, 80, 48, 16, "HND"),
    (3, 2, 1, 512, 64, 1, "NHD"), (1000, 8, 2, 128, 128, 128, "NHD"), (21, 0, 1, 256, 256, 16, "NHD")])
def test_write(dtype, kind, scales, tokens, heads, kv, size, part, block, layout):
    g = gen(tokens + size)
    packed = randn(g, tokens, heads + 2 * kv, size, dtype=dtype) * 3
    q, k, v = packed[:, :heads], packed[:, heads:heads + kv], packed[:, heads + kv:]
    v[0, 0] = 0  # a row of zeros
    if tokens > 5:
        k[2], v[3] = k[2] * 1e-4, v[3] * 100  # rows of other sizes
    blocks = -(-tokens // block) + 2
    kc, vc, ks, vs = new_cache(blocks, block, kv, size, kind, dtype, scales, g, layout)
    slots = torch.randperm(blocks * block, generator=g, device="cuda")[:tokens]
    if tokens > 5:
        slots[4] = -1
    pos = torch.randint(0, 5000, (tokens,), generator=g, device="cuda")
    packed0, caches0 = packed.clone(), [c.clone() for c in (kc, vc)]
    scales0 = [None if s is None else s.clone() for s in (ks, vs)]
    rows = [k.double(), v.double()]
    want_packed = packed0.clone()
    if part:
        tab = table(5000, part)
        rows[0] = ref.nearest(ref.rotated(k, pos, tab, scales != "head"), dtype)
        want_packed[:, :heads] = ref.nearest(ref.rotated(q, pos, tab, scales != "head"), dtype).to(dtype)
        ops.rotary_reshape_and_cache(pos, q if heads else None, k, v, tab, scales != "head", kc, vc, slots, ks, vs)
    else:
        ops.reshape_and_cache(k, v, kc, vc, slots, ks, vs)
    assert torch.equal(packed, want_packed)  # query rotated; key and value as they were
    ok = slots >= 0
    at = (slots[ok] // block, slots[ok] % block)
    for x, c, c0, s, s0 in zip(rows, (kc, vc), caches0, (ks, vs), scales0):
        want = c0.double()
        if kind == "same":
            want[at] = x[ok]
        else:
            if scales == "token":
                held, fresh = ref.quantised(x[ok], kind)
                s0[at] = fresh
            else:
                held, _ = ref.quantised(x[ok], kind, s0[:, None])
            want[at] = held
            assert torch.equal(s, s0)
        assert torch.equal(c.double(), want)


def test_write_is_the_two_calls():
    g = gen(3)
    for kind in (torch.float8_e4m3fn, torch.int8):
        q, k, v = (randn(g, 515, h, 128, dtype=torch.bfloat16) for h in (8, 4, 4))
        pos = torch.randint(0, 30000, (515,), generator=g, device="cuda")
        tab, slots = table(30000, 128), torch.randperm(560, generator=g, device="cuda")[:515]
        a, b = (new_cache(35, 16, 4, 128, kind, torch.bfloat16, "token", gen(1)) for _ in range(2))
        q2, k2 = q.clone(), k.clone()
        ops.rotary_reshape_and_cache(pos, q, k, v, tab, True, a[0], a[1], slots, a[2], a[3])
        ops.rotary_embedding(pos, q2, k2, 128, tab, True)
        ops.reshape_and_cache(k2, v, b[0], b[1], slots, b[2], b[3])
        assert torch.equal(q, q2)
        for x, y in zip(a, b):
            assert torch.equal(x.view(torch.int8), y.view(torch.int8))


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8])
def test_write_rounding_borders(kind):
    """Rows made of values at and beside the borders of the 8-bit type: with scale = max / largest a power of two, the
    quotients are exact and ties go to even; with other scales they lie beside the borders."""
    top = ref.LARGEST[kind]
    if kind == torch.int8:
        borders = torch.arange(-127, 127, dtype=torch.float64) + 0.5
    else:
        codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
        borders = (codes[1:] + codes[:-1]) / 2
        borders = torch.cat([borders, -borders])
    for given in (1.0, 0.0371, 0.017999, 3.3e-5, 7e-20, 1e-36):
        s = torch.tensor([given], dtype=torch.float32)
        x = borders * s.double()
        x16 = x.to(torch.bfloat16)
        x = torch.cat([x16] + [torch.nextafter(x16, torch.tensor(d, dtype=torch.bfloat16)) for d in (math.inf, -math.inf)])
        x = torch.nn.functional.pad(x, (0, -x.numel() % 64)).view(-1, 1, 64).cuda()
        n = x.shape[0]
        kc = torch.zeros(n, 1, 1, 64, device="cuda").to(kind)
        vc = torch.zeros_like(kc)
        slots = torch.arange(n, device="cuda")
        s = s.cuda()
        ops.reshape_and_cache(x, x, kc, vc, slots, s, s)
        want, _ = ref.quantised(x.double(), kind, s)
        assert torch.equal(kc[:, 0].double(), want) and torch.equal(vc[:, 0].double(), want), given
    assert top


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8])
def test_write_special_values(kind):
    x = torch.randn(6, 1, 64).to(torch.bfloat16)
    x[0, 0, 5] = math.inf
    x[1, 0, 6] = math.nan
    x[2, 0, 7] = -3e38
    x[3] = 0
    x[4] = torch.tensor(1e-40).to(torch.bfloat16)  # subnormal: its scale is far below the normal range
    x = x.cuda()
    cache = [torch.zeros(6, 1, 1, 64, device="cuda").to(kind) for _ in range(2)]
    scale = [torch.zeros(6, 1, 1, device="cuda") for _ in range(2)]
    slots = torch.arange(6, device="cuda")
    ops.reshape_and_cache(x, x, *cache, slots, *scale)
    back = (cache[0].double() * scale[0].double()[..., None])[:, 0, 0]
    assert back[0].isnan().all() and back[1].isnan().all()
    want, fresh = ref.quantised(x[2:].double(), kind)
    assert torch.equal(cache[0][2:, 0].double(), want) and torch.equal(scale[0][2:, 0], fresh)
    given = torch.tensor([0.01], device="cuda")
    ops.reshape_and_cache(x, x, *cache, slots, given, given)
    held = cache[1][:, 0, 0].double()
    assert held[0, 5] == ref.LARGEST[kind] and held[2, 7] == -ref.LARGEST[kind]
    assert held[1, 6].isnan() if kind != torch.int8 else held[1, 6] == 0


def test_write_slot_beyond_the_cache_sets_the_flag():
    g = gen(2)
    ops.device_error(reset=True)
    kc, vc, ks, vs = new_cache(2, 16, 1, 64, torch.int8, torch.bfloat16, "token", g)
    before = [t.clone() for t in (kc, vc, ks, vs)]
    k = randn(g, 2, 1, 64, dtype=torch.bfloat16)
    ops.reshape_and_cache(k, k, kc, vc, torch.tensor([32, -5], device="cuda"), ks, vs)
    assert ops.device_error(reset=True) == 1
    assert all(torch.equal(a, b) for a, b in zip(before, (kc, vc, ks, vs)))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("kind,scales", CACHES)
@pytest.mark.parametrize("lens,kv,size,block,starts", [
    ([1], 1, 64, 16, None), ([5, 0, 33, 64, 1], 3, 128, 16, None), ([100, 7], 2, 80, 48, [3, 60]), ([17] * 70, 1, 64, 8, None),
    ([3, 2] * 600, 1, 16, 4, None)])
def test_gather(dtype, kind, scales, lens, kv, size, block, starts):
    g = gen(len(lens))
    starts_ = starts or [0] * len(lens)
    needs = [max(1, -(-(n + s) // block)) for n, s in zip(lens, starts_)]
    blocks = sum(needs) + 1
    kc, vc, ks, vs = new_cache(blocks, block, kv, size, kind, dtype, scales, g)
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    bt = torch.full((len(lens), max(needs) + 2), -7, dtype=torch.int32, device="cuda")  # unused entries are not read
    at = 0
    for b, n in enumerate(needs):
        bt[b, :n] = order[at:at + n]
        at += n
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    total = int(cu[-1])
    outs = [torch.full((total + 3, kv, size), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    ops.device_error(reset=True)
    ops.gather_cache(kc, vc, bt, cu, *outs, ks, vs, seq_starts=None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda"))
    assert ops.device_error() == 0
    half = torch.finfo(dtype).eps / 2
    for c, s, o in zip((kc, vc), (ks, vs), outs):
        v = ref.values_of(c, s)
        want = torch.cat([ref.rows_of(v, bt[b], block, n, starts_[b]) for b, n in enumerate(lens)])
        got = o[:total].double()
        if kind == "same":
            assert torch.equal(got, want)
        else:
            tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0  # half a step of the subnormals
            assert ((got - want).abs() <= (half + 2.0 ** -23) * want.abs() + tiny).all()
        assert (o[total:] == 7).all()  # behind the last sequence


def test_gather_bad_pages_leave_rows_and_set_the_flag():
    g = gen(4)
    kc, vc, _, _ = new_cache(3, 16, 1, 64, "same", torch.bfloat16, "none", g)
    outs = [torch.full((40, 1, 64), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    bt = torch.tensor([[1, 3], [-1, 0]], dtype=torch.int32, device="cuda")
    ops.device_error(reset=True)
    ops.gather_cache(kc, vc, bt, torch.tensor([0, 20, 40], dtype=torch.int32, device="cuda"), *outs)
    assert ops.device_error(reset=True) == 1
    assert torch.equal(outs[0][:16], kc[1]) and (outs[0][16:36] == 7).all() and torch.equal(outs[0][36:], kc[0][:4])


# ------------------------------------------------------------------ attention
def make(seed, lens, counts, heads, kv, size, block, dtype, kind, scales, layout="NHD", spread=1.0):
    g = gen(seed)
    needs = [max(1, -(-n // block)) for n in lens]
    blocks = sum(needs) + 2
    kc, vc, ks, vs = new_cache(blocks, block, kv, size, kind, dtype, scales, g, layout)
    if kind != "same":
        top = ref.LARGEST[kind]
        for c in (kc, vc):
            c.copy_((randn(g, *c.shape) * top / 4).clamp(-top, top).to(kind))
        ks, vs = ks * 0.9 * 448 / top, vs * 0.9 * 448 / top
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    bt = torch.full((len(lens), max(needs)), 1 << 30, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(needs):
        bt[b, :n] = order[at:at + n]
        at += n
    cu = torch.tensor([0] + counts).cumsum(0).to(torch.int32).cuda()
    q = (randn(g, sum(counts), heads, size) * spread).to(dtype)
    return q, kc, vc, ks, vs, bt, torch.tensor(lens, dtype=torch.int32, device="cuda"), cu


def random_tree(seed, counts, words=None):
    """Ancestor words of random trees."""
    import random

    r = random.Random(seed)
    words = words or -(-max(counts) // 64)
    rows = []
    for n in counts:
        mine = []
        for i in range(n):
            up = mine[r.randrange(i)] if i and r.random() < 0.9 else 0
            mine.append(up | 1 << i)
        rows += mine
    out = torch.zeros(len(rows), words, dtype=torch.int64)
    for t, w in enumerate(rows):
        for x in range(words):
            part = (w >> (64 * x)) & (2 ** 64 - 1)
            out[t, x] = part - 2 ** 64 if part >= 2 ** 63 else part
    return out.cuda()


def check(q, kc, vc, ks, vs, bt, lens, cu, scale, mask, got, lse):
    want, wlse, (spread, total_v, reach) = ref.attention(q, ref.values_of(kc, ks), ref.values_of(vc, vs), bt, lens, cu, scale, mask)
    size, n = q.shape[2], int(lens.max())
    half = torch.finfo(q.dtype).eps / 2
    hp = half if ks is None else 2.0 ** -11
    es = (size + 4) * 2.0 ** -24 * reach + 2.0 ** -20 + n * 2.0 ** -24
    tol = half * want.abs() + (hp + 2 * es[..., None]) * spread * (1 + half)
    if ks is not None or q.dtype == torch.float16:
        ratio = 1.0 if vs is None else float(vs.max() / vs.min())
        tol += 2.0 ** -25 * ratio * total_v
    if q.dtype == torch.float16:
        tol += 2.0 ** -25
    err = (got.double() - want).abs()
    worst = (err / tol.clamp(min=1e-300)).max().item() if err.numel() else 0
    assert torch.isfinite(got).all() and (err <= tol).all(), f"error {worst:.2f} of its bound"
    empty = wlse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    lerr = (lse.double() - wlse).abs()[~empty]
    assert (lerr <= (es + 2.0 ** -22 * (1 + wlse.abs()))[~empty]).all()


ATTN = [  # lens, counts, heads, kv, size, block
    ([1], [1], 1, 1, 64, 16),
    ([1000], [1], 32, 8, 128, 16),
    ([17, 1, 64, 65, 300], [1, 1, 1, 1, 1], 8, 8, 128, 16),
    ([40, 33, 700, 5], [5, 33, 1, 5], 4, 2, 64, 48),
    ([129, 200], [13, 7], 14, 2, 128, 8),
    ([350, 64, 63], [64, 64, 3], 8, 1, 128, 64),
    ([300, 0, 9, 0], [2, 0, 9, 1], 6, 3, 64, 1),
    ([90], [70], 3, 1, 128, 128),
    ([2500, 130], [2, 4], 16, 1, 64, 16),
]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("kind,scales", CACHES)
@pytest.mark.parametrize("lens,counts,heads,kv,size,block", ATTN)
def test_attention(dtype, kind, scales, lens, counts, heads, kv, size, block):
    ops.device_error(reset=True)
    lens = [max(a, b) if a else 0 for a, b in zip(lens, counts)]
    counts = [c if n else 0 for c, n in zip(counts, lens)]
    x = make(7, lens, counts, heads, kv, size, block, dtype, kind, scales, "HND" if block == 16 else "NHD", 1.5)
    q, kc, vc, ks, vs, bt, sl, cu = x
    for mask in (None, random_tree(3, counts)) if max(counts) > 1 else (None,):
        got, lse = ops.tree_attention(q, kc, vc, bt, sl, cu, max(counts), size ** -0.5, tree_mask=mask, k_scale=ks, v_scale=vs, return_lse=True)
        check(*x, size ** -0.5, mask, got, lse)
    assert ops.device_error() == 0


def test_attention_rows_without_keys_and_wide_masks():
    counts = [3, 130]
    x = make(1, [3, 150], counts, 4, 2, 64, 16, torch.bfloat16, "same", "none")
    q, kc, vc, ks, vs, bt, sl, cu = x
    mask = random_tree(5, counts, words=4)
    mask[:3] = 0  # no context and nothing seen
    mask[1, 0] = 4
    got, lse = ops.tree_attention(q, kc, vc, bt, sl, cu, 130, 0.125, tree_mask=mask, return_lse=True)
    check(*x, 0.125, mask, got, lse)
    assert (got[0] == 0).all() and (got[2] == 0).all() and (lse[0] == -math.inf).all()


def test_attention_sharp_scores_and_negative_scale():
    for scale, spread in ((1.0, 8.0), (-0.3, 2.0), (0.0, 1.0)):
        x = make(2, [333, 70], [4, 1], 8, 4, 128, 16, torch.float16, torch.float8_e4m3fn, "token", spread=spread)
        q, kc, vc, ks, vs, bt, sl, cu = x
        got, lse = ops.tree_attention(q, kc, vc, bt, sl, cu, 4, scale, k_scale=ks, v_scale=vs, return_lse=True)
        check(*x, scale, None, got, lse)


def test_attention_scales_far_apart():
    """Value scales over nine orders of magnitude, growing along the keys."""
    x = make(2, [700], [2], 4, 1, 64, 16, torch.bfloat16, torch.int8, "token")
    q, kc, vc, ks, vs, bt, sl, cu = x
    at = torch.arange(700, device="cuda")
    vs[bt[0, at // 16].long(), at % 16, 0] = 10.0 ** (at / 80 - 6)
    got, lse = ops.tree_attention(q, kc, vc, bt, sl, cu, 2, 0.125, k_scale=ks, v_scale=vs, return_lse=True)
    check(*x, 0.125, None, got, lse)


@pytest.mark.parametrize("kind,scales", [("same", "none"), (torch.float8_e4m3fn, "token"), (torch.int8, "token"),
                                         (torch.float8_e4m3fn, "tensor")])
@pytest.mark.parametrize("heads,counts", [(2, [6, 3]), (16, [6, 3]), (8, [40, 3])])
def test_attention_garbage_where_nothing_is_seen(kind, scales, heads, counts):
    """NaN and infinities behind the sequences, and in drafted tokens that some of the others do not see."""
    x = make(4, [150, 21], counts, heads, 1, 64, 16, torch.bfloat16, kind, scales)
    q, kc, vc, ks, vs, bt, sl, cu = x
    mask = random_tree(8, counts)
    clean, _ = ops.tree_attention(q, kc, vc, bt, sl, cu, max(counts), 0.125, tree_mask=mask, k_scale=ks, v_scale=vs, return_lse=True)
    seen_by = ((mask[:counts[0], 0] >> 1) & 1).bool()  # who sees draft 1 of request 0
    assert seen_by.any() and not seen_by.all()

    def place(pos):
        return int(bt[0, pos // 16]), pos % 16

    def poison(p, s):
        if kind == torch.int8 or scales == "token":
            ks[p, s], vs[p, s] = math.nan, math.inf
        if kind != torch.int8:
            kc[p, s, 0, 3], vc[p, s, 0, 3] = math.nan, math.nan
            if kind == "same":
                vc[p, s, 0, 4] = math.inf

    for pos in range(150, 160):  # the rest of the last page
        poison(*place(pos))
    poison(*place(150 - counts[0] + 1))
    got, lse = ops.tree_attention(q, kc, vc, bt, sl, cu, max(counts), 0.125, tree_mask=mask, k_scale=ks, v_scale=vs, return_lse=True)
    rows = torch.cat([~seen_by, torch.ones(counts[1], dtype=torch.bool, device="cuda")])
    assert torch.equal(got[rows], clean[rows])
    assert got[: counts[0]][seen_by].isnan().any(-1).all() and lse[: counts[0]][seen_by].isnan().all()


def test_attention_values_of_drafts_not_finite_reach_only_their_rows():
    """Keys finite, one value infinite: the rows that see it get infinity in that dimension alone."""
    for heads, counts in ((2, [6]), (16, [12])):
        x = make(4, [90], counts, heads, 1, 64, 16, torch.float16, "same", "none")
        q, kc, vc, ks, vs, bt, sl, cu = x
        mask = random_tree(8, counts)
        clean = ops.tree_attention(q, kc, vc, bt, sl, cu, counts[0], 0.125, tree_mask=mask)
        pos = 90 - counts[0] + 1
        vc[int(bt[0, pos // 16]), pos % 16, 0, 7] = -math.inf
        got = ops.tree_attention(q, kc, vc, bt, sl, cu, counts[0], 0.125, tree_mask=mask)
        seen_by = ((mask[:, 0] >> 1) & 1).bool()
        want = clean.clone()
        want[..., 7][seen_by] = -math.inf
        assert torch.equal(got[~seen_by], want[~seen_by])
        assert torch.equal(got[seen_by].isinf(), want[seen_by].isinf()) and not got.isnan().any()


def test_attention_out_strides_padding_and_rows_outside():
    x = make(6, [50, 20], [3, 2], 4, 2, 64, 16, torch.bfloat16, "same", "none")
    q, kc, vc, ks, vs, bt, sl, cu = x
    padded = torch.zeros(9, 7, 64, dtype=q.dtype, device="cuda")[:, 1:5]
    padded[:5] = q
    buffer = torch.full((9, 4, 96), 7.0, dtype=q.dtype, device="cuda")
    got = ops.tree_attention(padded, kc, vc, bt, sl, cu, 4, 0.125, out=buffer[..., 16:80])
    want = ops.tree_attention(q, kc, vc, bt, sl, cu, 3, 0.125)
    assert torch.equal(got[:5], want) and got.data_ptr() == buffer[..., 16:].data_ptr()
    assert (buffer[5:] == 7).all() and (buffer[..., :16] == 7).all() and (buffer[..., 80:] == 7).all()


def test_attention_requests_that_do_not_fit():
    x = make(6, [50, 20, 30], [3, 2, 1], 4, 2, 64, 16, torch.bfloat16, "same", "none")
    q, kc, vc, ks, vs, bt, sl, cu = x
    want = ops.tree_attention(q, kc, vc, bt, sl, cu, 3, 0.125)
    ops.device_error(reset=True)
    for bad in (1, 20 * 16 + 1, -4):
        lens = sl.clone()
        lens[1] = bad  # shorter than its new tokens, beyond the table, negative
        got = ops.tree_attention(q, kc, vc, bt, lens, cu, 3, 0.125)
        assert ops.device_error(reset=True) == 1
        assert torch.equal(got[:3], want[:3]) and (got[3:5] == 0).all() and torch.equal(got[5:], want[5:])
    table_ = bt.clone()
    table_[1, 0] = -1
    got = ops.tree_attention(q, kc, vc, table_, sl, cu, 3, 0.125)
    assert ops.device_error(reset=True) == 1
    assert torch.equal(got[:3], want[:3]) and torch.equal(got[5:], want[5:])


def test_attention_many_requests():
    lens = [1 + (i * 37) % 90 for i in range(300)]
    x = make(6, lens, [1] * 300, 2, 1, 64, 16, torch.bfloat16, torch.int8, "token")
    q, kc, vc, ks, vs, bt, sl, cu = x
    got, lse = ops.tree_attention(q, kc, vc, bt, sl, cu, 1, 0.125, k_scale=ks, v_scale=vs, return_lse=True)
    check(*x, 0.125, None, got, lse)


def test_attention_repeats_bit_for_bit():
    x = make(6, [9000, 20, 3000], [7, 2, 1], 8, 2, 128, 16, torch.bfloat16, torch.float8_e4m3fn, "token")
    q, kc, vc, ks, vs, bt, sl, cu = x
    first = ops.tree_attention(q, kc, vc, bt, sl, cu, 7, 0.1, k_scale=ks, v_scale=vs)
    for _ in range(5):
        assert torch.equal(first, ops.tree_attention(q, kc, vc, bt, sl, cu, 7, 0.1, k_scale=ks, v_scale=vs))


# ------------------------------------------------------------------ together
def step(q, k, v, pos, tab, kc, vc, ks, vs, slots, bt, sl, cu, most, mask):
    ops.rotary_reshape_and_cache(pos, q, k, v, tab, True, kc, vc, slots, ks, vs)
    return ops.tree_attention(q, kc, vc, bt, sl, cu, most, 128 ** -0.5, tree_mask=mask, k_scale=ks, v_scale=vs)


@pytest.mark.parametrize("kind", ["same", torch.float8_e4m3fn, torch.int8])
def test_a_serving_step_eager_and_captured(kind):
    """Prefix written and read back, then a drafted tree: rotated, written, attended; the same from a replayed graph with
    new inputs and lengths."""
    g = gen(20)
    dtype, heads, kv, block, blocks = torch.bfloat16, 8, 2, 16, 64
    tab = table(1000, 128)
    kc, vc, ks, vs = new_cache(blocks, block, kv, 128, kind, dtype, "token", g)
    bt = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)[:40].view(2, 20)
    ctx, counts = [100, 250], [5, 9]

    def slots_of(b, pos):
        return bt[b, pos // block].long() * block + pos % block

    prefix = [randn(g, n, kv, 128, dtype=dtype) for n in ctx for _ in range(2)]
    for b, n in enumerate(ctx):
        pos = torch.arange(n, device="cuda")
        ops.rotary_reshape_and_cache(pos, None, prefix[2 * b], prefix[2 * b + 1], tab, True, kc, vc, slots_of(b, pos), ks, vs)
    back = [torch.empty(sum(ctx), kv, 128, dtype=dtype, device="cuda") for _ in range(2)]
    cu_ctx = torch.tensor([0, 100, 350], dtype=torch.int32, device="cuda")
    ops.gather_cache(kc, vc, bt, cu_ctx, *back, ks, vs)
    step_size = {"same": 0.0, torch.float8_e4m3fn: 2.0 ** -4, torch.int8: 0.5 / 127}[kind]
    top = prefix[1].abs().max()
    assert ((back[1][:100].double() - prefix[1].double()).abs() <= (step_size + 2.0 ** -8 * (kind != "same")) * top).all()

    pos = torch.cat([ctx[b] + torch.arange(n, device="cuda") for b, n in enumerate(counts)])
    slots = torch.cat([slots_of(b, ctx[b] + torch.arange(n, device="cuda")) for b, n in enumerate(counts)])
    sl = torch.tensor([105, 259], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 5, 14], dtype=torch.int32, device="cuda")
    mask = random_tree(2, counts)
    q, k, v = randn(g, 14, heads, 128, dtype=dtype), randn(g, 14, kv, 128, dtype=dtype), randn(g, 14, kv, 128, dtype=dtype)
    q0 = q.clone()
    eager = step(q, k, v, pos, tab, kc, vc, ks, vs, slots, bt, sl, cu, 9, mask)
    lse_ok = ops.tree_attention(q, kc, vc, bt, sl, cu, 9, 128 ** -0.5, tree_mask=mask, k_scale=ks, v_scale=vs, return_lse=True)
    check(q, kc, vc, ks, vs, bt, sl, cu, 128 ** -0.5, mask, *lse_ok)
    assert torch.equal(lse_ok[0], eager)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    q.copy_(q0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = step(q, k, v, pos, tab, kc, vc, ks, vs, slots, bt, sl, cu, 9, mask)
    q.copy_(q0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, eager)
    # other lengths and values through the same graph
    sl.copy_(torch.tensor([60, 40], dtype=torch.int32))
    q.copy_(q0)
    graph.replay()
    torch.cuda.synchronize()
    q.copy_(q0)
    assert torch.equal(captured, step(q, k, v, pos, tab, kc, vc, ks, vs, slots, bt, sl, cu, 9, mask))


def test_two_graphs_and_a_stream_at_once():
    """Calls that run at the same time keep apart: each has a workspace of its own."""
    xs = [make(s, [4000, 700], [3, 1], 8, 2, 128, 16, torch.bfloat16, "same", "none") for s in (1, 2, 3)]

    def call(x):
        q, kc, vc, ks, vs, bt, sl, cu = x
        return ops.tree_attention(q, kc, vc, bt, sl, cu, 3, 0.1)

    want = [call(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    graphs, outs = [], []
    for x, s in zip(xs[:2], streams):
        g_ = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g_, stream=s):
            outs.append(call(x))
        graphs.append(g_)
    for _ in range(20):
        for g_, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g_.replay()
        with torch.cuda.stream(streams[2]):
            third = call(xs[2])
        torch.cuda.synchronize()
        for a, b in zip(want, outs + [third]):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ borders between the kernels, long caches, refusals
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("kind,scales", [("same", "none"), (torch.float8_e4m3fn, "token"), (torch.int8, "head")])
@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("most", [7, 8, 9, 15, 16, 17, 128, 129])
def test_attention_at_the_row_borders(dtype, kind, scales, size, most):
    """The largest request fills a kernel's rows, or is one row short of them or beyond; trees and chains."""
    counts = [most, 1, max(1, most - 1)]
    x = make(12, [most + 200, 77, most + 3], counts, 2, 2, size, 32, dtype, kind, scales)
    q, kc, vc, ks, vs, bt, sl, cu = x
    for mask in (None, random_tree(5, counts)):
        got, lse = ops.tree_attention(q, kc, vc, bt, sl, cu, most, size ** -0.5, tree_mask=mask, k_scale=ks, v_scale=vs, return_lse=True)
        check(*x, size ** -0.5, mask, got, lse)


@pytest.mark.parametrize("kind,scales", [("same", "none"), (torch.float8_e4m3fn, "token"), (torch.int8, "token"),
                                         (torch.float8_e4m3fn, "tensor")])
def test_attention_garbage_with_few_rows(kind, scales):
    """NaN and infinities where nothing is seen, up to 8 rows a key / value head."""
    test_attention_garbage_where_nothing_is_seen(kind, scales, 1, [6, 3])


@pytest.mark.parametrize("dtype", HALF)
def test_attention_infinite_value_of_a_draft_with_few_rows(dtype):
    for heads, counts, sign in ((1, [6], -1), (2, [4], 1)):
        x = make(4, [90], counts, heads, 1, 128, 16, dtype, "same", "none")
        q, kc, vc, ks, vs, bt, sl, cu = x
        mask = torch.tensor([[1], [3], [1], [9], [19], [41]][: counts[0]], device="cuda")  # [3]: draft 1
        clean = ops.tree_attention(q, kc, vc, bt, sl, cu, counts[0], 0.125, tree_mask=mask)
        pos = 90 - counts[0] + 1
        vc[int(bt[0, pos // 16]), pos % 16, 0, 77] = sign * math.inf
        got = ops.tree_attention(q, kc, vc, bt, sl, cu, counts[0], 0.125, tree_mask=mask)
        seen_by = ((mask[:, 0] >> 1) & 1).bool()
        assert seen_by.any() and not seen_by.all()
        want = clean.clone()
        want[..., 77][seen_by] = sign * math.inf
        assert torch.equal(got, want)


def test_attention_more_tokens_than_announced():
    """A request with more than max_query_len tokens gives zeros and the flag; the others are served."""
    for most, counts in ((1, [1, 3, 1]), (2, [2, 5, 1]), (40, [40, 41, 3])):
        x = make(6, [80, 90, 70], counts, 4, 2, 64, 16, torch.bfloat16, "same", "none")
        q, kc, vc, ks, vs, bt, sl, cu = x
        ops.device_error(reset=True)
        got, lse = ops.tree_attention(q, kc, vc, bt, sl, cu, most, 0.125, return_lse=True)
        assert ops.device_error(reset=True) == 1
        a, b = counts[0], counts[0] + counts[1]
        assert (got[a:b] == 0).all() and (lse[a:b] == -math.inf).all()
        served = [0, 2]
        cu2 = torch.tensor([0, a, a + counts[2]], dtype=torch.int32, device="cuda")
        rest = [torch.cat([t[:a], t[b:]]) for t in (q, got, lse)]
        check(rest[0], kc, vc, ks, vs, bt[served], sl[served], cu2, 0.125, None, rest[1], rest[2])


def test_caches_beyond_32_bit_offsets():
    """Pages past 2^32 elements: written, read back and attended as in a small cache."""
    blocks, block, kv, size = 263000, 16, 8, 128  # 4.3e9 values each
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    g = gen(3)
    big = [torch.zeros(blocks, block, kv, size, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2)]
    small = [torch.zeros(8, block, kv, size, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2)]
    far = torch.tensor([[blocks - 1, 3, blocks - 2, 262200, 262145, 0]], dtype=torch.int32, device="cuda")
    near = torch.tensor([[7, 3, 2, 4, 5, 0]], dtype=torch.int32, device="cuda")
    n = 6 * block - 5
    k, v = (randn(g, n, kv, size, dtype=torch.bfloat16) for _ in range(2))
    at = torch.arange(n, device="cuda")
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    results = []
    for (kc, vc), table_ in ((big, far), (small, near)):
        ks, vs = (torch.zeros(kc.shape[:3], device="cuda") for _ in range(2))
        slots = table_[0, at // block].long() * block + at % block
        ops.reshape_and_cache(k, v, kc, vc, slots, ks, vs)
        out = [torch.empty_like(k) for _ in range(2)]
        ops.gather_cache(kc, vc, table_, cu, out[0], out[1], ks, vs)
        for tokens, heads in ((1, 32), (4, 32), (20, 64)):
            q = randn(gen(tokens), tokens, heads, size, dtype=torch.bfloat16)
            out.append(ops.tree_attention(q, kc, vc, table_, cu[1:], torch.tensor([0, tokens], dtype=torch.int32, device="cuda"),
                                          tokens, size ** -0.5, k_scale=ks, v_scale=vs))
        results.append(out)
        del ks, vs
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert results[0][2].abs().max() > 0


def test_written_tensors_must_not_be_one():
    g = gen(1)
    k, v = (randn(g, 3, 2, 64, dtype=torch.float16) for _ in range(2))
    kc, vc, ks, vs = new_cache(4, 16, 2, 64, torch.int8, torch.float16, "token", g)
    slots = torch.arange(3, device="cuda")
    with pytest.raises(RuntimeError, match="key_cache and value_cache are written"):
        ops.reshape_and_cache(k, v, kc, kc, slots, ks, vs)
    with pytest.raises(RuntimeError, match="k_scale and v_scale are written"):
        ops.reshape_and_cache(k, v, kc, vc, slots, ks, ks)
    with pytest.raises(RuntimeError, match="query and key are written"):
        ops.rotary_embedding(slots, k, k, 64, table(8, 64), True)
    bt = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="key_out and value_out are written"):
        ops.gather_cache(kc, vc, bt, cu, k, k, ks, vs)


def test_tensors_that_require_a_gradient_are_refused():
    x = make(6, [50], [2], 4, 2, 64, 16, torch.bfloat16, "same", "none")
    q, kc, vc, ks, vs, bt, sl, cu = x
    want = ops.tree_attention(q, kc, vc, bt, sl, cu, 2, 0.125)
    k = torch.zeros(2, 2, 64, dtype=q.dtype, device="cuda", requires_grad=True)
    pos = torch.arange(2, device="cuda")
    q.requires_grad_()
    calls = [lambda: ops.tree_attention(q, kc, vc, bt, sl, cu, 2, 0.125),
             lambda: ops.rotary_embedding(pos, q, None, 64, table(8, 64), True),
             lambda: ops.reshape_and_cache(k, k.detach(), kc, vc, pos),
             lambda: ops.rotary_reshape_and_cache(pos, q, k.detach(), k.detach(), table(8, 64), True, kc, vc, pos)]
    for call in calls:
        with pytest.raises(RuntimeError, match="requires a gradient"):
            call()
    with torch.no_grad():
        assert torch.equal(calls[0](), want)


def test_first_calls_inside_a_capture():
    """A process whose first calls are captured: nothing has been loaded or configured before."""
    import os
    import subprocess
    import sys

    code = """
import torch
from torch_mcpu_b200 import ops
for n in (1, 3, 40):  # a kernel each
    q = torch.randn(n, 16, 128, device="cuda").half()
    k = torch.randn(n, 4, 128, device="cuda").half()
    kc, vc = (torch.randn(8, 16, 4, 128, device="cuda").to(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.rand(8, 16, 4, device="cuda") + 0.5 for _ in range(2))
    bt = torch.arange(8, dtype=torch.int32, device="cuda")[None]
    sl, cu, cs = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([100], [0, n], [0, 100]))
    table = ops.rotary_cos_sin_cache(128, 128, device="cuda")
    pos = torch.arange(n, device="cuda")
    back = [torch.empty(100, 4, 128, device="cuda").half() for _ in range(2)]
    q0 = q.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rotary_reshape_and_cache(pos, q, k, k, table, True, kc, vc, pos, ks, vs)
        o = ops.tree_attention(q, kc, vc, bt, sl, cu, n, 0.1, k_scale=ks, v_scale=vs)
        ops.gather_cache(kc, vc, bt, cs, back[0], back[1], ks, vs)
    graph.replay()
    torch.cuda.synchronize()
    got = [o.clone(), back[0].clone(), back[1].clone(), q.clone()]
    ops.rotary_reshape_and_cache(pos, q0, k, k, table, True, kc, vc, pos, ks, vs)
    o = ops.tree_attention(q0, kc, vc, bt, sl, cu, n, 0.1, k_scale=ks, v_scale=vs)
    ops.gather_cache(kc, vc, bt, cs, back[0], back[1], ks, vs)
    assert all(torch.equal(a, b) for a, b in zip(got, [o, *back, q0])) and ops.device_error() == 0
print("same")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "same", done.stderr[-2000:]
