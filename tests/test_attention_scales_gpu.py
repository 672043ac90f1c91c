"""Tree attention over 8-bit caches whose value scales lie far apart, and over
probabilities far apart, against 64 bits.

Products p_j s_j (probability times value scale) are rounded to fp16 relative
to a reference of each row that follows the largest of them: the largest lies
at 2^7 or above when the sums are complete, so that what falls below the
normal range of fp16 is off by at most 2^-25 / 2^7 of it.  The tolerance of
an output (h: half a step of its type, eps / 2):
  h |o|                         the output's rounding
  (2^-11 + 2 es) sum p|v| / P   products rounded to fp16, and the error es of
                                the exponents: (D + 4) 2^-24 max(scale sum|qk|)
                                for the fp32 sums, 2^-20 for exp2 and its
                                argument's products, n 2^-24 for the sum P of n
                                probabilities
  2^-32 max(p s) sum|q| / P     products below the normal range of fp16, q the
                                values as they are held
  2^-25                         an fp16 output's subnormal step
"""

import math

import pytest
import torch

import attention_reference as ref
from test_attention_gpu import gen, make, random_tree
from torch_mcpu_b200 import ops

pytestmark = pytest.mark.gpu

FLOOR = 2.0 ** -32


def expected(q, kc, vc, ks, vs, bt, lens, cu, scale, mask, floor, hp=2.0 ** -11):
    """(out, lse, tolerance of out, es) per token and head, in 64 bits.  A token that sees nothing: zeros and -inf."""
    T, H, D = q.shape
    block, kv = kc.shape[1], kc.shape[2]
    half = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(T, H, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64, device=q.device)
    es_all = torch.zeros_like(lse)
    cu, lens = cu.tolist(), lens.tolist()
    for b, n in enumerate(lens):
        t0, m = cu[b], cu[b + 1] - cu[b]
        if n == 0 or m == 0:
            continue
        at = torch.arange(n, device=q.device)
        page, place = bt[b, at // block].long(), at % block
        held = vc.double()[page, place] if vc.dtype != torch.float8_e4m3fn else vc.view(torch.int8)[page, place].view(vc.dtype).double()
        k = kc.double()[page, place] if kc.dtype != torch.float8_e4m3fn else kc.view(torch.int8)[page, place].view(kc.dtype).double()
        one = torch.ones(n, kv, dtype=torch.float64, device=q.device)
        sk, sv = ((one if s is None else s.double()[page, place] if s.dim() == 3 else one * s.double()) for s in (ks, vs))
        k = k * sk[..., None]
        x = q[t0:t0 + m].double().view(m, kv, H // kv, D)
        score = torch.einsum("mkgd,nkd->kgmn", x, k) * scale
        reach = torch.einsum("mkgd,nkd->kgmn", x.abs(), k.abs()) * abs(scale)
        i, d = torch.arange(m, device=q.device), at - (n - m)
        if mask is None:
            seen = d[None] <= i[:, None]
        else:
            words = mask[t0:t0 + m][:, (d.clamp(min=0) // 64)]
            seen = (d < 0)[None] | (((words >> (d.clamp(min=0) % 64)) & 1) == 1)
        score = score.masked_fill(~seen, -math.inf)
        top = score.amax(-1, keepdim=True)
        p = torch.where(seen, torch.exp(score - top.clamp(min=-1e300)), 0.0)
        total = p.sum(-1, keepdim=True)
        safe = total.clamp(min=1e-300)
        w = p * sv.T[:, None, None]
        w = torch.where(seen, w, 0.0)
        o = torch.einsum("kgmn,nkd->kgmd", w, held) / safe
        spread = torch.einsum("kgmn,nkd->kgmd", w, held.abs()) / safe
        held_sum = torch.einsum("mn,nkd->kmd", seen.double(), held.abs())[:, None]
        es = (D + 4) * 2.0 ** -24 * torch.where(seen, reach, 0.0).amax(-1, keepdim=True) + 2.0 ** -20 + n * 2.0 ** -24
        bound = half * o.abs() + (hp + 2 * es) * spread * (1 + half) + floor * w.amax(-1, keepdim=True) * held_sum / safe
        if q.dtype == torch.float16:
            bound = bound + 2.0 ** -25
        for to, x in ((out, o), (tol, bound)):
            to[t0:t0 + m] = x.permute(2, 0, 1, 3).reshape(m, H, D)
        lse[t0:t0 + m] = (top + torch.log(total))[..., 0].permute(2, 0, 1).reshape(m, H)
        es_all[t0:t0 + m] = es[..., 0].permute(2, 0, 1).reshape(m, H)
    return out, lse, tol, es_all


def check(x, scale, mask, got, lse, floor=FLOOR, hp=2.0 ** -11):
    want, wlse, tol, es = expected(*x, scale, mask, floor, hp)
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    worst = (err / tol.clamp(min=1e-300)).max().item()
    assert (err <= tol).all(), f"error {worst:.3g} of its bound"
    empty = wlse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert ((lse.double() - wlse).abs()[~empty] <= (es + 2.0 ** -22 * (1 + wlse.abs()))[~empty]).all()
    # the bound is one that zeros, or half of the output, do not meet
    if not empty.all():
        assert ((0.5 * want).abs() > tol)[~empty].any()


# requests, tokens of each, query heads: up to 8 rows, up to 16, one row tile of 128 and two; the many requests give a block
# several key tiles of a row tile, the few ones split a row tile over blocks
SHAPES = {"8 rows": ([700, 333], [2, 1], 8), "8 rows, many": ([700] * 60, [1] * 60, 32), "16 rows": ([700, 150], [4, 1], 8),
          "16 rows, many": ([900] * 60, [2] * 60, 32), "one tile": ([700, 50, 300], [13, 1, 20], 8),
          "one tile, many": ([900] * 40, [10] * 40, 16), "two tiles": ([700, 200], [60, 3], 8),
          "two tiles, many": ([600] * 20, [40] * 20, 16)}


def place_of(x, b, pos):
    bt, block = x[5], x[1].shape[1]
    return bt[b, pos // block].long(), pos % block


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("order", ["growing", "falling", "random", "faint", "faint late", "unseen", "zeros first", "one huge"])
def test_value_scales(kind, shape, order):
    lens, counts, heads = SHAPES[shape]
    size = 64 if "two" in shape or shape == "16 rows" else 128
    kv = 4 if "many" in shape else 2
    dtype = torch.float16 if order in ("random", "zeros first") else torch.bfloat16
    x = make(11, lens, counts, heads, kv, size, 16, dtype, kind, "token")
    q, kc, vc, ks, vs, bt, sl, cu = x
    top = ref.LARGEST[kind]
    g = gen(3)
    mask = random_tree(7, counts) if max(counts) > 1 else None
    wide = dtype == torch.float16  # outputs of fp16 stay in its range
    q[..., 0] = 4.0
    for b, n in enumerate(lens):
        at = torch.arange(n, device="cuda")
        page, slot = place_of(x, b, at)
        if order == "growing":
            vs[page, slot] = (10.0 ** (at / (n / 9) - 6))[:, None]
        elif order == "falling":
            vs[page, slot] = (10.0 ** (3 - at / (n / 9)))[:, None]
        elif order == "random":
            vs[page, slot] = 10.0 ** (torch.rand(n, kv, generator=g, device="cuda") * (7 if wide else 9) - 6)
        elif order in ("faint", "faint late"):
            # one key with a huge value and next to no probability: its score is 120 below the others'
            j = 3 if order == "faint" else n - counts[b] - 2
            p, s = int(page[j]), int(slot[j])
            kc[p, s] = torch.zeros(kv, size, device="cuda").to(kind)
            kc[p, s, :, 0] = torch.tensor(-top, device="cuda").to(kind)
            ks[p, s] = 240.0 / top
            vs[p, s] = 1e9
        elif order == "unseen" and counts[b] > 1:
            j = n - counts[b] + 1
            vs[int(page[j]), int(slot[j])] = 1e20
        elif order == "zeros first":
            early = at < n // 2
            vs[page[early], slot[early]] = 0.0
        elif order == "one huge":
            vs[int(page[n // 3]), int(slot[n // 3])] = 1e5 if wide else 1e7
    ops.device_error(reset=True)
    got, lse = ops.tree_attention(q, kc, vc, bt, sl, cu, max(counts), 0.125, tree_mask=mask, k_scale=ks, v_scale=vs, return_lse=True)
    check(x, 0.125, mask, got, lse)
    assert ops.device_error() == 0


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("counts,heads", [([6, 3], 1), ([6, 3], 2), ([40, 3], 8), ([40, 3], 1)])
def test_scale_of_a_draft_matters_to_its_rows_alone(kind, counts, heads):
    """A draft that a row does not see changes no bit of that row, whatever its value scale."""
    x = make(4, [150, 21], counts, heads, 1, 64, 16, torch.bfloat16, kind, "token")
    q, kc, vc, ks, vs, bt, sl, cu = x
    mask = random_tree(8, counts)
    seen_by = ((mask[:, 0] >> 1) & 1).bool()
    seen_by[counts[0]:] = False
    assert seen_by.any() and not seen_by[:counts[0]].all()
    results = []
    for huge in (1.0, 1e3, 1e12, 1e29, 3e38):
        vs[place_of(x, 0, 150 - counts[0] + 1)] = huge
        results.append(ops.tree_attention(q, kc, vc, bt, sl, cu, max(counts), 0.125, tree_mask=mask, k_scale=ks, v_scale=vs))
    for r in results[1:]:
        assert torch.equal(r[~seen_by], results[0][~seen_by])


@pytest.mark.parametrize("kind,scales", [("same", "none"), (torch.float8_e4m3fn, "tensor"), (torch.int8, "head"), (torch.int8, "token")])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_many_faint_probabilities(kind, scales, shape):
    """One key takes next to all of the probability and has values of 0; the others, 2^-26 each, make the output: their
    products count although they lie below the normal range of fp16 beside the largest."""
    lens, counts, heads = SHAPES[shape]
    size, kv = 64, 4 if "many" in shape else 2
    x = make(13, lens, counts, heads, kv, size, 16, torch.float16, kind, scales)
    q, kc, vc, ks, vs, bt, sl, cu = x
    held = kc.dtype
    q[:] = 0
    q[..., 0] = 4.0
    kc.copy_(torch.zeros(kc.shape, device="cuda").to(held))
    vc.copy_((vc.float().abs() + 0.25).to(held))
    top = 36.0 if kind == "same" else ref.LARGEST[kind]
    if ks is not None:
        ks[:] = 36.0 / top
    for b, n in enumerate(lens):
        p, s = place_of(x, b, n // 2 if counts[b] < n // 2 else 0)
        kc[int(p), s, :, 0] = torch.tensor(top, device="cuda").to(held)  # its score: 4 * 36 / 8 = 18 above the others
        vc[int(p), s] = torch.zeros(kv, size, device="cuda").to(held)
    got, lse = ops.tree_attention(q, kc, vc, bt, sl, cu, max(counts), 0.125, k_scale=ks, v_scale=vs, return_lse=True)
    check(x, 0.125, None, got, lse)
