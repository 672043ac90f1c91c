"""Roundings of the rotary positions and of the cache's read-back: each result
is the exact value rounded once."""

import pytest
import torch

import attention_reference as ref
from test_attention_gpu import gen
from torch_mcpu_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8])
def test_read_back_is_rounded_once(dtype, kind):
    """Every value of the 8-bit type times many scales: products of up to 32 bits, exact in 64."""
    g = gen(1)
    tokens, kv, size, block = 2048, 8, 256, 16
    codes = torch.arange(256, device="cuda", dtype=torch.uint8).view(torch.int8)
    if kind == torch.float8_e4m3fn:
        codes = torch.where((codes & 127) == 127, torch.zeros_like(codes), codes)  # no NaN
    cache = codes.view(kind)[None, None, None].expand(tokens // block, block, kv, size).contiguous()
    scale = torch.rand(tokens // block, block, kv, generator=g, device="cuda") + 0.5
    scale *= torch.where(torch.rand(scale.shape, generator=g, device="cuda") < 0.5, 0.01, 1.0)
    far = scale.clone()
    if dtype == torch.bfloat16:  # scales of every size, the smallest and largest among them
        exponent = torch.randint(-149, 119, scale.shape, generator=g, device="cuda")
        far = torch.ldexp(scale.double() + 0.5, exponent).float()
    bt = torch.arange(tokens // block, dtype=torch.int32, device="cuda")[None]
    cu = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
    out = [torch.empty(tokens, kv, size, dtype=dtype, device="cuda") for _ in range(2)]
    ops.gather_cache(cache, cache, bt, cu, *out, scale, far)
    for s, o in zip((scale, far), out):
        want = (cache.double() * s.double()[..., None]).view(tokens, kv, size)
        rounded = ref.nearest(want, dtype)
        ok = rounded.abs() <= torch.finfo(dtype).max
        assert torch.equal(o.double()[ok], rounded[ok]) and o.double()[~ok].isinf().all()
    twice = [(cache.float() * s[..., None]).view(tokens, kv, size).to(dtype) for s in (scale, far)]
    assert not all(torch.equal(a, b) for a, b in zip(twice, out))  # there are products that two roundings get wrong


def test_read_back_of_rows_that_are_not_finite():
    cache = torch.ones(1, 4, 1, 16, device="cuda").to(torch.int8)
    cache[0, 0, 0, 3] = 0
    scale = torch.tensor([float("inf"), float("nan"), 3e38, 1.0], device="cuda").view(1, 4, 1)
    bt, cu = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    out = [torch.empty(4, 1, 16, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ops.gather_cache(cache, cache, bt, cu, *out, scale, scale)
    for o in out:
        assert o[0, 0, 0].isinf() and o[0, 0, 3].isnan() and o[1].isnan().all() and torch.isfinite(o[2:]).all()


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("tokens,heads,size,part", [(200, 5, 128, 128), (33, 3, 192, 64), (17, 2, 80, 20)])
def test_rotation_in_32_bits(neox, tokens, heads, size, part):
    """fma(a, c, -rn(b s)): half a step of b s and half a step of the result, also where the result all but vanishes."""
    g = gen(tokens)
    x = torch.randn(tokens, heads, size, generator=g, device="cuda")
    x[:, 0] *= 1e-3
    pos = torch.randint(0, 4000, (tokens,), generator=g, device="cuda")
    tab = ops.rotary_cos_sin_cache(4000, part, device="cuda")
    half = part // 2
    row = tab[pos]
    a, b = (slice(0, half), slice(half, part)) if neox else (slice(0, part, 2), slice(1, part, 2))
    x[:, 1, a], x[:, 1, b] = row[:, half:], row[:, :half] * (1 + 2.0 ** -14)  # pairs next to (sin, cos)
    want = ref.rotated(x, pos, tab, neox)
    sin = row[:, None, half:].double().abs()
    second = torch.zeros_like(want)
    second[..., a], second[..., b] = x[..., b].double().abs() * sin, x[..., a].double().abs() * sin
    rest = x[..., part:].clone()
    ops.rotary_embedding(pos, x, None, size, tab, neox)
    # a rounding of a value is off by 2^-24 of it; the result's is taken of what it is before, 2^-24 of the product away
    bound = 2.0 ** -24 * (second + want.abs()) * (1 + 2.0 ** -23) + 2.0 ** -48 * second
    assert ((x.double() - want).abs()[..., :part] <= bound[..., :part]).all()
    assert torch.equal(x[..., part:], rest)
