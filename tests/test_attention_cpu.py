"""Host side of the attention path, without a device: the rotary table and the
argument errors the C entry points return before anything is enqueued."""

import ctypes
import math
import struct

import pytest
import torch

from torch_mcpu_b200 import _lib, ops

CACHE = struct.Struct("=4Q13q6i")
P = 1 << 20  # a 16-byte-aligned address that is never followed


def cache(**kw):
    a = dict(key=P, value=P, ks=0, vs=0, blocks=4, k=(2048, 128, 64), v=(2048, 128, 64), s=(0, 0, 0), block=16, kv=2, head=64,
             dtype=1, mode=0)
    a.update(kw)
    return CACHE.pack(a["key"], a["value"], a["ks"], a["vs"], a["blocks"], *a["k"], *a["v"], *a["s"], *a["s"], a["block"], a["kv"],
                      a["head"], a["dtype"], a["mode"], 0)


BAD_CACHES = [
    (dict(dtype=0), b"cache holds"), (dict(dtype=2), b"cache holds"), (dict(dtype=8), b"scales"), (dict(dtype=10, mode=3), b"scales"),
    (dict(mode=1), b"scales"), (dict(dtype=8, mode=1), b"NULL"), (dict(head=72), b"multiple of 16"), (dict(head=528), b"at most 512"),
    (dict(block=0), b"sizes"), (dict(k=(2048, 127, 64)), b"16 bytes"), (dict(v=(2048, 128, -64)), b"16 bytes"), (dict(key=P + 2), b"aligned"),
    (dict(key=0), b"NULL"), (dict(blocks=-1), b"sizes")]


def write(c, **kw):
    a = dict(pos=P, tokens=3, q=P, heads=4, key=P, value=P, part=64, table=P, reach=10, dtype=1, slots=P)
    a.update(kw)
    lib = _lib.load()
    rc = lib.mcpu_rotary_reshape_and_cache(a["pos"], a["tokens"], a["q"], a["heads"], 256, 64, a["key"], 128, 64, a["value"], 128, 64,
                                           a["part"], a["table"], a["reach"], 1, a["dtype"], a["slots"], c, None)
    return rc, lib.mcpuGetLastErrorString()


def gather(c, **kw):
    a = dict(table=P, stride=8, width=8, batch=2, cu=P, k=P, v=P, tokens=5, dtype=1)
    a.update(kw)
    lib = _lib.load()
    rc = lib.mcpu_gather_cache(c, a["table"], a["stride"], a["width"], a["batch"], a["cu"], None, a["k"], a["v"], a["tokens"], a["dtype"], None)
    return rc, lib.mcpuGetLastErrorString()


def attend(c, **kw):
    a = dict(q=P, qt=256, qh=64, tokens=5, heads=4, out=P, ot=256, oh=64, dtype=1, table=P, stride=8, width=8, batch=2, lens=P, cu=P,
             most=3, mask=0, mstride=0, words=0, work=P, have=1 << 40)
    a.update(kw)
    lib = _lib.load()
    rc = lib.mcpu_tree_attention(a["q"], a["qt"], a["qh"], a["tokens"], a["heads"], a["out"], a["ot"], a["oh"], None, a["dtype"], c,
                                 a["table"], a["stride"], a["width"], a["batch"], a["lens"], a["cu"], a["most"], a["mask"], a["mstride"],
                                 a["words"], 0.1, a["work"], a["have"], None)
    return rc, lib.mcpuGetLastErrorString()


@pytest.mark.parametrize("kw,msg", BAD_CACHES)
@pytest.mark.parametrize("call", [write, gather, attend])
def test_bad_caches(call, kw, msg):
    rc, said = call(cache(**kw))
    assert rc == 4 and msg in said, said


@pytest.mark.parametrize("call,kw,msg", [
    (write, dict(part=24), b"multiple of 16"), (write, dict(part=63), b"even"), (write, dict(part=128), b"at most head_size"),
    (write, dict(reach=0), b"empty"), (write, dict(pos=0), b"NULL"), (write, dict(key=0), b"NULL"), (write, dict(slots=0), b"NULL"),
    (write, dict(tokens=-1), b"sizes"), (write, dict(dtype=0), b"bfloat16 or float16"), (write, dict(table=P + 4), b"aligned"),
    (gather, dict(stride=4), b"sizes"), (gather, dict(cu=0), b"NULL"), (gather, dict(k=P + 2), b"aligned"), (gather, dict(batch=-1), b"sizes"),
    (attend, dict(heads=3), b"multiple of num_kv_heads"), (attend, dict(most=0), b"max_query_len"), (attend, dict(most=257), b"max_query_len"),
    (attend, dict(have=16), b"workspace"), (attend, dict(work=0), b"NULL"), (attend, dict(mask=P, words=0), b"tree_mask"),
    (attend, dict(mask=P, words=1, mstride=1, most=65), b"tree_mask"), (attend, dict(qh=60), b"aligned"), (attend, dict(q=P + 8), b"aligned"),
    (attend, dict(batch=1 << 28, width=1 << 20, stride=1 << 20), b"too large"), (attend, dict(lens=0), b"NULL")])
def test_bad_arguments(call, kw, msg):
    rc, said = call(cache(), **kw)
    assert rc == 4 and msg in said, said


def test_attention_head_sizes_and_empty_cache():
    rc, said = attend(cache(head=96, k=(4096, 256, 128), v=(4096, 256, 128)))
    assert rc == 4 and b"64 or 128" in said
    rc, said = attend(cache(blocks=0))
    assert rc == 4 and b"no blocks" in said


def test_nothing_to_do_is_no_error():
    assert write(cache(), tokens=0)[0] == 0
    assert gather(cache(), tokens=0)[0] == 0 and gather(cache(), batch=0)[0] == 0
    assert attend(cache(), tokens=0)[0] == 0 and attend(cache(), batch=0)[0] == 0
    lib = _lib.load()
    assert lib.mcpu_rotary_embedding(None, 0, None, 4, 0, 0, None, 0, 0, 0, 64, None, 1, 1, 1, None) == 0


@pytest.mark.parametrize("part,reach,dtype,msg", [(63, 10, 1, b"even"), (0, 10, 1, b"even"), (64, 0, 1, b"empty"), (64, 10, 3, b"float32")])
def test_rotary_refusals(part, reach, dtype, msg):
    lib = _lib.load()
    rc = lib.mcpu_rotary_embedding(P, 3, P, 4, 256, 64, None, 0, 0, 0, part, P, reach, 1, dtype, None)
    assert rc == 4 and msg in lib.mcpuGetLastErrorString()


def test_workspace_grows_with_the_rows():
    lib = _lib.load()
    sizes = []
    for most in (1, 8, 64):
        n = ctypes.c_uint64()
        assert lib.mcpu_tree_attention_workspace_bytes(most, 8, 2, 128, ctypes.byref(n)) == 0
        sizes.append(n.value)
    assert 0 < sizes[0] <= sizes[1] <= sizes[2]


def test_device_tensors_are_required():
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    c = torch.zeros(1, 16, 2, 64, dtype=torch.bfloat16)
    i32, i64 = torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ops.rotary_embedding(i64, x, None, 64, torch.zeros(4, 64)),
                 lambda: ops.reshape_and_cache(x, x, c, c, i64),
                 lambda: ops.gather_cache(c, c, i32[None], i32, x, x),
                 lambda: ops.tree_attention(x, c, c, i32[None], i32, i32, 1, 0.1)):
        with pytest.raises(RuntimeError, match="device tensor"):
            call()


# ------------------------------------------------------------------ rotary table
def plain_angles(reach, part, base):
    """Angles with Python's integers and floats, position by position."""
    return [[p * base ** (-2 * i / part) for i in range(part // 2)] for p in range(reach)]


def test_table():
    t = ops.rotary_cos_sin_cache(50, 16, 10000.0)
    assert t.dtype == torch.float32 and t.shape == (50, 16)
    a = torch.tensor(plain_angles(50, 16, 10000.0), dtype=torch.float64)
    assert ((t[:, :8].double() - a.cos()).abs() <= 2.0 ** -25 + 1e-12).all()
    assert ((t[:, 8:].double() - a.sin()).abs() <= 2.0 ** -25 + 1e-12).all()


def test_table_scalings():
    part, base = 64, 10000.0
    plain = ops.rotary_cos_sin_cache(512, part, base)
    assert torch.equal(ops.rotary_cos_sin_cache(512, part, base, {"rope_type": "linear", "factor": 4.0})[::4], plain[:128])
    dyn = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 256}
    assert torch.equal(ops.rotary_cos_sin_cache(256, part, base, dyn), plain[:256])
    grown = base * (2.0 * 512 / 256 - 1.0) ** (part / (part - 2))
    assert torch.equal(ops.rotary_cos_sin_cache(512, part, base, dyn), ops.rotary_cos_sin_cache(512, part, grown))
    ll = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 128}
    t = ops.rotary_cos_sin_cache(100, part, base, ll)
    inv = [base ** (-2 * i / part) for i in range(part // 2)]
    for i, f in enumerate(inv):
        wave = 2 * math.pi / f
        if wave < 128 / 4:
            want = f
        elif wave > 128 / 1:
            want = f / 8
        else:
            s = (128 / wave - 1.0) / (4.0 - 1.0)
            want = (1 - s) * f / 8 + s * f
        assert abs(t[99, i].item() - math.cos(99 * want)) < 1e-6
    ya = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 512}
    t = ops.rotary_cos_sin_cache(100, part, base, ya)
    amp = 0.1 * math.log(4.0) + 1
    assert abs(t[0, 0].item() - amp) < 1e-6
    assert abs(t[50, 0].item() - amp * math.cos(50.0)) < 1e-6                       # fast dimension: not stretched
    assert abs(t[50, 31].item() - amp * math.cos(50.0 * inv[31] / 4)) < 1e-6      # slow one: by the factor


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=0), dict(max_position=0), dict(base=-1.0),
                                dict(scaling={"rope_type": "longrope"}), dict(scaling={"rope_type": "linear", "factor": 0}),
                                dict(scaling={"rope_type": "llama3", "factor": 8.0}), dict(scaling={"rope_type": "yarn", "factor": 2.0})])
def test_table_refusals(kw):
    a = dict(max_position=8, rotary_dim=8)
    a.update(kw)
    with pytest.raises(RuntimeError, match="rotary_cos_sin_cache"):
        ops.rotary_cos_sin_cache(**a)
