"""What the attention path's functions refuse and note on CUDA tensors:
gradients they cannot give, written tensors that overlap, arguments that are no
truth values."""

import os
import subprocess
import sys

import pytest
import torch

from test_attention_gpu import make, new_cache, gen, randn, table
from torch_mcpu_b200 import ops

pytestmark = pytest.mark.gpu


def calls():
    """Each function with its tensors by name: (call, tensors, names of those it writes)."""
    g = gen(2)
    half = torch.bfloat16
    kc, vc, ks, vs = new_cache(4, 16, 2, 64, torch.int8, half, "token", g)
    k16, v16 = (randn(g, 4, 16, 2, 64, dtype=half) for _ in range(2))
    q, k, v, k_out, v_out, out = (randn(g, 3, h, 64, dtype=half) for h in (4, 2, 2, 2, 2, 4))
    tab, pos = table(8, 64), torch.arange(3, device="cuda")
    bt = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    cu, sl = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 3], [3]))
    return [
        (lambda t: ops.rotary_embedding(pos, t["query"], t["key"], 64, t["table"], True),
         dict(query=q, key=k, table=tab), ("query", "key")),
        (lambda t: ops.reshape_and_cache(t["key"], t["value"], t["key_cache"], t["value_cache"], pos),
         dict(key=k, value=v, key_cache=k16, value_cache=v16), ("key_cache", "value_cache")),
        (lambda t: ops.rotary_reshape_and_cache(pos, t["query"], t["key"], t["value"], t["table"], True, kc, vc, pos, t["k_scale"],
                                                t["v_scale"]),
         dict(query=q, key=k, value=v, table=tab, k_scale=ks, v_scale=vs), ("query", "k_scale", "v_scale")),
        (lambda t: ops.gather_cache(t["key_cache"], t["value_cache"], bt, cu, t["key_out"], t["value_out"]),
         dict(key_cache=k16, value_cache=v16, key_out=k_out, value_out=v_out), ("key_out", "value_out")),
        (lambda t: ops.gather_cache(kc, vc, bt, cu, k_out, v_out, t["k_scale"], t["v_scale"]), dict(k_scale=ks, v_scale=vs), ()),
        (lambda t: ops.tree_attention(t["query"], t["key_cache"], t["value_cache"], bt, sl, cu, 3, 0.125, out=t["out"]),
         dict(query=q, key_cache=k16, value_cache=v16, out=out), ("out",)),
        (lambda t: ops.tree_attention(q, kc, vc, bt, sl, cu, 3, 0.125, k_scale=t["k_scale"], v_scale=t["v_scale"]),
         dict(k_scale=ks, v_scale=vs), ()),
    ]


def test_every_tensor_that_requires_a_gradient_is_refused():
    for call, tensors, _ in calls():
        call(tensors)
        for name, x in tensors.items():
            leaf = x.clone().requires_grad_()
            with pytest.raises(RuntimeError, match="requires a gradient"):
                call({**tensors, name: leaf})
            with torch.no_grad():
                call({**tensors, name: leaf})
            with torch.inference_mode():
                call({**tensors, name: leaf})


def test_written_tensors_count_as_changed():
    for call, tensors, written in calls():
        for name, x in tensors.items():
            before = x._version
            call(tensors)
            assert (x._version > before) == (name in written), name


def test_backward_pass_notices_a_saved_tensor_that_was_written():
    """In a process of its own: where the mcpu device is registered, torch's engine runs no backward pass on CUDA tensors."""
    code = """
import torch
from test_attention_arguments_gpu import calls
n = 0
for call, tensors, written in calls():
    for name in written:
        x = tensors[name]
        weight = torch.ones(x.shape, dtype=x.dtype, device="cuda", requires_grad=True)
        y = (weight * x).sum()
        call(tensors)
        try:
            y.backward()
        except RuntimeError as e:
            assert "modified by an inplace operation" in str(e), e
            n += 1
print("noticed", n, sum(len(w) for _, _, w in calls()))
"""
    here = os.path.dirname(os.path.abspath(__file__))
    paths = os.pathsep.join([here, os.path.dirname(here)])
    done = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(here), env={**os.environ, "PYTHONPATH": paths},
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
    said, n, of = done.stdout.split()
    assert said == "noticed" and n == of and int(n) > 5, done.stdout


def test_tensors_of_inference_mode_are_taken():
    with torch.inference_mode():
        for call, tensors, _ in calls():
            call(tensors)
    for call, tensors, _ in calls():
        with torch.inference_mode():
            call({n: x.clone() for n, x in tensors.items()})


def test_written_mcpu_tensors_count_as_changed():
    import torch_mcpu_b200.device  # noqa: F401

    q, k, tab = (x.cpu().to("mcpu") for x in calls()[0][1].values())
    pos = torch.arange(3).to("mcpu")
    for x in (q, k, tab):
        assert not x.requires_grad
    before = [x._version for x in (q, k, tab)]
    torch.ops.mcpu.rotary_embedding(pos, q, k, 64, tab, True)
    assert [x._version > b for x, b in zip((q, k, tab), before)] == [True, True, False]
    with pytest.raises(RuntimeError, match="requires a gradient"):
        torch.ops.mcpu.rotary_embedding(pos, q, k, 64, tab.clone().requires_grad_(), True)


def test_written_tensors_that_overlap_with_an_offset_are_refused():
    g = gen(4)
    half = torch.bfloat16
    pos = torch.arange(3, device="cuda")
    bt = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    tab = table(8, 64)
    packed = randn(g, 3, 8, 64, dtype=half)
    k, v = randn(g, 3, 2, 64, dtype=half), randn(g, 3, 2, 64, dtype=half)
    pages = randn(g, 9, 16, 2, 64, dtype=half)
    ks = torch.zeros(9, 16, 2, device="cuda")
    kc8, vc8 = (torch.zeros(4, 16, 2, 64, dtype=torch.int8, device="cuda") for _ in range(2))
    rows = randn(g, 8, 2, 64, dtype=half)
    for call, why in (
            (lambda: ops.rotary_embedding(pos, packed[:, :4], packed[:, 3:5], 64, tab), "query and key are written"),
            (lambda: ops.rotary_embedding(pos, packed[:, 2:6], packed[:, 1:3], 64, tab), "query and key are written"),
            (lambda: ops.rotary_embedding(pos[:2], packed[:2, :4], packed[1:, 2:4], 64, tab), "query and key are written"),
            (lambda: ops.rotary_embedding(pos, packed.view(3, 512)[:, :256], packed.view(3, 512)[:, 248:504], 64, tab),
             "query and key are written"),
            (lambda: ops.reshape_and_cache(k, v, pages[:4], pages[3:7], pos), "key_cache and value_cache are written"),
            (lambda: ops.reshape_and_cache(k, v, pages[:8:2], pages[2::2], pos), "key_cache and value_cache are written"),
            (lambda: ops.reshape_and_cache(k, v, pages.view(-1)[:8192].view(4, 16, 2, 64), pages.view(-1)[2048 - 64:][:8192].view(4, 16, 2, 64), pos),
             "key_cache and value_cache are written"),
            (lambda: ops.reshape_and_cache(k, v, kc8, vc8, pos, ks[:4], ks[2:6]), "k_scale and v_scale are written"),
            (lambda: ops.rotary_reshape_and_cache(pos, packed[:, :4], packed[:, 3:5], v, tab, True, pages[:4], pages[4:8], pos),
             "query is written"),
            (lambda: ops.rotary_reshape_and_cache(pos, packed[:, :4], k, packed[:, 2:4], tab, True, pages[:4], pages[4:8], pos),
             "query is written"),
            (lambda: ops.gather_cache(pages[:4], pages[4:8], bt, cu, rows[:3], rows[2:5]), "key_out and value_out are written"),
            (lambda: ops.tree_attention(rows[:3], pages[:4], pages[4:8], bt, cu[1:], cu, 3, 0.1, out=rows[1:4]), "out is written")):
        before = [x.clone() for x in (packed, pages, ks, rows)]
        with pytest.raises(RuntimeError, match=why):
            call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(before, (packed, pages, ks, rows)))


def test_interleaved_tensors_are_taken():
    """Views of one tensor that share no element, in the layouts that programs have."""
    g = gen(5)
    half = torch.bfloat16
    pos = torch.arange(3, device="cuda")
    bt = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    tab = table(8, 64)
    packed = randn(g, 3, 8, 64, dtype=half)
    flat = packed.view(3, 512)
    by_group = randn(g, 3, 2, 4, 64, dtype=half)  # key heads, then its two query heads, key and value
    want = packed.clone()
    ops.rotary_embedding(pos, want, None, 64, tab)
    for q, k in ((packed[:, :4], packed[:, 4:6]), (packed[:, 2:], packed[:, :2]), (flat[:, :256], flat[:, 256:384]),
                 (packed[..., 0:8:2, :], packed[..., 1:8:2, :]), (by_group[:, :, 0], by_group[:, :, 2]),
                 (packed.transpose(0, 1)[:3, :3], packed.transpose(0, 1)[3:6, 3:6])):
        ops.rotary_embedding(pos[:q.shape[0]], q, k, 64, tab)
    ops.rotary_reshape_and_cache(pos, packed[:, :4], packed[:, 4:6], packed[:, 6:], tab, True,
                                 *randn(g, 2, 4, 16, 2, 64, dtype=half).unbind(0), pos)
    k, v = randn(g, 3, 2, 64, dtype=half), randn(g, 3, 2, 64, dtype=half)
    for both in (randn(g, 2, 4, 16, 2, 64, dtype=half), randn(g, 4, 2, 16, 2, 64, dtype=half).transpose(0, 1),
                 randn(g, 4, 16, 2, 2, 64, dtype=half).permute(2, 0, 1, 3, 4), randn(g, 4, 16, 2, 2, 64, dtype=half).permute(3, 0, 1, 2, 4),
                 randn(g, 4, 16, 2, 128, dtype=half).view(4, 16, 2, 2, 64).permute(3, 0, 1, 2, 4),
                 randn(g, 2, 4, 2, 16, 64, dtype=half).transpose(2, 3), randn(g, 4, 2, 2, 16, 64, dtype=half).permute(1, 0, 3, 2, 4)):
        ops.reshape_and_cache(k, v, both[0], both[1], pos)
        outs = randn(g, 2, 3, 2, 64, dtype=half)
        ops.gather_cache(both[0], both[1], bt, cu, outs[0], outs[1])
        assert torch.equal(outs[0], k) and torch.equal(outs[1], v)
    kc8, vc8 = (torch.zeros(4, 16, 2, 64, dtype=torch.int8, device="cuda") for _ in range(2))
    for s in (torch.zeros(4, 16, 2, 2, device="cuda").unbind(-1), torch.zeros(4, 2, 16, 2, device="cuda").unbind(1),
              torch.zeros(2, 4, 16, 2, device="cuda").unbind(0)):
        ops.reshape_and_cache(k, v, kc8, vc8, pos, *s)
    shifted = randn(g, 4, 4, 64, dtype=half)
    ops.rotary_embedding(pos, shifted[:3, :2], shifted[1:, 2:], 64, tab)  # a token further in the other heads
    q = packed[:, 2:6]
    want = ops.tree_attention(q, both[0], both[1], bt, cu[1:], cu, 3, 0.1)
    assert torch.equal(ops.tree_attention(q, both[0], both[1], bt, cu[1:], cu, 3, 0.1, out=packed[:, 6:].repeat(1, 2, 1)), want)
    assert torch.equal(ops.tree_attention(q, both[0], both[1], bt, cu[1:], cu, 3, 0.1, out=q), want)  # in place of the queries


def test_arguments_that_are_no_truth_values():
    import numpy as np

    neither = np.zeros(2)
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    kc, vc = (torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pos, tab = torch.arange(3, device="cuda"), table(8, 64)
    bt = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    cu, sl = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 3], [3]))
    for call, name in ((lambda: ops.rotary_embedding(pos, q, None, 64, tab, neither), "is_neox"),
                       (lambda: ops.rotary_reshape_and_cache(pos, q, q.clone(), q.clone(), tab, neither, kc, vc, pos), "is_neox"),
                       (lambda: ops.tree_attention(q, kc, vc, bt, sl, cu, 3, 0.1, return_lse=neither), "return_lse")):
        with pytest.raises(RuntimeError, match=name + " must be a bool"):
            call()


def test_expanded_tensors():
    """Dimensions of stride 0: refused where they are written, taken where they are read."""
    g = gen(6)
    half = torch.bfloat16
    pos, tab = torch.arange(3, device="cuda"), table(8, 64)
    kc, vc = (randn(g, 4, 16, 2, 64, dtype=half) for _ in range(2))
    one = randn(g, 1, 1, 64, dtype=half)
    k = one.expand(3, 2, 64)  # the same row for all heads and tokens
    ops.reshape_and_cache(k, k, kc, vc, pos)
    assert torch.equal(kc[0, :3], k) and torch.equal(vc[0, :3], k)
    q = randn(g, 3, 4, 64, dtype=half)
    ops.rotary_reshape_and_cache(pos, q, k, k, tab, True, kc, vc, pos)
    inside = q[:1, :1].expand(3, 2, 64)  # a row of the queries that are rotated
    with pytest.raises(RuntimeError, match="query is written"):
        ops.rotary_reshape_and_cache(pos, q, inside, k, tab, True, kc, vc, pos)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.reshape_and_cache(k, k, kc[:1].expand(4, 16, 2, 64), kc, pos)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.reshape_and_cache(k, k, kc[:, :, :1].expand(4, 16, 2, 64), kc[:, :, 1:].expand(4, 16, 2, 64), pos)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.rotary_embedding(pos, q, inside, 64, tab)
