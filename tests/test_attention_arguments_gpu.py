"""What the attention path's functions refuse and note on CUDA tensors:
gradients they cannot give, written tensors that overlap, arguments that are no
truth values."""

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
    """A tensor that autograd has saved and a call has written since is noticed by the backward pass."""
    for call, tensors, written in calls():
        for name in written:
            x = tensors[name]
            weight = torch.ones(x.shape, device="cuda", requires_grad=True)
            if x.dtype != torch.float32:
                weight = torch.ones(x.shape, dtype=x.dtype, device="cuda", requires_grad=True)
            y = (weight * x).sum()
            call(tensors)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()
        for name, x in tensors.items():
            before = x._version
            call(tensors)
            assert (x._version > before) == (name in written), name


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
