"""The attention path on mcpu tensors (torch.ops.mcpu): a serving step gives
the bits it gives on CUDA tensors, and the registrations refuse what the
Python functions refuse."""

import pytest
import torch

from torch_mcpu_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mcpu():
    import torch_mcpu_b200.device  # noqa: F401

    assert torch.mcpu.is_available()


def step(o, x, kind):
    """Rotate and write a drafted step, attend, read the cache back."""
    attend = lambda *a, **k: o.tree_attention(*a, **k)  # noqa: E731
    scales = (x["ks"], x["vs"]) if kind != torch.bfloat16 else (None, None)
    o.rotary_reshape_and_cache(x["pos"], x["q"], x["k"], x["v"], x["tab"], True, x["kc"], x["vc"], x["slots"], *scales)
    o.rotary_embedding(x["pos"], x["k"], None, 64, x["tab"], False)
    more = {"return_lse": True} if o is ops else {}
    out, lse = attend(x["q"], x["kc"], x["vc"], x["bt"], x["lens"], x["cu"], 5, 0.125, x["mask"], *scales, **more)
    o.gather_cache(x["kc"], x["vc"], x["bt"], x["cu_all"], x["ko"], x["vo"], *scales)
    return out, lse


def inputs(kind):
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)  # noqa: E731
    blocks = 6
    x = dict(q=r(7, 4, 64), k=r(7, 2, 64), v=r(7, 2, 64), kc=r(blocks, 16, 2, 64).to(kind), vc=r(blocks, 16, 2, 64).to(kind),
             ks=torch.rand(blocks, 16, 2, generator=g) * 0.01, vs=torch.rand(blocks, 16, 2, generator=g) * 0.01,
             pos=torch.tensor([20, 21, 22, 23, 24, 3, 4]), tab=ops.rotary_cos_sin_cache(64, 64),
             bt=torch.tensor([[4, 1], [2, 0]], dtype=torch.int32), lens=torch.tensor([25, 5], dtype=torch.int32),
             cu=torch.tensor([0, 5, 7], dtype=torch.int32), cu_all=torch.tensor([0, 25, 30], dtype=torch.int32),
             mask=torch.tensor([[1], [3], [5], [11], [21], [1], [3]]), ko=r(30, 2, 64), vo=r(30, 2, 64))
    x["slots"] = torch.cat([x["bt"][0].long()[x["pos"][:5] // 16] * 16 + x["pos"][:5] % 16, 2 * 16 + x["pos"][5:]])
    return x


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float8_e4m3fn, torch.int8])
def test_serving_step_matches_the_cuda_tensors(mcpu, kind):
    host = inputs(kind)
    on_cuda = {n: t.cuda() for n, t in host.items()}
    want = step(ops, on_cuda, kind)
    torch.cuda.synchronize()
    on_mcpu = {n: t.to("mcpu") for n, t in host.items()}
    got = step(torch.ops.mcpu, on_mcpu, kind)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b.cpu())
    for n in ("q", "k", "ko", "vo"):
        assert torch.equal(on_mcpu[n].cpu(), on_cuda[n].cpu()), n
    for n in ("kc", "vc") + (("ks", "vs") if kind != torch.bfloat16 else ()):
        assert torch.equal(on_mcpu[n].cpu().view(torch.int8), on_cuda[n].cpu().view(torch.int8)), n


def test_refusals(mcpu):
    x = {n: t.to("mcpu") for n, t in inputs(torch.int8).items()}
    with pytest.raises(RuntimeError, match="needs k_scale"):
        torch.ops.mcpu.reshape_and_cache(x["k"], x["v"], x["kc"], x["vc"], x["slots"])
    with pytest.raises(RuntimeError, match="slot_mapping"):
        torch.ops.mcpu.reshape_and_cache(x["k"], x["v"], x["kc"], x["vc"], x["slots"][:3], x["ks"], x["vs"])
    with pytest.raises(RuntimeError, match="seq_lens"):
        torch.ops.mcpu.tree_attention(x["q"], x["kc"], x["vc"], x["bt"], x["cu"], x["cu"], 5, 0.1, None, x["ks"], x["vs"])


def test_refusals_on_cuda_tensors():
    x = {n: t.cuda() for n, t in inputs(torch.int8).items()}
    attend = lambda **k: ops.tree_attention(**{**dict(  # noqa: E731
        query=x["q"], key_cache=x["kc"], value_cache=x["vc"], block_table=x["bt"], seq_lens=x["lens"], cu_query_lens=x["cu"],
        max_query_len=5, scale=0.1, tree_mask=x["mask"], k_scale=x["ks"], v_scale=x["vs"]), **k})
    for kw, why in ((dict(query=x["q"][..., :32]), "query must be"), (dict(query=x["q"][:, :3]), "evenly"),
                    (dict(block_table=x["bt"].long()), "block_table"), (dict(seq_lens=x["lens"].long()), "seq_lens"),
                    (dict(cu_query_lens=x["cu"][:2]), "cu_query_lens"), (dict(max_query_len=300), "max_query_len"),
                    (dict(tree_mask=x["mask"].int()), "tree_mask"), (dict(tree_mask=x["mask"][:3]), "tree_mask"),
                    (dict(k_scale=None), "needs k_scale"), (dict(k_scale=x["ks"][:2], v_scale=x["vs"][:2]), "scales must"),
                    (dict(k_scale=x["ks"].half(), v_scale=x["vs"].half()), "float32"), (dict(out=x["q"].float()), "out must"),
                    (dict(out=x["q"][:1].expand(7, 4, 64)), "overlap"), (dict(query=x["q"].cpu()), "device tensor"),
                    (dict(seq_lens=x["lens"].cpu()), "seq_lens is on"), (dict(query="q"), "must be a tensor"),
                    (dict(value_cache=x["vc"].to(torch.bfloat16)), "caches must hold"), (dict(scale="x"), "must be a float")):
        with pytest.raises(RuntimeError, match=why):
            attend(**kw)
    tab = x["tab"]
    for args, why in (((x["pos"][:3], x["q"], None, 64, tab), "positions"), ((x["pos"], x["q"], x["k"].half(), 64, tab), "must both be"),
                      ((x["pos"], x["q"], x["k"][:3], 64, tab), "tokens"), ((x["pos"], x["q"], None, 48, tab), "must be"),
                      ((x["pos"], x["q"], None, 64, tab.double()), "cos_sin_cache"), ((x["pos"], x["q"], x["q"], 64, tab), "overlap"),
                      ((x["pos"], x["q"][:1].expand(7, 4, 64), None, 64, tab), "overlap")):
        with pytest.raises(RuntimeError, match=why):
            ops.rotary_embedding(*args)
    for kw, why in ((dict(key_out=x["ko"].transpose(0, 1)), "one shape"), (dict(cu_seq_lens=x["cu_all"][:2]), "cu_seq_lens"),
                    (dict(key_out=x["ko"].float(), value_out=x["vo"].float()), "bfloat16 or float16")):
        a = dict(key_cache=x["kc"], value_cache=x["vc"], block_table=x["bt"], cu_seq_lens=x["cu_all"], key_out=x["ko"],
                 value_out=x["vo"], k_scale=x["ks"], v_scale=x["vs"])
        with pytest.raises(RuntimeError, match=why):
            ops.gather_cache(**{**a, **kw})
    for kw, why in ((dict(key_cache=x["kc"][:1].expand(6, 16, 2, 64)), "overlap"), (dict(value=x["v"][:3]), "key and value must be"),
                    (dict(k_scale=x["ks"][:1].expand(6, 16, 2)), "overlap"), (dict(value=x["v"].half()), "one type")):
        a = dict(key=x["k"], value=x["v"], key_cache=x["kc"], value_cache=x["vc"], slot_mapping=x["slots"], k_scale=x["ks"],
                 v_scale=x["vs"])
        with pytest.raises(RuntimeError, match=why):
            ops.reshape_and_cache(**{**a, **kw})
