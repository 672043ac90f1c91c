"""A single new token whose mask does not let it see itself: what its own key
and value hold (NaN, infinities) does not reach its output."""

import math

import pytest
import torch

from test_attention_gpu import make
from torch_mcpu_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,kind,scales", [
    (torch.bfloat16, "same", "none"), (torch.float16, "same", "none"), (torch.bfloat16, torch.float8_e4m3fn, "token"),
    (torch.bfloat16, torch.float8_e4m3fn, "tensor"), (torch.float16, torch.int8, "token")])
@pytest.mark.parametrize("heads,counts", [(4, [1, 1, 1]), (12, [1, 1, 1]), (32, [1, 1, 1]), (2, [1, 1, 40]), (4, [1, 1, 60])])
def test_single_token_that_does_not_see_itself(dtype, kind, scales, heads, counts):
    lens = [150, 1, 90]  # a context, none, and a request beside them
    x = make(4, lens, counts, heads, 1, 64, 16, dtype, kind, scales)
    q, kc, vc, ks, vs, bt, sl, cu = x
    mask = torch.zeros(sum(counts), 1, dtype=torch.int64, device="cuda")
    mask[2:, 0] = torch.arange(counts[2], device="cuda") * 0 + 1
    call = lambda: ops.tree_attention(q, kc, vc, bt, sl, cu, max(counts), 0.125, tree_mask=mask, k_scale=ks, v_scale=vs,  # noqa: E731
                                      return_lse=True)
    ops.device_error(reset=True)
    clean = call()
    for bad in (math.nan, math.inf, -math.inf):
        for b, n in enumerate(lens[:2]):
            p, s = int(bt[b, (n - 1) // 16]), (n - 1) % 16
            if kind != torch.int8:
                kc[p, s, 0, 3], vc[p, s, 0, 5] = bad, bad  # e4m3: NaN
            if scales == "token":
                ks[p, s], vs[p, s] = bad, bad
        got = call()
        assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])
        assert (got[0][1] == 0).all() and (got[1][1] == -math.inf).all()
        assert torch.isfinite(got[0]).all()
    assert ops.device_error() == 0
