"""Paged cache: calls that the documentation allows and that are easily got wrong."""
import math

import pytest
import torch

from oracle import paged_oracle as P
from paged_cases import local_stride, paged_inputs
from test_paged_gpu import call, module

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16


@pytest.mark.parametrize("impl", ["auto", "generic"])
@pytest.mark.parametrize("kind", ["tokens", "trees", "chains"])
@pytest.mark.parametrize("fp8", [False, True])
def test_requests_that_store_nothing(impl, kind, fp8):
    """A batch padded with idle requests: seqlens 0, query rows all the same, and a block table that still names pages.  Their
    rows attend nothing; the others' are what they are without them."""
    hq, hkv, d, bs = 8, 2, 64, 64
    pat = local_stride(hkv, 8, 2, 3)
    n = 1 if kind == "tokens" else 200 if kind == "chains" else 20
    ctx = [100, 0, 230, 0, 0, 17]
    x = paged_inputs(5, hq, hkv, d, ctx, [n] * 6, 16, bf16, fp8=fp8, tree=kind == "trees")
    idle = [1, 3, 4]
    for b in idle:
        x["seqlens"][b] = 0
    assert (x["table"][idle, 0] >= 0).all()
    out, lse = call(module(bs, pat, seq_dim=1, impl=impl), x, single=n == 1, return_lse=True)
    keep = torch.ones(6 * n, dtype=torch.bool, device="cuda")
    for b in idle:
        keep[x["cu"][b]:x["cu"][b + 1]] = False
    assert (out[~keep] == 0).all() and (lse[:, ~keep] == -math.inf).all()
    # the oracle has no keys for them either
    ref, ref_lse, _ = P.attend(x["q"], x["k"], x["v"], x["table"], x["seqlens"], pat, bs, cu=x["cu"], words=x["words"],
                               kv_scales=x["kv_scales"] or (1.0, 1.0))
    assert torch.equal(torch.isinf(lse).cpu(), torch.isinf(ref_lse))
    assert (out.cpu().double() - ref).abs().max() < 0.02
