"""Paged attention where logits are NaN: a row that attends one is NaN, with a NaN LSE; every other row keeps its bits."""
import math

import numpy as np
import pytest
import torch

from oracle import paged_oracle as P
from paged_cases import E4M3, local_stride, paged_inputs
from test_paged_gpu import call, device, module

pytestmark = pytest.mark.gpu
bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
NAN = float("nan")
IMPLS = ["auto", "generic"]
TYPES = [(bf16, False), (f16, False), (bf16, True), (f16, True)]


def spoil(cache, page, slot):
    """All of a token's heads become NaN (e4m3 has one byte pattern for it)."""
    if cache.dtype == E4M3:
        cache.view(torch.uint8)[page, slot] = 0x7f
    else:
        cache[page, slot] = NAN


def expect(x, pat, bs, impl, single, **kw):
    """The call's outputs, compared with the oracle's: NaN where that has NaN, finite elsewhere."""
    mod = module(bs, pat, seq_dim=1, impl=impl)
    c = device(x)
    out, lse = call(mod, x, c, single=single, return_lse=True, **kw)
    ref, ref_lse, _ = P.attend(x["q"], x["k"], x["v"], x["table"], x["seqlens"], pat, bs, cu=x["cu"], words=x["words"],
                               kv_scales=x["kv_scales"] or (1.0, 1.0))
    out, lse = out.cpu(), lse.cpu()
    bad = torch.isnan(ref_lse).T                       # (T, Hq)
    assert torch.equal(torch.isnan(lse).T, bad)
    assert torch.isnan(out[bad]).all() and torch.isfinite(out[~bad]).all()
    return out, lse, bad


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("dtype,fp8", TYPES)
@pytest.mark.parametrize("bad", [NAN, math.inf])
@pytest.mark.parametrize("kind", ["tokens", "trees", "chains"])
def test_query_rows(impl, dtype, fp8, bad, kind):
    """A NaN in a row of q makes all its logits NaN; an infinity makes some of them +inf, whose softmax is NaN, too."""
    hq, hkv, d, bs = 8, 2, 128, 64
    pat = local_stride(hkv, 32, 3, 4)
    ctx = [0, 64, 700, 1900, 130]
    new = {"tokens": [1] * 5, "trees": [3, 64, 1, 17, 40], "chains": [5, 1, 70, 33, 200]}[kind]
    x = paged_inputs(3, hq, hkv, d, ctx, new, 16, dtype, fp8=fp8, tree=kind == "trees")
    single = kind == "tokens"
    clean, clean_lse = call(module(bs, pat, seq_dim=1, impl=impl), x, single=single, return_lse=True)
    rows = [(0, 1), (2, 7), (x["cu"][3], 0), (x["cu"][4] - 1, 3)]
    x["q"] = x["q"].clone()
    for i, (t, h) in enumerate(rows):
        x["q"][t, h, 37 * i] = bad
    if math.isinf(bad):
        # every key's share of the logit is positive: +inf, and NaN of it
        for i, (t, h) in enumerate(rows):
            x["k"] = x["k"].clone()
            raw = x["k"].view(torch.uint8) if fp8 else x["k"].view(torch.int16)
            raw[..., 37 * i] = raw[..., 37 * i] & (0x7f if fp8 else 0x7fff) | 1
        clean, clean_lse = call(module(bs, pat, seq_dim=1, impl=impl),
                                {**x, "q": torch.where(torch.isfinite(x["q"]), x["q"], 0.5)}, single=single, return_lse=True)
    mod = module(bs, pat, seq_dim=1, impl=impl)
    out, lse = call(mod, x, single=single, return_lse=True)
    hit = torch.zeros(out.shape[:2], dtype=torch.bool, device="cuda")
    for t, h in rows:
        hit[t, h] = True
    assert torch.isnan(out[hit]).all() and torch.isnan(lse.T[hit]).all()
    assert torch.equal(out[~hit], clean[~hit]) and torch.equal(lse.T[~hit], clean_lse.T[~hit])


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("dtype,fp8", TYPES)
@pytest.mark.parametrize("S", [1, 17, 33, 49, 64, 65, 81])
def test_a_nan_key_alone_in_its_quarter(impl, dtype, fp8, S):
    """The new token's own key is NaN, the first of 16 keys or of a block: the row is NaN, not what the others give."""
    hq, hkv, d, bs = 8, 2, 128, 64
    pat = local_stride(hkv, 4, 4, 2)
    x = paged_inputs(S, hq, hkv, d, [S - 1, 70], [1, 1], 16, dtype, fp8=fp8, tree=False)
    spoil(x["k"], x["table"][0, (S - 1) // 16], (S - 1) % 16)
    _, _, bad = expect(x, pat, bs, impl, True)
    assert bad[0].all() and not bad[1].any()


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("tree", [False, True])
def test_a_nan_page_among_patterns(impl, fp8, tree):
    """Pages of NaN keys, first, last and in the middle of what a row attends; rows and heads that skip them stay finite."""
    hq, hkv, d, bs, page = 4, 2, 64, 64, 16
    pat = local_stride(hkv, 16, 2, 3)
    ctx, new = [300, 650, 64, 20], ([9, 40, 1, 64] if tree else [1, 1, 1, 1])
    reached = []
    for block in (0, 1, 3, 4, 8, 9, 10):
        x = paged_inputs(block, hq, hkv, d, ctx, new, page, bf16, fp8=fp8, tree=tree, width=48)
        for b in range(4):
            for pi in range(block * bs // page, (block + 1) * bs // page):
                if x["table"][b, pi].item() >= 0:
                    for s in range(page):
                        spoil(x["k"], x["table"][b, pi], s)
        _, _, bad = expect(x, pat, bs, impl, not tree)
        reached.append(bad.any().item())
        assert not bad.all()
    assert sum(reached) >= 5               # a single token's rows skip some block altogether


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n,heads", [(1, 4), (7, 4), (40, 4), (3, 1)])
def test_a_nan_page_anywhere_in_a_share(fp8, n, heads):
    """One request over the whole machine: its blocks are cut into shares, each with a maximum of its own.  Wherever a block
    of NaN keys lies, first in a share or not, every row is NaN."""
    hkv, d, bs, page, nb = 1, 128, 64, 64, 40
    pat = np.tril(np.ones((1, nb, nb), bool))
    L = nb * bs - 70
    x = paged_inputs(1, heads, hkv, d, [L], [n], page, bf16, fp8=fp8, tree=n > 1)
    mod, c = module(bs, pat, seq_dim=1, impl="sm100"), device(x)
    keep = c["k"].view(torch.uint8).clone()
    for block in range(L // page):
        c["k"].view(torch.uint8).copy_(keep)
        c["k"].view(torch.uint8)[c["table"][0, block]] = 0x7f if fp8 else 0xff
        out, lse = call(mod, x, c, single=n == 1, return_lse=True)
        assert torch.isnan(out).all() and torch.isnan(lse).all(), block
    from dkernel_b200 import _lib
    assert _lib.wait_status() == 0
