"""Paged K/V cache: step tables, cache writes, attention of drafted tokens, committed branches, against the definitions
in 64 bits."""
import math
import random

import numpy as np
import pytest
import torch

from oracle import paged_oracle as P
from paged_cases import (E4M3, check_attention, local_stride, logit_error, paged_inputs, random_pattern, random_trees, words_of)

pytestmark = pytest.mark.gpu
bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32


def module(bs, pattern, **kw):
    import warnings
    from dkernel_b200 import SparseAttention
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        return SparseAttention(bs, torch.from_numpy(pattern.astype(np.uint8)).cuda(), **kw)


def device(x, copy_k=None):
    """The call's tensors on the GPU; K and V keep the strides that they have."""
    c = dict(x)
    if x["both"] is not None:
        both = x["both"].cuda()
        c["k"], c["v"] = both[:, 0], both[:, 1]
    else:
        c["k"], c["v"] = x["k"].cuda(), x["v"].cuda()
    c["q"], c["table"] = x["q"].cuda(), x["table"].cuda()
    c["lens"] = torch.tensor(x["seqlens"], dtype=torch.int32).cuda()
    c["cu_q"] = torch.tensor(x["cu"], dtype=torch.int32).cuda()
    c["mask"] = None if x["words"] is None else P.as_int64(x["words"]).cuda()
    return c


def call(mod, x, c=None, single=False, **kw):
    c = device(x) if c is None else c
    return mod(c["q"], c["k"], c["v"], block_tables=c["table"], seqlens=c["lens"], cu_seqlen_q=None if single else c["cu_q"],
               tree_mask=c["mask"], kv_scales=x["kv_scales"], **kw)


def reference(x, pattern, bs, scale=None):
    return P.attend(x["q"], x["k"], x["v"], x["table"], x["seqlens"], pattern, bs, cu=x["cu"], words=x["words"],
                    scale=scale, kv_scales=x["kv_scales"] or (1.0, 1.0), seq_dim=x["seq_dim"])


def run_case(hq, hkv, d, ctx, new, page, dtype, bs, pattern, *, impl=None, scale=None, seed=0, **kw):
    x = paged_inputs(seed, hq, hkv, d, ctx, new, page, dtype, **kw)
    mod = module(bs, pattern, seq_dim=x["seq_dim"], impl=impl or "auto")
    single = all(n == 1 for n in new)
    out, lse = call(mod, x, single=single, sm_scale=scale, return_lse=True)
    ref, ref_lse, _ = reference(x, pattern, bs, scale)
    check_attention(out, lse, ref, ref_lse, x, d, scale or 1 / math.sqrt(d))


IMPLS = ["auto", "generic"]


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("hq,hkv,d,dtype,fp8", [
    (8, 2, 128, bf16, False), (4, 4, 64, f16, False), (8, 1, 128, f16, True), (6, 2, 96, bf16, False),
    (5, 5, 64, bf16, True), (14, 2, 64, f16, False), (4, 2, 48, bf16, False), (2, 1, 128, f32, False),
])
def test_draft_trees(impl, hq, hkv, d, dtype, fp8):
    """Contexts that end at, before and behind block and page borders, trees of 1 to 64 drafts, one kv head each."""
    ctx = [0, 1, 63, 64, 65, 200, 511, 300]
    new = [3, 64, 1, 17, 40, 0, 33, 61]
    run_case(hq, hkv, d, ctx, new, 16, dtype, 64, local_stride(hkv, 16, 3, 4), impl=impl, fp8=fp8)


@pytest.mark.parametrize("page", [1, 8, 16, 32, 64, 128, 24])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
def test_page_and_block_sizes(page, bs):
    """Pages finer and coarser than the pattern's blocks, ends inside both."""
    run_case(4, 2, 64, [130, 77, 256, 0], [9, 30, 64, 2], page, bf16, bs, local_stride(2, 64 * 16 // bs, 2, 3), seed=page + bs)


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("heads", ["one", "kv", "q"])
def test_user_patterns(impl, heads):
    """Random patterns: rows without a diagonal, rows that attend nothing, a pattern of its own for every q head."""
    hq, hkv = 6, 2
    n = {"one": 1, "kv": hkv, "q": hq}[heads]
    run_case(hq, hkv, 64, [100, 640, 900, 31], [20, 64, 5, 33], 32, f16, 64, random_pattern(n, 16, 0.3, 3), impl=impl, seed=5)


@pytest.mark.parametrize("bs", [16, 32])
def test_user_patterns_of_small_blocks(bs):
    hq, hkv = 4, 2
    run_case(hq, hkv, 64, [100, 301], [20, 64], 16, bf16, bs, random_pattern(hq, 512 // bs, 0.3, 4), seed=6)


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (3, 3, 64), (20, 1, 64)])
def test_chains_of_any_length(impl, hq, hkv, d):
    """Without a tree mask: single tokens, multi-token steps, prompt chunks longer than a tile."""
    run_case(hq, hkv, d, [0, 70, 0, 500, 64], [300, 129, 1, 7, 64], 16, bf16, 64, local_stride(hkv, 16, 3, 4), impl=impl,
             tree=False, seed=2)


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("fp8", [False, True])
def test_single_tokens(impl, fp8):
    """One query token per request, no cu_seqlen_q: contexts from none at all to long ones."""
    ctx = [0, 1, 15, 16, 63, 64, 1000, 2047, 1500]
    run_case(8, 2, 128, ctx, [1] * len(ctx), 16, bf16, 64, local_stride(2, 32, 4, 4), impl=impl, tree=False, fp8=fp8)


def test_single_tokens_are_the_decode_route():
    """Pages in order hold what a contiguous cache holds: the two decode routes agree to their rounding."""
    hq, hkv, d, bs, S = 8, 2, 128, 64, 1024
    mod = module(bs, local_stride(hkv, 16, 4, 4), seq_dim=1)
    g = torch.Generator().manual_seed(3)
    lens = torch.tensor([1024, 640, 64, 1], dtype=torch.int32)
    B = lens.numel()
    q = torch.randn((B, 1, hq, d), generator=g).to(bf16).cuda()
    k, v = (torch.randn((B, S, hkv, d), generator=g).to(bf16).cuda() for _ in range(2))
    want = mod(q, k, v, left_paddings=torch.zeros(B, dtype=torch.int32).cuda(), seqlens=lens.cuda())
    table = torch.arange(B * S // 32, dtype=torch.int32).view(B, -1).cuda()
    got = mod(q[:, 0], k.view(-1, 32, hkv, d), v.view(-1, 32, hkv, d), block_tables=table, seqlens=lens.cuda())
    assert ((got - want[:, 0]).float().abs() <= 2.0 ** -7 * want[:, 0].float().abs() + 1e-4).all()


@pytest.mark.parametrize("seq_dim,combined", [(1, True), (2, False), (2, True)])
def test_cache_layouts(seq_dim, combined):
    run_case(8, 2, 64, [100, 300], [20, 11], 16, bf16, 64, local_stride(2, 8, 2, 3), seq_dim=seq_dim, combined=combined)


@pytest.mark.parametrize("impl", IMPLS)
def test_missing_pages(impl):
    """Page numbers of -1, too large ones, and a table that ends early: those tokens do not exist."""
    hq, hkv, d, bs = 4, 2, 64, 64
    pat = local_stride(hkv, 8, 2, 2)
    x = paged_inputs(1, hq, hkv, d, [200, 130, 40, 10], [20, 30, 4, 3], 16, bf16)
    x["table"][0, 3] = -1
    x["table"][0, 12:] = -1
    x["table"][1, 5] = x["k"].size(0)
    x["table"][1, 0] = 2 ** 31 - 1
    x["table"][3, :] = -1                     # nothing left
    x["table"] = x["table"][:, :10].contiguous()
    x["k"][:] = x["k"]
    mod = module(bs, pat, seq_dim=1, impl=impl)
    out, lse = call(mod, x, return_lse=True)
    ref, ref_lse, _ = reference(x, pat, bs)
    check_attention(out, lse, ref, ref_lse, x, d, 1 / math.sqrt(d))
    assert (out[-3:] == 0).all() and torch.isinf(lse[:, -3:]).all()


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_attend_cannot_reach_it(impl, bad):
    """Infinities and NaN in free pages, behind a request's end, in other branches' drafts, and in context blocks that
    only some rows or heads attend."""
    hq, hkv, d, bs, page = 4, 2, 128, 64, 16
    pat = random_pattern(hq, 16, 0.5, 9)
    pat[:, np.arange(16), np.arange(16)] = True
    x = paged_inputs(4, hq, hkv, d, [300, 190, 50], [40, 12, 9], page, bf16, combined=False)
    used = torch.zeros(x["k"].shape[:2], dtype=torch.bool)
    for b, n in enumerate(x["seqlens"]):
        for s in range(n):
            used[x["table"][b, s // page], s % page] = True
    clean = reference(x, pat, bs)
    for c in ("k", "v"):
        x[c][~used] = bad

    def slot(b, s):
        return x["table"][b, s // page], s % page

    # the last draft of every request, seen by itself alone
    spoiled = torch.zeros(x["q"].size(0), dtype=torch.bool)
    for b, n in enumerate(x["new"]):
        j = n - 1
        x["words"][x["cu"][b] + j] |= 1 << j
        for i in range(n):
            if x["words"][x["cu"][b] + i] >> j & 1:
                spoiled[x["cu"][b] + i] = True
        for c in ("k", "v"):
            x[c][slot(b, x["ctx"][b] + j)] = bad
    # a context block that head 0 skips where others attend it
    row = 300 // bs
    skip = [c for c in range(row) if not pat[0, row, c] and pat[1:, row, c].any()]
    assert skip
    x["v"][slot(0, skip[0] * bs + 5)] = bad
    mod = module(bs, pat, seq_dim=1, impl=impl)
    out, lse = call(mod, x, return_lse=True)
    ref, ref_lse, _ = reference(x, pat, bs)
    fine = torch.isfinite(ref) & torch.isfinite(ref_lse).T[:, :, None]
    assert fine[~spoiled][:, 0].any() and not fine.all()
    keep = fine.all(-1)
    out, lse = out.cpu(), lse.cpu()
    assert torch.isfinite(out[keep].float()).all()
    e = (out.double() - ref)[keep].abs()
    assert (e <= 2.0 ** -8 * 1.01 * ref[keep].abs() + 2e-3).all()
    assert torch.equal(clean[0][keep & ~spoiled[:, None]], ref[keep & ~spoiled[:, None]])
    # an infinity in an attended V is one in the output, a NaN a NaN
    vis = torch.isfinite(ref_lse).T[:, :, None] & ~torch.isfinite(ref)
    if math.isinf(bad):
        assert torch.equal(torch.isnan(out)[vis], torch.isnan(ref)[vis])
    else:
        assert torch.isnan(out)[vis].all()


@pytest.mark.parametrize("impl", IMPLS)
def test_rows_behind_the_last_request_stay(impl):
    hq, hkv, d, bs = 4, 2, 64, 64
    pat = local_stride(hkv, 8, 2, 3)
    x = paged_inputs(8, hq, hkv, d, [100, 30], [20, 5], 16, f16)
    mod = module(bs, pat, seq_dim=1, impl=impl)
    c = device(x)
    pad = 7
    c["q"] = torch.cat([c["q"], torch.full((pad, hq, d), float("nan"), dtype=f16, device="cuda")])
    c["mask"] = torch.cat([c["mask"], torch.full((pad,), -1, dtype=torch.int64, device="cuda")])
    out = torch.full((c["q"].size(0), hq + 1, d), 7.0, dtype=f16, device="cuda")
    o2 = module(bs, pat, seq_dim=1, impl=impl, out=out[:, 1:])
    got = call(o2, x, c)
    assert (out[:, 0] == 7).all() and (out[-pad:] == 7).all()
    ref, _, _ = reference(x, pat, bs)
    check_attention(got[:-pad], None, ref, None, x, d, 1 / math.sqrt(d))


@pytest.mark.parametrize("impl", IMPLS)
def test_odd_strides_and_scales(impl):
    """q as a slice of a fused projection, (heads, tokens) order, unaligned views; scales of either sign."""
    hq, hkv, d, bs = 4, 2, 64, 64
    pat = local_stride(hkv, 8, 2, 3)
    x = paged_inputs(8, hq, hkv, d, [100, 30], [20, 33], 16, bf16)
    mod = module(bs, pat, seq_dim=1, impl=impl)
    for scale in (0.3, -0.2):
        ref, ref_lse, _ = reference(x, pat, bs, scale)
        for kind in range(4):
            c = device(x)
            T = c["q"].size(0)
            if kind == 1:
                wide = torch.zeros((T, hq + 2 * hkv, d), dtype=bf16, device="cuda")
                wide[:, :hq] = c["q"]
                c["q"] = wide[:, :hq]
            elif kind == 2:
                c["q"] = c["q"].transpose(0, 1).contiguous().transpose(0, 1)
            elif kind == 3:
                flat = torch.zeros(c["q"].numel() + 1, dtype=bf16, device="cuda")
                flat[1:] = c["q"].reshape(-1)
                c["q"] = flat[1:].view(T, hq, d)
            out, lse = call(mod, x, c, sm_scale=scale, return_lse=True)
            check_attention(out, lse, ref, ref_lse, x, d, scale)


def test_caches_that_tma_cannot_read():
    """A slot stride that is no multiple of 16 bytes: served all the same."""
    hq, hkv, d, bs = 2, 1, 64, 64
    pat = local_stride(hkv, 8, 2, 3)
    x = paged_inputs(8, hq, hkv, d, [100, 30], [20, 33], 16, bf16)
    c = device(x)
    for n in ("k", "v"):
        wide = torch.zeros(c[n].shape[:3] + (d + 1,), dtype=bf16, device="cuda")
        wide[..., :d] = c[n]
        c[n] = wide[..., :d]
    out, lse = call(module(bs, pat, seq_dim=1), x, c, return_lse=True)
    ref, ref_lse, _ = reference(x, pat, bs)
    check_attention(out, lse, ref, ref_lse, x, d, 1 / math.sqrt(d))


def test_masks_that_are_no_trees():
    """Rows without their own bit, words of 0 and of all ones, drafts past the 64 that a word can name."""
    hq, hkv, d, bs = 4, 2, 64, 64
    pat = local_stride(hkv, 8, 2, 3)
    x = paged_inputs(8, hq, hkv, d, [100, 0, 60], [20, 4, 70], 16, bf16)
    T = x["q"].size(0)
    rng = random.Random(5)
    x["words"] = [rng.choice([0, (1 << 64) - 1, rng.getrandbits(64), 1 << 63]) for _ in range(T)]
    out, lse = call(module(bs, pat, seq_dim=1), x, return_lse=True)
    ref, ref_lse, _ = reference(x, pat, bs)
    check_attention(out, lse, ref, ref_lse, x, d, 1 / math.sqrt(d))
    assert torch.isinf(ref_lse).any()          # a request without context has rows that attend nothing


def test_positions_past_the_pattern():
    """Rows past the pattern's last attend nothing; the request's earlier rows are served."""
    pat = local_stride(2, 4, 2, 2)
    run_case(4, 2, 64, [250, 100, 300], [12, 5, 3], 16, bf16, 64, pat, tree=False)


def both_ways(x, pat, bs, **kw):
    """The tensor-core kernel and the CUDA-core form of one call."""
    single = all(n == 1 for n in x["new"])
    got = [call(module(bs, pat, seq_dim=x["seq_dim"], impl=impl), x, single=single, return_lse=True, **kw) for impl in ("sm100", "generic")]
    return got


@pytest.mark.parametrize("bs,heads,fp8,tree", [(64, "q", False, True), (64, "kv", True, True), (32, "q", True, True), (16, "kv", False, False),
                                               (64, "kv", False, False), (16, "q", False, True)])
def test_shares_that_end_anywhere(bs, heads, fp8, tree):
    """The items' blocks are cut into equal shares for the CTAs: batches of all sizes, rows with few blocks and without a
    diagonal, so that cuts fall at the first, the last and no block of a row, inside and between items."""
    hq, hkv, d, page = 4, 2, 64, 16
    rng = random.Random(bs)
    nb = 1024 // bs
    for trial in range(24):
        density = rng.choice([0.05, 0.3, 0.9])
        pat = random_pattern({"q": hq, "kv": hkv}[heads], nb, density, trial)
        if trial % 3 == 0:
            pat[:, np.arange(nb), np.arange(nb)] = True
        B = rng.randint(1, 24)
        new = [rng.choice([1, 2, 5, rng.randint(1, 64)]) for _ in range(B)]
        ctx = [rng.choice([0, 64, rng.randint(0, 900)]) for _ in range(B)]
        x = paged_inputs(trial, hq, hkv, d, ctx, new, page, bf16, fp8=fp8, tree=tree)
        (a, la), (b, lb) = both_ways(x, pat, bs)
        # twice the bound of each against 64 bits
        scale = 1 / math.sqrt(d)
        e = logit_error(x, d, scale)
        vmax = P.dequant(x["v"], (x["kv_scales"] or (1.0, 1.0))[1]).abs().max().item()
        assert ((a - b).abs().float() <= 2 * (2.0 ** -8 * b.abs().float() * 1.01 + (4 * e + 2.0 ** -15) * vmax)).all(), (trial, B)
        assert torch.equal(torch.isinf(la), torch.isinf(lb))
        assert (la - lb).nan_to_num(0.0).abs().max() <= 2 * (2 * e + 2.0 ** -20 + 2.0 ** -22 * 16), (trial, B)


def test_empty_batches():
    pat = local_stride(2, 4, 2, 2)
    mod = module(64, pat, seq_dim=1)
    k = torch.zeros((3, 16, 2, 64), dtype=bf16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.zeros((0, 4, 64), dtype=bf16, device="cuda")
    out = mod(q, k, k, block_tables=torch.zeros((0, 4), **i32), seqlens=torch.zeros(0, **i32))
    assert out.shape == q.shape
    out = mod(q, k, k, block_tables=torch.zeros((2, 4), **i32), seqlens=torch.tensor([5, 0], **i32),
              cu_seqlen_q=torch.zeros(3, **i32), tree_mask=torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert out.shape == q.shape
    # a cache without pages, a table without columns, a pattern without blocks: rows that attend nothing
    q = torch.ones((2, 4, 64), dtype=bf16, device="cuda")
    lens = torch.tensor([5, 70], **i32)
    none = module(64, np.zeros((1, 4, 4)), seq_dim=1)
    for m, kk, table in ((mod, k[:0], torch.zeros((2, 8), **i32)), (mod, k, torch.zeros((2, 0), **i32)),
                         (none, k, torch.zeros((2, 8), **i32))):
        out, lse = m(q, kk, kk, block_tables=table, seqlens=lens, return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()


def test_refusals():
    from dkernel_b200 import SparseAttention, commit_paged_draft, plan_paged_step, write_paged_kv
    pat = local_stride(2, 4, 2, 2)
    x = paged_inputs(8, 4, 2, 64, [100, 30], [20, 33], 16, bf16)
    mod, c = module(64, pat, seq_dim=1), device(x)
    good = dict(block_tables=c["table"], seqlens=c["lens"], cu_seqlen_q=c["cu_q"], tree_mask=c["mask"])
    mod(c["q"], c["k"], c["v"], **good)
    for change in (dict(seqlens=None), dict(cu_seqlen_q=None), dict(tree_mask=c["mask"][1:]), dict(tree_mask=c["mask"].int()),
                   dict(block_tables=c["table"][:1]), dict(block_tables=c["table"].long()), dict(seqlens=c["lens"].float()),
                   dict(seqlens=c["lens"].cpu()), dict(left_paddings=c["lens"]), dict(cu_seqlen_k=c["cu_q"]),
                   dict(kv_scales=(1.0, 1.0)), dict(block_tables=None)):
        with pytest.raises(AssertionError):
            mod(c["q"], c["k"], c["v"], **{**good, **change})
    for q, k, v in ((c["q"][None], c["k"], c["v"]), (c["q"], c["k"][:-1], c["v"]), (c["q"], c["k"].half(), c["v"].half()),
                    (c["q"][..., :32], c["k"], c["v"]), (c["q"][:, :3], c["k"], c["v"]), (c["q"], c["k"].to(E4M3), c["v"].to(E4M3)),
                    (c["q"], c["k"].transpose(2, 3), c["v"].transpose(2, 3))):
        with pytest.raises(AssertionError):
            mod(q, k, v, **good)
    with pytest.raises(AssertionError):
        module(64, pat, seq_dim=1, causal=False)(c["q"], c["k"], c["v"], **good)
    q = c["q"].clone().requires_grad_()
    with pytest.raises(AssertionError, match="no backward"):
        mod(q, c["k"], c["v"], **good).float().sum().backward()
    # head dims beyond every kernel
    big = torch.zeros((1, 16, 1, 264), dtype=bf16, device="cuda")
    from dkernel_b200._lib import BsaError
    with pytest.raises(BsaError, match="256"):
        module(64, pat[:1], seq_dim=1)(big[0, :1], big, big, block_tables=c["table"][:1], seqlens=c["lens"][:1])

    slots = torch.zeros(5, dtype=torch.int64, device="cuda")
    k5 = torch.zeros((5, 2, 64), dtype=bf16, device="cuda")
    for bad in (dict(slots=slots.int()), dict(k=k5[:4]), dict(k=k5.half(), v=k5.half()), dict(kv_scales=(1.0, 1.0)),
                dict(k_cache=c["k"].to(E4M3), v_cache=c["v"].to(E4M3)), dict(v=k5.half()), dict(slots=slots.cpu()),
                dict(k_cache=c["k"].to(E4M3), v_cache=c["v"].to(E4M3), kv_scales=(1.0, 0.0)), dict(v_cache=c["v"][1:])):
        kw = {**dict(k=k5, v=k5, k_cache=c["k"], v_cache=c["v"], slots=slots), **bad}
        with pytest.raises(AssertionError):
            write_paged_kv(**kw)
    i32 = dict(dtype=torch.int32, device="cuda")
    st = dict(block_tables=c["table"].clone(), page_counts=torch.zeros(2, **i32), free_pages=torch.zeros(9, **i32),
              num_free=torch.zeros(1, **i32), context_lens=torch.zeros(2, **i32), new_lens=torch.zeros(2, **i32))
    for bad in (dict(page_counts=torch.zeros(3, **i32)), dict(num_free=torch.zeros(1, device="cuda")),
                dict(free_pages=torch.zeros(18, **i32)[::2]), dict(context_lens=torch.zeros(2)), dict(block_tables=c["table"].long()),
                dict(tree_mask=slots)):
        with pytest.raises(AssertionError):
            plan_paged_step(**{**st, **bad}, page_size=16, max_new_tokens=4)
    many = torch.zeros(9000, **i32)
    with pytest.raises(BsaError, match="8192"):
        plan_paged_step(many[:, None].clone(), many, st["free_pages"], st["num_free"], many, many, page_size=16, max_new_tokens=4)
    acc = torch.zeros(2, **i32)
    for bad in (dict(accepted=acc[:1]), dict(accepted=acc.float()), dict(tree_mask=c["mask"].int()), dict(v_cache=c["v"].half()),
                dict(block_tables=c["table"][:1])):
        kw = {**dict(k_cache=c["k"], v_cache=c["v"], block_tables=c["table"], context_lens=acc, cu_seqlen_q=c["cu_q"],
                     accepted=acc, tree_mask=c["mask"]), **bad}
        with pytest.raises(AssertionError):
            commit_paged_draft(**kw)


# ------------------------------------------------------------------ cache writes
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hkv,d,seq_dim", [(2, 128, 1), (3, 40, 2), (1, 7, 1)])
def test_write(dtype, fp8, hkv, d, seq_dim):
    """Bit for bit: rounding to the nearest e4m3 value, ties to even, saturation, NaN; skipped slots; strided input."""
    from dkernel_b200 import write_paged_kv
    pages, page, T = 9, 16, 101
    g = torch.Generator().manual_seed(1)
    kv = (torch.randn((T, 2, hkv, d), generator=g) * 3).to(dtype)
    # values at and between e4m3 steps, past its end, signed zeros, infinities, NaN
    special = torch.tensor([0.0, -0.0, 448.0, 463.9, 464.0, 465.0, -1e5, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 18.0, 19.0,
                            float("inf"), -float("inf"), float("nan")])
    flat = kv.view(-1)
    flat[:special.numel()] = (special * (0.5 if fp8 else 1.0)).to(dtype)
    scales = (0.5, 0.037) if fp8 else None
    shape = (pages, page, hkv, d) if seq_dim == 1 else (pages, hkv, page, d)
    cdt = E4M3 if fp8 else dtype
    order = torch.randperm(pages * page, generator=g)[:T]
    order[::7] = -1
    order[3] = pages * page           # one past the end
    got, want = [], []
    caches = [torch.full(shape, 1.0).to(cdt).cuda() for _ in range(2)]
    dev = kv.cuda()
    write_paged_kv(dev[:, 0], dev[:, 1], *caches, order.cuda(), seq_dim=seq_dim, kv_scales=scales)
    for i in range(2):
        ref = torch.full(shape, 1.0).to(cdt)
        view = ref.view(torch.uint8) if fp8 else ref
        val = kv[:, i]
        if fp8:
            y = val.float() / torch.tensor(scales[i], dtype=f32)
            val = torch.where(torch.isnan(y), y, y.clamp(-448, 448)).to(E4M3).view(torch.uint8)
        for t in range(T):
            s = int(order[t])
            if 0 <= s < pages * page:
                if seq_dim == 1:
                    view[s // page, s % page] = val[t]
                else:
                    view[s // page, :, s % page] = val[t]
        a, b = caches[i].cpu().view(torch.uint8), ref.view(torch.uint8)
        if fp8:      # one NaN is as good as another
            nan = ((a & 0x7f) == 0x7f) & ((b & 0x7f) == 0x7f)
            a, b = torch.where(nan, 0, a), torch.where(nan, 0, b)
            assert torch.equal(a, b)
        else:
            assert torch.equal(caches[i].cpu().nan_to_num(7.0), ref.nan_to_num(7.0))


def test_write_to_a_combined_cache_and_from_transposed_input():
    from dkernel_b200 import write_paged_kv
    both = torch.zeros((5, 2, 16, 2, 64), dtype=bf16, device="cuda")
    k = torch.randn((2, 64, 33), device="cuda").to(bf16).permute(2, 0, 1)          # head dim not contiguous
    slots = torch.randperm(80, device="cuda")[:66][::2]                           # and slots not either
    write_paged_kv(k, k + 1, both[:, 0], both[:, 1], slots)
    assert torch.equal(both[:, 0].reshape(80, 2, 64)[slots], k)
    assert torch.equal(both[:, 1].reshape(80, 2, 64)[slots], k + 1)
    assert both[:, 0].reshape(80, -1).any(1).sum() == 33


# ------------------------------------------------------------------ a step's tables
def _step_state(rng, B, W, P, ctx, extra):
    total = sum(-(-c // P) for c in ctx)
    pages = list(range(total + extra))
    rng.shuffle(pages)
    table, counts, at = [], [], 0
    for c in ctx:
        n = min(W, -(-c // P))
        table.append(pages[at:at + n] + [-1] * (W - n))
        counts.append(n)
        at += n
    free = pages[at:]
    return table, counts, free + [-5] * (total + extra - len(free)), len(free)


@pytest.mark.parametrize("B,P,W,extra,tokens,tree", [
    (1, 16, 8, 4, 3, True), (7, 16, 40, 60, 50, False), (40, 8, 30, 25, 400, True), (300, 1, 40, 500, 2000, False),
    (1500, 64, 6, 800, 9000, False), (5, 16, 3, 100, 200, False), (2000, 16, 4, 0, 100, True),
])
def test_step_tables(B, P, W, extra, tokens, tree):
    """Growth, shrinking, ended requests, a stack that runs empty, tables that are too narrow, more new tokens than the
    batch takes; several steps in a row on the same state."""
    from dkernel_b200 import plan_paged_step
    rng = random.Random(B)
    ctx = [rng.randint(0, W * P) for _ in range(B)]
    table, counts, stack, top = _step_state(rng, B, W, P, ctx, extra)
    i32 = dict(dtype=torch.int32, device="cuda")
    wide = torch.full((B, W + 3), -9, **i32)           # rows inside a wider table
    wide[:, :W] = torch.tensor(table, dtype=torch.int32)
    dt, dc, ds, dn = wide[:, :W], torch.tensor(counts, **i32), torch.tensor(stack, **i32), torch.tensor([top], **i32)
    for it in range(4):
        new = [rng.choice([0, 1, rng.randint(0, 2 * P), -3]) for _ in range(B)]
        # the next context: some accepted, some rolled back, some ended
        if it:
            ctx = [rng.choice([0, c, max(0, c - rng.randint(0, 3 * P)), c + 1]) for c in ctx]
            new = [0 if c == 0 and rng.random() < 0.7 else n for c, n in zip(ctx, new)]
        words = [rng.getrandbits(64) for _ in range(tokens)] if tree else None
        want = P_step = P_ref(table, counts, stack, top, ctx, new, P, tokens, words)
        got = plan_paged_step(dt, dc, ds, dn, torch.tensor(ctx, **i32), torch.tensor(new, **i32), page_size=P,
                              max_new_tokens=tokens, tree_mask=P_mask(words))
        assert got.cu_seqlen_q.tolist() == want["cu"] and got.seqlens.tolist() == want["seqlens"]
        assert dc.tolist() == want["counts"] and dn.item() == want["num_free"] and got.short.item() == want["short"]
        assert dt.tolist() == want["table"]
        assert ds.tolist() == want["stack"]
        assert got.slots.tolist() == want["slots"] and got.positions.tolist() == want["positions"]
        table, counts, stack, top = want["table"], want["counts"], want["stack"], want["num_free"]
        assert (wide[:, W:] == -9).all()
        held = sum(counts)
        assert held + top == len(stack)               # no page is lost or handed out twice


def P_ref(*a):
    return P.step(*a)


def P_mask(words):
    return None if words is None else P.as_int64(words).cuda()


def test_step_without_requests():
    from dkernel_b200 import plan_paged_step
    i32 = dict(dtype=torch.int32, device="cuda")
    e = torch.zeros(0, **i32)
    n = torch.tensor([4], **i32)
    got = plan_paged_step(torch.zeros((0, 5), **i32), e, torch.arange(4, **i32), n, e, e, page_size=16, max_new_tokens=3)
    assert got.cu_seqlen_q.tolist() == [0] and got.slots.tolist() == [-1] * 3 and n.item() == 4 and got.short.item() == 0


# ------------------------------------------------------------------ committed branches
@pytest.mark.parametrize("dtype,d,seq_dim,combined", [(bf16, 128, 1, False), (f32, 64, 2, False), (E4M3, 96, 1, True), (f16, 7, 1, False)])
@pytest.mark.parametrize("tree", [True, False])
def test_commit(dtype, d, seq_dim, combined, tree):
    from dkernel_b200 import commit_paged_draft
    ctx, new = [100, 0, 33, 15, 64, 500, 7], [64, 5, 1, 30, 0, 17, 64]
    x = paged_inputs(3, 2, 2, d, ctx, new, 16, f32 if dtype == E4M3 else dtype, seq_dim=seq_dim, combined=combined, tree=tree)
    if dtype == E4M3:
        x["both"] = x["both"].to(E4M3)
        x["k"], x["v"] = x["both"][:, 0], x["both"][:, 1]
    x["table"][5, 32] = -1                      # a page that is missing: its drafts do not move
    acc = [63, -1, 0, 22, 0, 16, 64]
    if tree:
        # a chain that is out of order, and the longest branch there is
        x["words"][x["cu"][3]:x["cu"][4]] = [(1 << 22) | (1 << 9) | (1 << 1) if j == 22 else 1 << j for j in range(30)]
        x["words"][63] = (1 << 64) - 1 - 2
    c = device(x)
    i32 = dict(dtype=torch.int32, device="cuda")
    ctx_d = torch.tensor(ctx, **i32)
    lens = commit_paged_draft(c["k"], c["v"], c["table"], ctx_d, c["cu_q"], torch.tensor(acc, **i32), tree_mask=c["mask"],
                              seq_dim=seq_dim)
    words = x["words"]
    for name in ("k", "v"):
        want, want_lens = P.commit(x[name], x["table"], ctx, x["cu"], acc, words, seq_dim)
        a, b = c[name].cpu().contiguous().view(torch.uint8), want.contiguous().view(torch.uint8)
        assert torch.equal(a, b)
    assert lens.tolist() == want_lens and ctx_d.tolist() == ctx


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("fp8", [False, True])
def test_speculative_decoding_end_to_end(fp8):
    """Steps of drafting, verifying and committing on one pool of pages; after every commit the pages hold exactly the
    sequence that the accepted tokens spell, and attention over them equals attention over that sequence."""
    from dkernel_b200 import commit_paged_draft, plan_paged_step, write_paged_kv
    hq, hkv, d, bs, page, B, W = 8, 2, 64, 64, 16, 5, 24
    pat = local_stride(hkv, 6, 2, 3)
    mod = module(bs, pat, seq_dim=1)
    rng = random.Random(11)
    g = torch.Generator().manual_seed(11)
    i32 = dict(dtype=torch.int32, device="cuda")
    pages = 70
    cdt = E4M3 if fp8 else bf16
    scales = (0.03, 0.03) if fp8 else None
    kc = torch.full((pages, page, hkv, d), float("nan")).to(cdt).cuda()
    vc = kc.clone()
    table, counts = torch.full((B, W), -1, **i32), torch.zeros(B, **i32)
    free, top = torch.randperm(pages, generator=g).to(torch.int32).cuda(), torch.tensor([pages], **i32)
    ctx = torch.zeros(B, **i32)
    story = [[] for _ in range(B)]               # (k, v) of the accepted tokens, per request
    for it in range(6):
        if it == 0:                              # prompts, as chains
            new = [70, 1, 130, 64, 33]
            trees = [list(range(-1, n - 1)) for n in new]
        else:
            new = [rng.randint(1, 40) for _ in range(B)]
            trees = random_trees(rng, new)
        if it == 3:                              # request 1 has ended, a new one takes its place
            ctx[1] = 0
            story[1] = []
        T = sum(new)
        mask = None if it == 0 else P.as_int64(words_of(trees)).cuda()
        step = plan_paged_step(table, counts, free, top, ctx, torch.tensor(new, **i32), page_size=page, max_new_tokens=T,
                               tree_mask=mask)
        assert step.short.item() == 0
        q, k, v = (torch.randn((T, h, d), generator=g).to(bf16) for h in (hq, hkv, hkv))
        write_paged_kv(k.cuda(), v.cuda(), kc, vc, step.slots, kv_scales=scales)
        out, lse = mod(q.cuda(), kc, vc, block_tables=table, seqlens=step.seqlens, cu_seqlen_q=step.cu_seqlen_q, tree_mask=mask,
                       kv_scales=scales, return_lse=True)
        cu = step.cu_seqlen_q.tolist()
        x = dict(q=q, k=torch.where(torch.isnan(kc.float()), 0.0, kc.float()).cpu(),
                 v=torch.where(torch.isnan(vc.float()), 0.0, vc.float()).cpu(), kv_scales=scales)
        if fp8:
            x["k"], x["v"] = x["k"].to(E4M3), x["v"].to(E4M3)
        ref, ref_lse, _ = P.attend(q, x["k"], x["v"], table.cpu(), step.seqlens.tolist(), pat, bs, cu=cu,
                                   words=None if it == 0 else words_of(trees), kv_scales=scales or (1.0, 1.0))
        check_attention(out, lse, ref, ref_lse, x, d, 1 / math.sqrt(d))
        acc = [n - 1 for n in new] if it == 0 else [rng.randint(-1, n - 1) for n in new]
        ctx = commit_paged_draft(kc, vc, table, ctx, step.cu_seqlen_q, torch.tensor(acc, **i32), tree_mask=mask)
        quant = (lambda t, s: (t.float() / torch.tensor(s)).clamp(-448, 448).to(E4M3).float()) if fp8 else (lambda t, s: t.float())
        for b in range(B):
            path, j = [], acc[b]
            while j >= 0:
                path.append(j)
                j = trees[b][j]
            for j in reversed(path):
                t = cu[b] + j
                story[b].append((quant(k[t], (scales or (1, 1))[0]), quant(v[t], (scales or (1, 1))[1])))
            assert ctx[b].item() == len(story[b])
            for s, (kk, vv) in enumerate(story[b]):
                pg = table[b, s // page].item()
                assert torch.equal(kc[pg, s % page].float().cpu(), kk) and torch.equal(vc[pg, s % page].float().cpu(), vv)


# ------------------------------------------------------------------ how it runs
def test_which_kernel_serves():
    """The tensor-core kernel serves every 16-bit call with its pages, blocks and strides; asked for by name it refuses the
    others, with the reason."""
    from dkernel_b200._lib import BsaError
    hq, hkv, bs = 4, 2, 64
    for d, dtype, page, fp8, why in ((128, bf16, 16, False, None), (48, f16, 8, False, None), (64, bf16, 128, True, None),
                                     (64, f32, 16, False, "dtype"), (160, bf16, 16, False, "head dim"), (40, bf16, 16, True, "head dim"),
                                     (64, bf16, 24, False, "page size"), (64, bf16, 4, False, "page size")):
        x = paged_inputs(1, hq, hkv, d, [70, 3], [5, 9], page, dtype, fp8=fp8)
        mod = module(bs, local_stride(hkv, 4, 2, 2), seq_dim=1, impl="sm100")
        if why is None:
            call(mod, x)
        else:
            with pytest.raises(BsaError, match=why):
                call(mod, x)
    mod = module(128, local_stride(hkv, 4, 2, 2), seq_dim=1, impl="sm100")       # refined to blocks of 64
    call(mod, paged_inputs(1, hq, hkv, 64, [70, 3], [5, 9], 16, bf16))


def test_same_bits_every_time():
    x = paged_inputs(2, 8, 2, 128, [900, 333, 10], [60, 17, 1], 16, bf16)
    mod, c = module(64, local_stride(2, 16, 3, 4), seq_dim=1), device(x)
    first = call(mod, x, c, return_lse=True)
    for _ in range(5):
        again = call(mod, x, c, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_long_cache():
    """Pages whose offsets pass 2^32 bytes and 2^31 elements."""
    from dkernel_b200 import commit_paged_draft, write_paged_kv
    hkv, d, page, pages = 8, 128, 64, 40000            # 2.6e9 elements
    kc = torch.empty((pages, page, hkv, d), dtype=bf16, device="cuda")
    vc = torch.empty_like(kc)
    hq, bs = 8, 64
    g = torch.Generator().manual_seed(1)
    T = 150
    k, v = (torch.randn((T, hkv, d), generator=g).to(bf16) for _ in range(2))
    used = [39999, 17, 35000]
    slots = torch.tensor([used[t // page] * page + t % page for t in range(T)]).cuda()
    write_paged_kv(k.cuda(), v.cuda(), kc, vc, slots)
    assert torch.equal(kc[39999].cpu(), k[:64]) and torch.equal(vc[35000, :T - 128].cpu(), v[128:])
    pat = local_stride(hkv, 4, 3, 2)
    n = 10
    q = torch.randn((n, hq, d), generator=g).to(bf16)
    words = [P.tree_word([j - 2 if j > 1 else -1 for j in range(n)], j) for j in range(n)]
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.tensor([used], **i32)
    args = dict(block_tables=table, seqlens=torch.tensor([T], **i32), cu_seqlen_q=torch.tensor([0, n], **i32),
                tree_mask=P.as_int64(words).cuda())
    small = torch.zeros((3, page, hkv, d), dtype=bf16)
    small.view(-1, hkv, d)[:T] = k
    small_v = torch.zeros_like(small)
    small_v.view(-1, hkv, d)[:T] = v
    ref, ref_lse, _ = P.attend(q, small, small_v, torch.tensor([[0, 1, 2]]), [T], pat, bs, cu=[0, n], words=words)
    x = dict(q=q, k=small, v=small_v, kv_scales=None)
    for impl in IMPLS:
        out, lse = module(bs, pat, seq_dim=1, impl=impl)(q.cuda(), kc, vc, return_lse=True, **args)
        check_attention(out, lse, ref, ref_lse, x, d, 1 / math.sqrt(d))
    lens = commit_paged_draft(kc, vc, table, torch.tensor([T - n], **i32), args["cu_seqlen_q"], torch.tensor([9], **i32),
                              tree_mask=args["tree_mask"])
    assert lens.item() == T - n + 5
    assert torch.equal(kc[35000, 12:17].cpu(), k[T - n + 1::2]) and torch.equal(vc[35000, 12:17].cpu(), v[T - n + 1::2])


def test_other_streams_and_two_graphs():
    """A step captured into two graphs (each with its workspace), replayed in turn and at the same time on two streams, with
    new inputs in the captured buffers; an eager call on a side stream."""
    from dkernel_b200 import commit_paged_draft, plan_paged_step, write_paged_kv
    hq, hkv, d, bs, page, B, W = 8, 2, 128, 64, 16, 6, 40
    pat = local_stride(hkv, 16, 3, 4)
    mod = module(bs, pat, seq_dim=1)
    i32 = dict(dtype=torch.int32, device="cuda")
    new = [9, 33, 1, 64, 17, 5]
    T, pages = sum(new), 260
    rng = random.Random(7)

    class Server:
        def __init__(self, seed):
            g = torch.Generator().manual_seed(seed)
            self.g = g
            self.kc, self.vc = (torch.randn((pages, page, hkv, d), generator=g).to(bf16).cuda() for _ in range(2))
            self.table, self.counts = torch.full((B, W), -1, **i32), torch.zeros(B, **i32)
            self.free, self.top = torch.randperm(pages, generator=g).to(torch.int32).cuda(), torch.tensor([pages], **i32)
            self.ctx, self.new = torch.zeros(B, **i32), torch.tensor(new, **i32)
            self.q, self.k, self.v = (torch.zeros((T, h, d), dtype=bf16, device="cuda") for h in (hq, hkv, hkv))
            self.mask, self.acc = torch.zeros(T, dtype=torch.int64, device="cuda"), torch.zeros(B, **i32)

        def fill(self):
            trees = random_trees(rng, new)
            self.words = words_of(trees)
            self.ctx.copy_(torch.tensor([rng.randint(0, 500) for _ in range(B)], dtype=torch.int32))
            for t in (self.q, self.k, self.v):
                t.copy_(torch.randn(t.shape, generator=self.g).to(bf16))
            self.mask.copy_(P.as_int64(self.words))
            self.acc.copy_(torch.tensor([rng.randint(-1, n - 1) for n in new], dtype=torch.int32))

        def step(self):
            st = plan_paged_step(self.table, self.counts, self.free, self.top, self.ctx, self.new, page_size=page,
                                 max_new_tokens=T, tree_mask=self.mask)
            write_paged_kv(self.k, self.v, self.kc, self.vc, st.slots)
            out, lse = mod(self.q, self.kc, self.vc, block_tables=self.table, seqlens=st.seqlens, cu_seqlen_q=st.cu_seqlen_q,
                           tree_mask=self.mask, return_lse=True)
            lens = commit_paged_draft(self.kc, self.vc, self.table, self.ctx, st.cu_seqlen_q, self.acc, tree_mask=self.mask)
            return out, lse, lens, st

        def state(self):
            return [t.clone() for t in (self.kc, self.vc, self.table, self.counts, self.free, self.top)]

        def restore(self, s):
            for t, x in zip((self.kc, self.vc, self.table, self.counts, self.free, self.top), s):
                t.copy_(x)

    servers, graphs, outs, streams = [Server(1), Server(2)], [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s, st in zip(servers, streams):
        s.fill()
        keep = s.state()
        with torch.cuda.stream(st):
            s.step()                                   # everything is loaded before the capture
        torch.cuda.synchronize()
        s.restore(keep)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            outs.append(s.step())
        graphs.append(graph)
    for rounds in range(4):
        want = []
        for s in servers:
            s.fill()
            keep = s.state()
            with torch.cuda.stream(streams[0]):        # eagerly, on a side stream
                streams[0].wait_stream(torch.cuda.current_stream())
                res = s.step()
            torch.cuda.current_stream().wait_stream(streams[0])
            want.append([t.clone() for t in res[:3]] + s.state())
            s.restore(keep)
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):         # at the same time
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for s, o, w in zip(servers, outs, want):
            for got, ref in zip(list(o[:3]) + s.state(), w):
                assert torch.equal(got.view(torch.uint8) if got.is_floating_point() else got,
                                   ref.view(torch.uint8) if ref.is_floating_point() else ref)
    from dkernel_b200 import _lib
    assert _lib.wait_status() == 0


CHILD = r"""
import hashlib, json, sys
sys.path[:0] = [%(root)r, %(root)r + "/tests"]
import torch
import test_paged_gpu as t
from dkernel_b200 import _lib
from paged_cases import local_stride, paged_inputs, random_pattern
out = {}
def run(name, x, pat, bs, single=False):
    o, l = t.call(t.module(bs, pat, seq_dim=x["seq_dim"], impl="sm100"), x, single=single, return_lse=True)
    h = hashlib.md5(torch.nan_to_num(o.float()).cpu().numpy().tobytes())
    h.update(torch.nan_to_num(l, neginf=-1e30).cpu().numpy().tobytes())
    out[name] = h.hexdigest()
bf16, f16 = torch.bfloat16, torch.float16
ctx, new = [0, 63, 500, 333, 900], [64, 3, 40, 0, 61]
run("trees", paged_inputs(1, 8, 2, 128, ctx, new, 16, bf16), local_stride(2, 16, 3, 4), 64)
run("e4m3", paged_inputs(2, 8, 2, 128, ctx, new, 32, bf16, fp8=True), local_stride(2, 16, 3, 4), 64)
run("rows", paged_inputs(3, 6, 2, 64, ctx, new, 8, f16), random_pattern(6, 16, 0.3, 2), 64)
run("small", paged_inputs(4, 4, 4, 96, ctx, new, 16, f16), random_pattern(4, 64, 0.3, 2), 16)
run("chains", paged_inputs(5, 20, 1, 64, [0, 70, 300], [300, 129, 7], 64, bf16, tree=False), local_stride(1, 16, 3, 4), 64)
run("tokens", paged_inputs(6, 8, 2, 128, [0, 64, 1000], [1, 1, 1], 16, bf16, fp8=True, tree=False), local_stride(2, 16, 3, 4), 64, True)
x = paged_inputs(7, 4, 2, 64, [200, 130], [20, 30], 16, bf16)
x["table"][0, 3] = -1; x["table"][1, 5] = 10 ** 6
run("missing", x, local_stride(2, 8, 2, 2), 64)
torch.cuda.synchronize()
print(json.dumps(dict(status=_lib.wait_status(), lib=_lib.LIB_PATH, out=out)))
"""


def test_checking_build_runs_clean():
    """The same calls through the release and the bounds-checking library: no check fires, the outputs are the same bits."""
    import json
    import os
    import subprocess
    import sys
    from dkernel_b200 import _build
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    got = []
    for lib in (_build.LIB, _build.LIB_DEBUG):
        assert os.path.exists(lib)
        r = subprocess.run([sys.executable, "-c", CHILD % dict(root=root)], capture_output=True, text=True, timeout=300,
                           env={**os.environ, "BSA_B200_LIB": lib})
        assert r.returncode == 0, r.stdout + r.stderr
        got.append(json.loads(r.stdout.strip().splitlines()[-1]))
    assert got[0]["status"] == got[1]["status"] == 0
    assert got[0]["lib"] != got[1]["lib"] and got[0]["out"] == got[1]["out"]


def test_many_rows_that_a_nan_reaches():
    """Every row of a long context attends a NaN: all are recomputed, none of the kernel's waits gives up meanwhile."""
    from dkernel_b200 import _lib
    hq, hkv, d, page, n, L = 4, 1, 64, 64, 64, 16000
    mod = module(64, np.tril(np.ones((1, 256, 256))), seq_dim=1, impl="sm100")
    x = paged_inputs(2, hq, hkv, d, [L], [n], page, bf16)
    x["v"][x["table"][0, 100], 5] = float("nan")
    out, lse = call(mod, x, return_lse=True)
    torch.cuda.synchronize()
    assert _lib.wait_status() == 0
    assert torch.isnan(out).all() and torch.isfinite(lse).all()
