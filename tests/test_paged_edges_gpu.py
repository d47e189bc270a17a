"""Paged cache: calls that the documentation allows and that are easily got wrong."""
import math

import pytest
import torch

from oracle import paged_oracle as P
from paged_cases import local_stride, paged_inputs
from test_paged_gpu import call, device, module

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


@pytest.mark.parametrize("tokens", [4096, 6000])
def test_page_counts_outside_the_table(tokens):
    """Counts that no step wrote, past the table's width or negative: the request holds its whole row, or nothing, and no
    token gets a slot of its neighbour's, in the step of one launch and in that of two."""
    from dkernel_b200 import plan_paged_step
    i32 = dict(dtype=torch.int32, device="cuda")
    page, W = 16, 4
    table = torch.arange(3 * W, **i32).view(3, W).contiguous()
    table[1] = -1
    counts = torch.tensor([9, -5, W + 1], **i32)
    stack, top = torch.arange(100, 110, **i32), torch.tensor([10], **i32)
    ctx, new = [10, 0, 63], [2000, 20, 2000]
    got = plan_paged_step(table, counts, stack, top, torch.tensor(ctx, **i32), torch.tensor(new, **i32), page_size=page,
                          max_new_tokens=tokens)
    assert counts.tolist() == [W, 2, W] and top.item() == 8 and got.short.item() == 0
    assert table.tolist() == [[0, 1, 2, 3], [109, 108, -1, -1], [8, 9, 10, 11]]
    want = []
    for b, pages in enumerate(table.tolist()):
        for i in range(new[b]):
            at = ctx[b] + i
            want.append(pages[at // page] * page + at % page if at < W * page and pages[at // page] >= 0 else -1)
    assert got.slots.tolist() == want + [-1] * (tokens - len(want))


def test_commit_behind_every_page():
    """Context lengths up to the largest int32, where no page is: nothing moves, lengths saturate."""
    from dkernel_b200 import commit_paged_draft
    i32 = dict(dtype=torch.int32, device="cuda")
    for page in (1, 16):
        k, v = (torch.randn((4, page, 2, 64), device="cuda").to(bf16) for _ in range(2))
        keep = [k.clone(), v.clone()]
        table = torch.arange(4, **i32)[None].repeat(3, 1)
        ctx = torch.tensor([2 ** 31 - 1, 2 ** 31 - 20, -7], **i32)
        n = 64
        words = P.as_int64([(1 << 64) - 2 if j == 63 else 1 << j for j in range(n)] * 3).cuda()
        acc = torch.tensor([63, 63, -1], **i32)
        lens = commit_paged_draft(k, v, table, ctx, torch.tensor([0, n, 2 * n, 3 * n], **i32), acc, tree_mask=words)
        assert lens.tolist() == [2 ** 31 - 1, 2 ** 31 - 1, 0]
        assert torch.equal(k, keep[0]) and torch.equal(v, keep[1])


def test_calls_for_the_cuda_cores_say_so():
    """16-bit calls that the tensor-core kernel does not serve are reported, once per reason; fp32, calls by name, and calls
    without a page are not."""
    import warnings
    from dkernel_b200 import ops
    pat = local_stride(2, 4, 2, 2)

    def warned(d=64, dtype=bf16, page=16, fp8=False, impl="auto", width=None):
        x = paged_inputs(1, 4, 2, d, [70, 3], [5, 9], page, dtype, fp8=fp8)
        if width is not None:
            x["table"] = x["table"][:, :width]
        with warnings.catch_warnings(record=True) as got:
            warnings.simplefilter("always")
            call(module(64, pat, seq_dim=1, impl=impl), x)
        return [str(w.message) for w in got if issubclass(w.category, RuntimeWarning)]

    keep = set(ops._warned_fallback)
    try:
        ops._warned_fallback.clear()
        assert not warned() and not warned(dtype=torch.float32) and not warned(page=24, impl="generic") and not warned(width=0)
        assert ["page size" in m for m in warned(page=24)] == [True]
        assert not warned(page=24)
        assert ["head dim" in m for m in warned(d=40, fp8=True)] == [True]
    finally:
        ops._warned_fallback.clear()
        ops._warned_fallback.update(keep)


def test_contiguous_tensors_off_the_16_byte_boundary():
    """Slices of a larger buffer that are contiguous and start 2 bytes off are copied, not handed to the CUDA cores."""
    pat = local_stride(2, 8, 2, 3)

    def off(t):
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    x = paged_inputs(8, 4, 2, 64, [100, 30], [20, 33], 16, bf16)
    mod, c = module(64, pat, seq_dim=1, impl="sm100"), device(x)
    want = call(mod, x, c)
    q = off(c["q"])
    assert q.data_ptr() % 16 == 2 and q.is_contiguous()
    assert torch.equal(call(mod, x, {**c, "q": q}), want)
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn((2, 200, h, 64), generator=g).to(bf16).cuda() for h in (4, 2, 2))
    with torch.no_grad():
        assert torch.equal(mod(off(q), off(k), off(v)), mod(q, k, v))
        last = [q[:, -1:].contiguous(), k, v]
        assert torch.equal(mod(*map(off, last)), mod(*last))


def test_broadcast_queries():
    """One query row for all heads, or for all tokens (stride 0), on the tensor-core kernel."""
    pat = local_stride(2, 8, 2, 3)
    x = paged_inputs(8, 4, 2, 64, [100, 30], [20, 33], 16, bf16)
    mod, c = module(64, pat, seq_dim=1, impl="sm100"), device(x)
    for q in (c["q"][:, :1].expand(-1, 4, -1), c["q"][:1].expand(53, -1, -1), c["q"][:1, :1].expand(53, 4, -1)):
        assert torch.equal(call(mod, x, {**c, "q": q}), call(mod, x, {**c, "q": q.contiguous()}))
    x = paged_inputs(8, 1, 1, 64, [100, 30], [20, 33], 16, bf16)
    mod, c = module(64, pat[:1], seq_dim=1, impl="sm100"), device(x)
    q = c["q"].as_strided((53, 1, 64), (0, 0, 1))
    assert torch.equal(call(mod, x, {**c, "q": q}), call(mod, x, {**c, "q": q.contiguous()}))


def test_forward_mode_tangents_are_refused():
    """There is no derivative: a tangent on q or the caches raises, as on the contiguous route, with and without no_grad."""
    import torch.autograd.forward_ad as fwd
    pat = local_stride(2, 8, 2, 3)
    x = paged_inputs(8, 4, 2, 64, [100, 30], [20, 33], 16, bf16)
    mod, c = module(64, pat, seq_dim=1), device(x)
    want = call(mod, x, c)
    with fwd.dual_level():
        assert torch.equal(call(mod, x, c), want)
        for name in ("q", "k", "v"):
            dual = {**c, name: fwd.make_dual(c[name], torch.ones_like(c[name]))}
            with pytest.raises(NotImplementedError):
                call(mod, x, dual)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call(mod, x, dual)


def test_a_wait_that_gave_up_stops_the_kernels_and_not_the_stream():
    """While the status word is set the attention call raises and writes nothing, and what follows it in the stream still
    follows what was in front of it; clearing the word restores service."""
    from dkernel_b200 import _lib, plan_paged_step
    pat = local_stride(2, 8, 2, 3)
    x = paged_inputs(8, 4, 2, 64, [100, 30], [20, 33], 16, bf16)
    out = torch.empty((53, 4, 64), dtype=bf16, device="cuda")
    mod, c = module(64, pat, seq_dim=1, impl="sm100", out=out), device(x)
    want = call(mod, x, c).clone()
    i32 = dict(dtype=torch.int32, device="cuda")
    B, W, page = 4000, 40, 16

    def state():
        return [torch.full((B, W), -1, **i32), torch.zeros(B, **i32), torch.arange(B * W, **i32), torch.tensor([B * W], **i32)]

    lens = torch.full((B,), W * page - 1, **i32)
    new = torch.ones(B, **i32)
    ref = state()
    ref_step = plan_paged_step(*ref, lens, new, page_size=page, max_new_tokens=B)
    torch.cuda.synchronize()
    assert _lib.wait_status() == 0
    assert _lib.lib().bsa_selftest_wait_timeout(1000, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    code = _lib.wait_status(reset=False)
    assert code != 0
    out.fill_(7.0)
    got = state()
    torch.cuda.synchronize()
    with pytest.raises(_lib.BsaError):
        # the step's kernel lets its successor start early
        plan_paged_step(*got, lens, new, page_size=page, max_new_tokens=B)
    with pytest.raises(_lib.BsaError):
        call(mod, x, c)
    after = [t.clone() for t in got]
    torch.cuda.synchronize()
    assert (out == 7.0).all()
    assert all(torch.equal(a, r) for a, r in zip(after, ref))
    assert _lib.wait_status() == code and _lib.wait_status() == 0
    assert torch.equal(call(mod, x, c), want)
    assert ref_step.short.item() == 0


@pytest.mark.parametrize("tokens", [1, 40])
def test_attention_right_behind_the_step(tokens):
    """The step's tables are read by a kernel that may be resident before they are written: pages change hands in every
    step, and the attention call behind it gives what it gives after a synchronisation."""
    from dkernel_b200 import plan_paged_step
    hq, hkv, d, bs, page, B, W = 8, 2, 64, 64, 16, 48, 40
    pat = local_stride(hkv, 10, 3, 4)
    mod = module(bs, pat, seq_dim=1, impl="sm100")
    i32 = dict(dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(4)
    pages = B * W
    k, v = (torch.randn((pages, page, hkv, d), generator=g).to(bf16).cuda() for _ in range(2))
    q = torch.randn((B * tokens, hq, d), generator=g).to(bf16).cuda()
    table, counts = torch.full((B, W), -1, **i32), torch.zeros(B, **i32)
    free, top = torch.randperm(pages, generator=g).to(torch.int32).cuda(), torch.tensor([pages], **i32)
    new = torch.full((B,), tokens, **i32)
    lens = torch.randint(0, W * page - tokens, (60, B), generator=g).to(torch.int32).cuda()
    lens[::3] = 0
    torch.cuda.synchronize()
    for it in range(60):
        st = plan_paged_step(table, counts, free, top, lens[it], new, page_size=page, max_new_tokens=B * tokens)
        kw = dict(block_tables=table, seqlens=st.seqlens, cu_seqlen_q=None if tokens == 1 else st.cu_seqlen_q, return_lse=True)
        got = mod(q, k, v, **kw)
        torch.cuda.synchronize()
        want = mod(q, k, v, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), it
