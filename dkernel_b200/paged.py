"""A paged K/V cache around :class:`dkernel_b200.SparseAttention`: a step's tables, cache writes and the
commit of accepted drafts (no counterpart in the reference, whose caches are contiguous).

One step of a server that drafts tokens (speculative decoding)::

    step = plan_paged_step(block_tables, page_counts, free_pages, num_free, context_lens, new_lens,
                           page_size=16, max_new_tokens=T, tree_mask=tree_mask)
    # q, k, v of the drafted tokens at step.positions
    write_paged_kv(k, v, k_cache, v_cache, step.slots)
    out = attn(q, k_cache, v_cache, block_tables=block_tables, seqlens=step.seqlens,
               cu_seqlen_q=step.cu_seqlen_q, tree_mask=tree_mask)
    # the program compares and picks the last accepted draft of every request
    context_lens = commit_paged_draft(k_cache, v_cache, block_tables, context_lens, step.cu_seqlen_q,
                                      accepted, tree_mask=tree_mask)

Everything stays on the device and runs on the current stream; nothing synchronises, so a step can be captured
into a CUDA graph, once each call has been made outside a capture: a module's first one with given head counts reads
its pattern from the device (a pattern per query head) or refines it (blocks of 128 tokens), and keeps the result.
Pages of different requests are distinct, as ``plan_paged_step`` hands them out.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor

from . import _lib
from .ops import _FP8, _block_tables, _index32, _paged_cache, _tree_mask


class PagedStep(NamedTuple):
    """What :func:`plan_paged_step` returns, all on the device."""
    cu_seqlen_q: Tensor     # (batch + 1,) int32: first new token of each request
    seqlens: Tensor         # (batch,) int32: stored tokens per request, the new ones included
    slots: Tensor           # (max_new_tokens,) int64: where each new token's K and V go; -1 = nowhere
    positions: Tensor       # (max_new_tokens,) int32: each new token's position in its sequence
    short: Tensor           # (1,) int32: pages that the stack could not give; see plan_paged_step for tables that are too narrow


def _state32(t: Tensor, shape: Optional[Tuple[int, ...]], device_index: int, name: str) -> Tensor:
    """A tensor that is updated in place: no copy can stand in for it."""
    assert t.dtype == torch.int32 and t.get_device() == device_index and t.is_contiguous() and \
        (t.shape == shape if shape is not None else t.dim() == 1), \
        f"{name} must be contiguous int32 {shape or '1-D'} on the call's device, got {t.dtype} {tuple(t.shape)} on {t.device}"
    return t


def plan_paged_step(block_tables: Tensor, page_counts: Tensor, free_pages: Tensor, num_free: Tensor,
                    context_lens: Tensor, new_lens: Tensor, *, page_size: int, max_new_tokens: int,
                    tree_mask: Optional[Tensor] = None) -> PagedStep:
    """Block tables, slot map and positions of a step, built on the GPU from the requests' lengths.

    Request b keeps ``context_lens[b]`` tokens and gets ``new_lens[b]`` more; afterwards it holds exactly the pages
    that they need.  Surplus pages (rejected drafts; a request with both lengths 0 has ended) are pushed on the
    stack ``free_pages[:num_free]`` in the order of request and page, missing ones popped from its top in that order.
    Updated in place, all int32: ``block_tables`` (batch, pages per request), ``page_counts`` (batch,),
    ``free_pages`` (any size that holds all pages), ``num_free`` (1,).  Where the stack runs empty the table gets -1,
    the tokens have slot -1 (their keys and values are stored nowhere) and ``short`` counts the missing pages; a later step
    with the same lengths gets them once pages are free.  No page helps a request that has outgrown its row of the table:
    its tokens past the row have slot -1, too, and are not counted in ``short``; such requests are those with
    ``seqlens > block_tables.size(1) * page_size``.
    ``max_new_tokens`` is the size of the packed batch: outputs behind the last request are slot -1, position 0, and
    new tokens past it are dropped.  With ``tree_mask`` (max_new_tokens,) int64, see ``SparseAttention.forward``, a
    position is the context's length plus the number of other drafts attended, else they count up."""
    _lib.require_cuda(block_tables, "block_tables")
    dev = block_tables.get_device()
    batch = block_tables.size(0)
    _block_tables(block_tables, batch, dev)
    page_size, max_new_tokens = int(page_size), int(max_new_tokens)
    assert page_size >= 1 and max_new_tokens >= 0, f"{page_size=}, {max_new_tokens=}"
    _state32(page_counts, (batch,), dev, "page_counts")
    _state32(free_pages, None, dev, "free_pages")
    _state32(num_free, (1,), dev, "num_free")
    context_lens = _index32(context_lens, (batch,), dev, "context_lens")
    new_lens = _index32(new_lens, (batch,), dev, "new_lens")
    mask = _tree_mask(tree_mask, max_new_tokens, dev)
    # one allocation for the four int32 outputs
    ints = torch.empty(2 * batch + 2 + max_new_tokens, dtype=torch.int32, device=block_tables.device)
    cu, seqlens, short, positions = ints.split_with_sizes((batch + 1, batch, 1, max_new_tokens))
    slots = torch.empty(max_new_tokens, dtype=torch.int64, device=block_tables.device)
    p = _lib.PagedStepParams.from_buffer_copy(_lib.PAGED_STEP_PACK.pack(
        block_tables.data_ptr(), block_tables.stride(0), page_counts.data_ptr(), free_pages.data_ptr(),
        num_free.data_ptr(), context_lens.data_ptr(), new_lens.data_ptr(), _lib.ptr(mask),
        cu.data_ptr(), seqlens.data_ptr(), slots.data_ptr(), positions.data_ptr(), short.data_ptr(),
        batch, block_tables.size(1), free_pages.numel(), page_size, max_new_tokens))
    _lib.launch(_lib.lib().bsa_paged_step, p, dev, "bsa_paged_step")
    return PagedStep(cu, seqlens, slots, positions, short)


def write_paged_kv(k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, slots: Tensor, *,
                   seq_dim: Optional[int] = None, kv_scales: Optional[Tuple[float, float]] = None) -> None:
    """Stores ``k[t]`` and ``v[t]``, (tokens, kv heads, dim) with any token and head strides, in slot ``slots[t]``
    (int64, page * page size + offset) of the paged caches, (pages, page size, kv heads, dim) or, for ``seq_dim=2``,
    (pages, kv heads, page size, dim).  Slots outside the cache (-1) are skipped; slots are distinct.  Caches have k's
    type or are ``float8_e4m3fn``: then ``kv_scales = (k_scale, v_scale)`` and the cache holds ``k / k_scale`` rounded
    to nearest even and saturated at 448, ready for ``kv_scales`` of the attention call."""
    seq_dim = 1 if seq_dim is None else seq_dim
    assert seq_dim in (1, 2)
    _lib.require_cuda(k, "k")
    dev = k.get_device()
    assert v.get_device() == k_cache.get_device() == v_cache.get_device() == slots.get_device() == dev, \
        "k, v, the caches and slots must be on one device"
    pages, page_size, hkv, d, strides = _paged_cache(k_cache, v_cache, seq_dim)
    tokens = slots.size(0)
    assert slots.shape == (tokens,) and slots.dtype == torch.int64, f"slots must be 1-D int64, got {slots.dtype}"
    assert k.shape == v.shape == (tokens, hkv, d), \
        f"k and v are {tuple(k.shape)} and {tuple(v.shape)}, expected {(tokens, hkv, d)}"
    assert k.dtype == v.dtype, f"k and v dtypes differ: {k.dtype}, {v.dtype}"
    code = _lib.dtype_code(k.dtype)
    if k_cache.dtype == _FP8:
        assert kv_scales is not None and len(kv_scales) == 2, "float8_e4m3fn caches need kv_scales=(k_scale, v_scale)"
        k_scale, v_scale = float(kv_scales[0]), float(kv_scales[1])
        assert k_scale > 0 and v_scale > 0, f"kv_scales must be positive, got {kv_scales}"
        cache_code = _lib.BSA_F8E4M3
    else:
        assert kv_scales is None, "kv_scales only applies to float8_e4m3fn caches"
        assert k_cache.dtype == k.dtype, f"the caches are {k_cache.dtype}, k is {k.dtype}"
        k_scale = v_scale = 1.0
        cache_code = code
    if d > 1 and (k.stride(2) != 1 or v.stride(2) != 1):
        k, v = k.contiguous(), v.contiguous()
    if not slots.is_contiguous():
        slots = slots.contiguous()
    k_st, k_sh, _ = k.stride()
    v_st, v_sh, _ = v.stride()
    p = _lib.PagedWriteParams.from_buffer_copy(_lib.PAGED_WRITE_PACK.pack(
        k.data_ptr(), v.data_ptr(), k_st, k_sh, v_st, v_sh, k_cache.data_ptr(), v_cache.data_ptr(), *strides,
        slots.data_ptr(), tokens, hkv, d, page_size, pages, code, cache_code, k_scale, v_scale))
    _lib.launch(_lib.lib().bsa_paged_write, p, dev, "bsa_paged_write")


def commit_paged_draft(k_cache: Tensor, v_cache: Tensor, block_tables: Tensor, context_lens: Tensor,
                       cu_seqlen_q: Tensor, accepted: Tensor, *, tree_mask: Optional[Tensor] = None,
                       seq_dim: Optional[int] = None) -> Tensor:
    """The accepted branch of every request's drafts becomes part of its context.

    ``accepted[b]`` is the number of the last accepted draft of request b (-1, or any number that is not one of its
    drafts: none).  Its branch is the drafts that it attends under ``tree_mask``, and itself (without ``tree_mask``
    drafts 0..accepted[b]); their keys and values move, in the order of their numbers, to the places right behind the
    context.  The other drafts' slots hold leftovers afterwards.  Every token of the branch needs its page: one whose slot
    was -1 in the step is stored nowhere, so nothing moves to its place behind the context, which keeps what lay there, and
    it counts in the new length all the same.  Accept nothing for a request that the step left without a page.  Returns the new context lengths (int32, a new tensor;
    ``context_lens`` stays as it is).  Positions do not change, so rotated keys need nothing further."""
    seq_dim = 1 if seq_dim is None else seq_dim
    assert seq_dim in (1, 2)
    _lib.require_cuda(k_cache, "k_cache")
    dev = k_cache.get_device()
    assert v_cache.get_device() == dev, "the caches must be on one device"
    pages, page_size, hkv, d, strides = _paged_cache(k_cache, v_cache, seq_dim)
    batch = context_lens.size(0)
    context_lens = _index32(context_lens, (batch,), dev, "context_lens")
    cu_seqlen_q = _index32(cu_seqlen_q, (batch + 1,), dev, "cu_seqlen_q")
    accepted = _index32(accepted, (batch,), dev, "accepted")
    _block_tables(block_tables, batch, dev)
    total = 0x7fffffff
    if tree_mask is not None:
        total = tree_mask.size(0)
        tree_mask = _tree_mask(tree_mask, total, dev)
    code = _lib.BSA_F8E4M3 if k_cache.dtype == _FP8 else _lib.dtype_code(k_cache.dtype)
    out = torch.empty(batch, dtype=torch.int32, device=k_cache.device)
    p = _lib.PagedCommitParams.from_buffer_copy(_lib.PAGED_COMMIT_PACK.pack(
        k_cache.data_ptr(), v_cache.data_ptr(), *strides, block_tables.data_ptr(), block_tables.stride(0),
        context_lens.data_ptr(), cu_seqlen_q.data_ptr(), accepted.data_ptr(), _lib.ptr(tree_mask), out.data_ptr(),
        batch, hkv, d, total, block_tables.size(1), page_size, pages, code))
    _lib.launch(_lib.lib().bsa_paged_commit, p, dev, "bsa_paged_commit")
    return out


__all__ = ["PagedStep", "plan_paged_step", "write_paged_kv", "commit_paged_draft"]
