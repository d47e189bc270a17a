"""Paged K/V cache and draft-tree attention from their definitions, on the CPU in 64 bits (test infrastructure)."""
import math

import numpy as np
import torch


def tree_word(parents, j):
    """Drafts that draft j attends: its ancestors and itself, as a set of bits."""
    w = 0
    while j >= 0:
        w |= 1 << j
        j = parents[j]
    return w


def as_int64(words):
    return torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], dtype=torch.int64)


def dequant(cache, scale=1.0):
    return cache.to(torch.float32).double() * scale if cache.dtype == torch.float8_e4m3fn else cache.double()


def slot_major(cache, seq_dim):
    """(pages, page size, kv heads, dim)."""
    return cache if seq_dim == 1 else cache.transpose(1, 2)


def attend(q, k_cache, v_cache, block_tables, seqlens, pattern, bs, *, cu=None, words=None, scale=None, kv_scales=(1.0, 1.0),
           seq_dim=1):
    """q (T, Hq, D); pattern (1 | Hkv | Hq, M, N) numpy; words: Python ints, one per query, or None for chains.
    Returns (out (T, Hq, D) float64, lse (Hq, T) float64, touched (T,) bool)."""
    q = q.double()
    T, Hq, D = q.shape
    kc, vc = (slot_major(dequant(c, s), seq_dim) for c, s in zip((k_cache, v_cache), kv_scales))
    pages, ps, Hkv, _ = kc.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    pattern = np.asarray(pattern).astype(bool)
    hp, M, N = pattern.shape
    out = torch.zeros((T, Hq, D), dtype=torch.float64)
    lse = torch.full((Hq, T), -math.inf, dtype=torch.float64)
    touched = torch.zeros(T, dtype=torch.bool)
    B = len(seqlens)
    cu = list(range(B + 1)) if cu is None else [int(x) for x in cu]
    for b in range(B):
        t0, n = cu[b], cu[b + 1] - cu[b]
        S = int(seqlens[b])
        L = S - n
        sees = []
        for i in range(n):
            if words is None:
                sees.append(set(range(i + 1)))
            else:
                sees.append({j for j in range(min(n, 64)) if words[t0 + i] >> j & 1})
        pos = [L + len(sees[i] - {i}) for i in range(n)]
        row = block_tables[b].tolist()
        where, slot = [], []
        for s in range(S):
            pi = s // ps
            pg = row[pi] if pi < len(row) else -1
            if 0 <= pg < pages:
                where.append(s)
                slot.append((pg, s % ps))
        if slot:
            pg, sl = (torch.tensor(x) for x in zip(*slot))
        for i in range(n):
            touched[t0 + i] = True
            if not slot:
                continue
            r = pos[i] // bs
            for h in range(Hq):
                kvh = h // (Hq // Hkv)
                pat = pattern[0 if hp == 1 else h if hp == Hq else kvh]
                on = []
                for s in where:
                    p = s if s < L else pos[s - L]
                    ok = s < L or (s - L) in sees[i]
                    on.append(ok and r < M and p // bs < N and bool(pat[r, p // bs]))
                on = torch.tensor(on)
                if not on.any():
                    continue
                k, v = kc[pg[on], sl[on], kvh], vc[pg[on], sl[on], kvh]
                x = (k @ q[t0 + i, h]) * scale
                lse[h, t0 + i] = torch.logsumexp(x, 0)
                out[t0 + i, h] = torch.softmax(x, 0) @ v
    return out, lse, touched


def step(block_tables, page_counts, free_pages, num_free, context_lens, new_lens, page_size, max_tokens, words=None):
    """Lists in, dict of lists out."""
    table = [list(r) for r in block_tables]
    counts, stack, top = list(page_counts), list(free_pages), num_free
    W = len(table[0]) if table else 0
    cu = [0]
    for n in new_lens:
        cu.append(min(max_tokens, cu[-1] + max(0, n)))
    ctx = [max(0, c) for c in context_lens]
    lens = [c + cu[b + 1] - cu[b] for b, c in enumerate(ctx)]
    target = [min(W, -(-n // page_size)) for n in lens]
    for b, row in enumerate(table):
        for i in range(target[b], counts[b]):
            stack[top] = row[i]
            top += 1
            row[i] = -1
        counts[b] = min(counts[b], target[b])
    short = 0
    for b, row in enumerate(table):
        for i in range(counts[b], target[b]):
            if top > 0:
                top -= 1
                row[i] = stack[top]
                counts[b] += 1
            else:
                row[i] = -1
                short += 1
    slots, positions = [-1] * max_tokens, [0] * max_tokens
    for b, c in enumerate(ctx):
        n = cu[b + 1] - cu[b]
        for i in range(n):
            t, at = cu[b] + i, c + i
            if at // page_size < counts[b]:
                slots[t] = table[b][at // page_size] * page_size + at % page_size
            depth = i
            if words is not None:
                depth = len({j for j in range(min(n, 64)) if words[t] >> j & 1} - {i})
            positions[t] = c + depth
    return dict(cu=cu, seqlens=lens, slots=slots, positions=positions, short=short, table=table, counts=counts,
                stack=stack, num_free=top)


def commit(cache, block_tables, context_lens, cu, accepted, words=None, seq_dim=1):
    """(cache with the accepted branches in place, new lengths); `cache` is not changed."""
    cache = cache.clone()
    view = slot_major(cache, seq_dim)
    pages, ps = view.shape[:2]
    lens = []

    def place(b, at):
        row = block_tables[b]
        pg = int(row[at // ps]) if at // ps < len(row) else -1
        return (pg, at % ps) if 0 <= pg < pages else None

    for b, L in enumerate(context_lens):
        n, a = cu[b + 1] - cu[b], int(accepted[b])
        if not (0 <= a < n) or (words is not None and a >= 64):
            lens.append(L)
            continue
        path = list(range(a + 1)) if words is None else sorted({j for j in range(min(n, 64)) if words[cu[b] + a] >> j & 1} | {a})
        rows = [None if (s := place(b, L + j)) is None else view[s[0], s[1]].clone() for j in path]
        for r, x in enumerate(rows):
            d = place(b, L + r)
            if x is not None and d is not None:
                view[d[0], d[1]] = x
        lens.append(L + len(path))
    return cache, lens
