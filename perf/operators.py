"""The paged K/V cache and the attention that reads it, as cases that can be timed and compared.

A case is a dict of plain values; its ``kind`` names the operator:

  step     block tables, slot map and positions of a step, from the requests' lengths
  write    new keys and values into the pages, as they are or as e4m3
  attend   block-sparse attention of drafted tokens (trees, chains, single tokens) over the pages
  commit   the accepted branch of a draft tree becomes part of the context

With ``own`` false ``run`` computes the operators from elementary torch operations in fp32; with ``own`` true it
makes the calls of this package.  Lengths follow from the case alone, everything else from the seed.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0

# The pattern of the package's benchmark: 64-token blocks, a band of 16 blocks, one block column in 8.
BENCH = dict(hq=32, hkv=8, dim=128, block=64, local=16, stride=8)


def listed():
    return [
        # One user's next token over a context of some thousand tokens: the smallest call, latency counts.
        dict(name="attend_one", kind="attend", dtype="bf16", fp8=False, batch=1, lo=4001, hi=4001, draft=1, tree=False,
             page=64, max_seq=8192, **BENCH),
        # One user's draft tree: what one step of speculative decoding verifies.
        dict(name="attend_one_tree", kind="attend", dtype="bf16", fp8=False, batch=1, lo=7013, hi=7013, draft=61,
             tree=True, page=16, max_seq=8192, **BENCH),
        # Batched single-token decode at the benchmark's shape, on pages.
        dict(name="attend_tokens", kind="attend", dtype="bf16", fp8=False, batch=64, lo=1024, hi=8192, draft=1,
             tree=False, page=16, max_seq=8192 + 64, **BENCH),
        # The same batch verifying trees of up to 29 drafted tokens.
        dict(name="attend_trees", kind="attend", dtype="bf16", fp8=False, batch=64, lo=1024, hi=8100, draft=29,
             tree=True, page=64, max_seq=8192, **BENCH),
        # Wide trees on an 8-bit cache.
        dict(name="attend_trees_e4m3", kind="attend", dtype="bf16", fp8=True, batch=48, lo=1024, hi=8100, draft=60,
             tree=True, page=32, max_seq=8192, **BENCH),
        # Chains of a few drafted tokens, every head with keys of its own and a pattern of its own, narrow heads.
        dict(name="attend_chains", kind="attend", dtype="fp16", fp8=False, batch=16, lo=500, hi=16000, draft=7,
             tree=False, page=32, max_seq=16384, hq=16, hkv=16, dim=64, block=32, local=16, stride=8),
        # A serving step after admission: a handful of requests, each a few tokens.
        dict(name="step_small", kind="step", batch=16, lo=100, hi=8000, new=7, page=16, max_seq=8192, tree=True),
        # A full server: hundreds of requests, some starting with whole prompts, some finished.
        dict(name="step_large", kind="step", batch=768, lo=1, hi=16000, new=400, page=16, max_seq=16640, tree=False),
        # Keys and values of one decode step's drafts.
        dict(name="write_drafts", kind="write", dtype="bf16", fp8=False, tokens=64 * 29, hkv=8, dim=128, page=64),
        # A prompt chunk of a long document into an 8-bit cache.
        dict(name="write_prompt_e4m3", kind="write", dtype="bf16", fp8=True, tokens=65000, hkv=8, dim=128, page=32),
        # The accepted branches of a batch of trees.
        dict(name="commit_batch", kind="commit", dtype="bf16", fp8=False, batch=64, lo=100, hi=1000, draft=61, hkv=8,
             dim=128, page=16),
        # The same on a full server with an 8-bit cache.
        dict(name="commit_large_e4m3", kind="commit", dtype="bf16", fp8=True, batch=500, lo=50, hi=400, draft=64, hkv=8,
             dim=128, page=32),
    ]


# ------------------------------------------------------------------ more of the same ranges
# (q heads, kv heads, head dim)
HEADS = [(32, 8, 128), (32, 8, 128), (32, 32, 128), (16, 4, 64), (16, 16, 64), (32, 4, 128), (24, 8, 96)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "step", "write", "commit"])
    if kind == "step":
        hi = _log(rng, 100, 16000)
        c = dict(kind=kind, batch=_log(rng, 1, 768), lo=max(1, hi // rng.choice([2, 16, 100])), hi=hi,
                 new=_log(rng, 1, 400), page=rng.choice([16, 32, 64, 128]), tree=rng.random() < 0.5)
        if c["tree"]:
            c["new"] = min(c["new"], 64)
        c["max_seq"] = -(-(hi + c["new"]) // 128) * 128
        return c
    hq, hkv, dim = rng.choice(HEADS)
    fp8 = rng.random() < 0.3
    c = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16"]), fp8=fp8, hkv=hkv, dim=dim,
             page=rng.choice([16, 16, 32, 64, 128]))
    if kind == "write":
        c["tokens"] = _log(rng, 1, 65000)
        return c
    if kind == "commit":
        hi = _log(rng, 64, 1000)
        c.update(batch=_log(rng, 1, 200), lo=max(1, hi // 4), hi=hi, draft=rng.randint(1, 64))
        return c
    hi = _log(rng, 64, 50000)
    tree = rng.random() < 0.6
    draft = rng.choice([1, 1, rng.randint(2, 16), _log(rng, 16, 200)])
    c.update(hq=hq, batch=_log(rng, 1, 64), lo=max(1, hi // rng.choice([1, 2, 8])), hi=hi, tree=tree,
             draft=min(draft, 64) if tree else draft, block=rng.choice([64, 64, 64, 32, 128]),
             local=rng.choice([4, 8, 16, 32]), stride=rng.choice([4, 8, 16]))
    c["max_seq"] = -(-(hi + c["draft"]) // 512) * 512
    return c


def draw(rng):
    """One more case; drawn again while it would cost more than the largest listed ones."""
    flops = max(work(c)["flops"] for c in listed())
    while True:
        c = _draw(rng)
        # slots x kv heads x dim of the benchmark's decode cache
        if c["kind"] in ("attend", "commit") and c["batch"] * c["hi"] * c["hkv"] * c["dim"] > 64 * 8192 * 8 * 128 // 2:
            continue
        w = work(c)
        if w["flops"] <= flops and w["bytes"] <= 1e9:
            return c


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """Contexts and new tokens per request: spread over [lo, hi] in an order of their own, odd ones among them."""
    r = random.Random("%d/%d/%d" % (case["batch"], case["lo"], case["hi"]))
    ctx = [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    most = case["new"] if case["kind"] == "step" else case["draft"]
    new = [r.randint(max(1, most // 2), most) for _ in ctx]
    if case["kind"] == "step":
        for b in range(3, case["batch"], 16):      # requests that have ended give their pages back
            ctx[b] = new[b] = 0
    return ctx, new


def _trees(rng, sizes):
    """Per request: the parent of every drafted token (-1: none), and the branch that is accepted.

    The branch's tokens lie past its own length (drafts are laid out level by level, so they do where levels are
    wide), which makes committing it twice the same as committing it once."""
    parents, paths = [], []
    for n in sizes:
        c = rng.randint(1, max(1, min(8, n // 2)))
        path = sorted(rng.sample(range(c, n), c)) if n >= 2 * c else list(range(min(c, n)))
        par = [rng.randint(-1, j - 1) for j in range(n)]
        for r, j in enumerate(path):
            par[j] = path[r - 1] if r else -1
        parents.append(par)
        paths.append(path)
    return parents, paths


def _masks(parents):
    """One 64-bit word per drafted token: bit j = it attends drafted token j (its ancestors and itself)."""
    words = []
    for par in parents:
        mine = []
        for j, p in enumerate(par):
            mine.append((1 << j) | (mine[p] if p >= 0 else 0))
        words += [w - (1 << 64) if w >> 63 else w for w in mine]
    return words


def _pages_of(case, lens, rng):
    """A block table with pages in random order, and how many pages there are."""
    page = case["page"]
    counts = [-(-n // page) for n in lens]
    num = sum(counts) + 7
    order = list(range(num))
    rng.shuffle(order)
    width = max(1, -(-case["max_seq"] // page)) if "max_seq" in case else max(1, max(counts))
    rows, at = [], 0
    for c in counts:
        rows.append(order[at:at + c] + [-1] * (width - c))
        at += c
    return torch.tensor(rows, dtype=torch.int32), num, counts, order[at:]


def _cache(case, num, gen):
    shape = (num, case["page"], case["hkv"], case["dim"])
    x = torch.randn(shape, dtype=DTYPES[case["dtype"]], device="cuda", generator=gen)
    return (x * 16.0).to(E4M3) if case["fp8"] else x


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _pattern(case):
    """(kv heads, blocks, blocks) bool: a causal band of `local` blocks and, per kv head, one column in `stride`."""
    n = -(-case["max_seq"] // case["block"])
    h = torch.arange(case["hkv"], device="cuda")[:, None, None]
    i = torch.arange(n, device="cuda")[None, :, None]
    j = torch.arange(n, device="cuda")[None, None, :]
    return (j <= i) & ((i - j < case["local"]) | ((j + h + 1) % case["stride"] == 0))


def _inputs(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    s = dict(case=case)
    if kind == "write":
        T = case["tokens"]
        num = -(-T // case["page"]) + 3
        dt = DTYPES[case["dtype"]]
        shape = (T, case["hkv"], case["dim"])
        # keys and values as slices of one projection, as models compute them
        kv = torch.randn((T, 2, case["hkv"], case["dim"]), dtype=dt, device="cuda", generator=gen)
        s["k"], s["v"] = kv[:, 0], kv[:, 1]
        assert s["k"].shape == shape
        cdt = E4M3 if case["fp8"] else dt
        cache = (num, case["page"], case["hkv"], case["dim"])
        s["k_cache"] = torch.zeros(cache, dtype=torch.uint8 if case["fp8"] else dt, device="cuda").view(cdt)
        s["v_cache"] = torch.zeros(cache, dtype=torch.uint8 if case["fp8"] else dt, device="cuda").view(cdt)
        s["kv_scales"] = (0.011, 0.009) if case["fp8"] else None
        order = torch.randperm(num, device="cuda", generator=gen)
        t = torch.arange(T, device="cuda")
        s["slots"] = order[t // case["page"]] * case["page"] + t % case["page"]
        return s
    ctx, new = _lengths(case)
    s["ctx"], s["new"] = ctx, new
    s["cu"] = _cu(new)
    T = s["cu"][-1]
    total = [a + b for a, b in zip(ctx, new)]
    i32 = dict(dtype=torch.int32, device="cuda")
    s["context_lens"] = torch.tensor(ctx, **i32)
    s["cu_seqlen_q"] = torch.tensor(s["cu"], **i32)
    s["seqlens"] = torch.tensor(total, **i32)
    s["tree_mask"] = s["paths"] = None
    if kind == "commit" or case["tree"]:
        parents, s["paths"] = _trees(rng, new)
        s["masks"] = _masks(parents)
        s["tree_mask"] = torch.tensor(s["masks"], dtype=torch.int64, device="cuda")
    if kind == "step":
        # the pages that the contexts fill; requests that ended still hold some
        held = [c if t else 40 for c, t in zip(ctx, total)]
        table, num, counts, free = _pages_of(case, held, rng)
        extra = sum(-(-t // case["page"]) for t in total)
        s["block_tables"] = table.cuda()
        s["page_counts"] = torch.tensor(counts, **i32)
        stack = torch.full((num + extra,), -1, dtype=torch.int32)
        fresh = list(range(num, num + extra)) + free
        rng.shuffle(fresh)
        stack[:len(fresh)] = torch.tensor(fresh, dtype=torch.int32)
        s["free_pages"], s["num_free"] = stack.cuda(), torch.tensor([len(fresh)], **i32)
        s["new_lens"] = torch.tensor(new, **i32)
        s["tokens"] = T + 5
        if s["tree_mask"] is not None:
            s["tree_mask"] = torch.cat([s["tree_mask"], s["tree_mask"].new_zeros(5)])
        return s
    table, num, _, _ = _pages_of(case, total, rng)
    s["block_tables"] = table.cuda()
    s["k_cache"], s["v_cache"] = _cache(case, num, gen), _cache(case, num, gen)
    s["kv_scales"] = (0.0625, 0.0625) if case["fp8"] else None
    if kind == "commit":
        s["accepted"] = torch.tensor([p[-1] for p in s["paths"]], **i32)
        return s
    s["q"] = torch.randn((T, case["hq"], case["dim"]), dtype=DTYPES[case["dtype"]], device="cuda", generator=gen)
    s["pattern"] = _pattern(case)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["kind"] == "attend":
        from dkernel_b200 import SparseAttention
        s["attn"] = SparseAttention(case["block"], s["pattern"], seq_dim=1)
    return s


# ------------------------------------------------------------------ the plain forms
def _popcount(x):
    n = torch.zeros_like(x)
    for j in range(64):
        n += (x >> j) & 1
    return n


def _depths(mask, index):
    """Drafted tokens that each token attends besides itself."""
    return _popcount(mask) - ((mask >> index) & 1)


def _plain_step(s):
    case = s["case"]
    page, T, B = case["page"], s["tokens"], case["batch"]
    table, counts, stack = s["block_tables"], s["page_counts"], s["free_pages"]
    W, N = table.size(1), stack.numel()
    dev = table.device
    ctx, num_free = s["context_lens"].long(), s["num_free"].long()
    cu = torch.zeros(B + 1, dtype=torch.long, device=dev)
    cu[1:] = s["new_lens"].long().cumsum(0).clamp(max=T)
    seqlens = ctx + cu[1:] - cu[:-1]
    held = counts.long()
    target = ((seqlens + page - 1) // page).clamp(max=W)
    i = torch.arange(W, device=dev)[None]
    # give back, in request order
    back = (held - target).clamp(min=0)
    at = num_free + (back.cumsum(0) - back)[:, None] + i - target[:, None]
    gives = (i >= target[:, None]) & (i < held[:, None])
    longer = torch.cat([stack, stack.new_zeros(1)])
    longer[torch.where(gives, at, N).reshape(-1)] = table.reshape(-1)
    free = num_free + back.sum()
    # take from the top, in request order
    need = (target - held).clamp(min=0)
    start = need.cumsum(0) - need
    nth = start[:, None] + i - held[:, None]
    takes = (i >= held[:, None]) & (i < target[:, None])
    got = takes & (nth < free)
    fresh = longer[torch.where(got, free - 1 - nth, N)]
    table.copy_(torch.where(got, fresh, torch.where(takes | gives, -1, table)))
    counts.copy_(torch.where(target < held, target, held + torch.minimum((free - start).clamp(min=0), need)))
    stack.copy_(longer[:N])
    s["num_free"].copy_((free - need.sum()).clamp(min=0))
    short = (need.sum() - free).clamp(min=0)
    # slots and positions
    t = torch.arange(T, device=dev)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    real = b < B
    b = b.clamp(max=B - 1)
    index = t - cu[b]
    place = ctx[b] + index
    p = place // page
    ok = real & (p < counts[b])
    slots = torch.where(ok, table[b, p.clamp(max=W - 1)].long() * page + place % page, -1)
    depth = index if s["tree_mask"] is None else _depths(s["tree_mask"], index)
    positions = torch.where(real, ctx[b] + depth, 0)
    return [cu.int(), seqlens.int(), slots, positions.int(), short.int(), table, counts, stack, s["num_free"]]


def _plain_write(s):
    flat = lambda c: c.view(-1, *c.shape[2:])
    for x, cache, i in ((s["k"], s["k_cache"], 0), (s["v"], s["v_cache"], 1)):
        if s["kv_scales"] is not None:
            x = (x.float() / s["kv_scales"][i]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3).view(torch.uint8)
            cache = cache.view(torch.uint8)
        flat(cache)[s["slots"]] = x
    return [s["k_cache"], s["v_cache"]]


def _plain_attend(s):
    case = s["case"]
    page, bs, hq, hkv = case["page"], case["block"], case["hq"], case["hkv"]
    scale = 1.0 / math.sqrt(case["dim"])
    out = torch.empty_like(s["q"])
    dev = out.device
    for b, (L, n, t0) in enumerate(zip(s["ctx"], s["new"], s["cu"])):
        S = L + n
        pages = s["block_tables"][b, :-(-S // page)].long()
        k, v = (c.view(torch.uint8)[pages].view(E4M3) if case["fp8"] else c[pages] for c in (s["k_cache"], s["v_cache"]))
        k, v = (x.reshape(-1, hkv, case["dim"])[:S].float().permute(1, 0, 2) for x in (k, v))
        if case["fp8"]:
            k, v = k * s["kv_scales"][0], v * s["kv_scales"][1]
        i = torch.arange(n, device=dev)
        if s["tree_mask"] is None:
            among, depth = i[None, :] <= i[:, None], i
        else:
            mask = s["tree_mask"][t0:t0 + n]
            among, depth = ((mask[:, None] >> i) & 1).bool(), _depths(mask, i)
        pos = torch.cat([torch.arange(L, device=dev), L + depth])
        ok = s["pattern"][:, (L + depth) // bs][:, :, pos // bs]                  # (hkv, n, S)
        ok = ok & torch.cat([torch.ones((n, L), dtype=torch.bool, device=dev), among], 1)
        q = s["q"][t0:t0 + n].float().reshape(n, hkv, -1, case["dim"]).permute(1, 2, 0, 3)   # (hkv, G, n, d)
        x = torch.matmul(q, k[:, None].transpose(-1, -2)) * scale
        x = x.masked_fill(~ok[:, None], -math.inf)
        m = x.amax(-1, keepdim=True)
        e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
        l = e.sum(-1, keepdim=True)
        o = torch.matmul(e, v[:, None]) / torch.where(l == 0, 1.0, l)
        out[t0:t0 + n] = o.permute(2, 0, 1, 3).reshape(n, hq, -1).to(out.dtype)
    return out


def _plain_commit(s):
    case = s["case"]
    page, n = case["page"], 64
    cu, ctx, acc = s["cu_seqlen_q"].long(), s["context_lens"].long(), s["accepted"].long()
    dev = ctx.device
    word = s["tree_mask"][cu[:-1] + acc] | (torch.ones_like(acc) << acc)
    j = torch.arange(n, device=dev)
    on = ((word[:, None] >> j) & 1).bool()                       # (B, n): draft j is on the branch
    rank = on.long().cumsum(1) - 1
    b, j = (on & (rank != j)).nonzero(as_tuple=True)
    place = lambda at: s["block_tables"][b, at // page].long() * page + at % page
    src, dst = place(ctx[b] + j), place(ctx[b] + rank[b, j])
    for c in (s["k_cache"], s["v_cache"]):
        c = (c.view(torch.uint8) if case["fp8"] else c).view(-1, *c.shape[2:])
        c[dst] = c[src]
    return [s["k_cache"], s["v_cache"], (ctx + on.sum(1)).int()]


def run(state):
    s = state
    kind = s["case"]["kind"]
    if not own:
        return {"step": _plain_step, "write": _plain_write, "attend": _plain_attend, "commit": _plain_commit}[kind](s)
    import dkernel_b200 as D
    if kind == "step":
        st = D.plan_paged_step(s["block_tables"], s["page_counts"], s["free_pages"], s["num_free"], s["context_lens"],
                               s["new_lens"], page_size=s["case"]["page"], max_new_tokens=s["tokens"],
                               tree_mask=s["tree_mask"])
        return [st.cu_seqlen_q, st.seqlens, st.slots, st.positions, st.short, s["block_tables"], s["page_counts"],
                s["free_pages"], s["num_free"]]
    if kind == "write":
        D.write_paged_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], kv_scales=s["kv_scales"])
        return [s["k_cache"], s["v_cache"]]
    if kind == "attend":
        single = s["case"]["draft"] == 1
        return s["attn"](s["q"], s["k_cache"], s["v_cache"], block_tables=s["block_tables"], seqlens=s["seqlens"],
                         cu_seqlen_q=None if single else s["cu_seqlen_q"], tree_mask=None if single else s["tree_mask"],
                         kv_scales=s["kv_scales"])
    lens = D.commit_paged_draft(s["k_cache"], s["v_cache"], s["block_tables"], s["context_lens"], s["cu_seqlen_q"],
                                s["accepted"], tree_mask=s["tree_mask"])
    return [s["k_cache"], s["v_cache"], lens]


# ------------------------------------------------------------------ what cannot be left out
def _attended(case, position, head):
    """Context tokens that a query at `position` attends under kv head `head`, by counting blocks."""
    bs, local, stride = case["block"], case["local"], case["stride"]
    row = position // bs
    first = max(0, row - local + 1)
    # columns below the band with (column + head + 1) divisible by the stride
    far = (first + head) // stride - head // stride if first else 0
    return far * bs + position - first * bs


def work(case):
    kind = case["kind"]
    if kind == "write":
        n = 2 * case["tokens"] * case["hkv"] * case["dim"]
        return {"bytes": n * 2 + n * (1 if case["fp8"] else 2) + 8 * case["tokens"], "flops": n}
    ctx, new = _lengths(case)
    T, B = sum(new), case["batch"]
    if kind == "step":
        pages = sum(abs(-(-(c + n) // case["page"]) - -(-(c if c + n else 40) // case["page"])) for c, n in zip(ctx, new))
        return {"bytes": 28 * B + 8 * pages + T * (20 if case["tree"] else 12), "flops": 4 * T + 8 * B}
    size = 1 if case["fp8"] else 2
    if kind == "commit":
        # about half of the accepted tokens of each tree
        moves = sum(max(1, min(8, n // 2)) // 2 for n in new)
        return {"bytes": 4 * moves * case["hkv"] * case["dim"] * size + 24 * B, "flops": B}
    group = case["hq"] // case["hkv"]
    keys = flops = 0
    for L, n in zip(ctx, new):
        for h in range(case["hkv"]):
            seen = _attended(case, L, h)
            keys += seen + n
            flops += 4 * n * group * case["dim"] * (seen + (n + 1) // 2)
    return {"bytes": 2 * keys * case["dim"] * size + 2 * T * case["hq"] * case["dim"] * 2, "flops": flops}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def _exact_step(s):
    """Request by request, with a Python list as the stack."""
    case = s["case"]
    page, T = case["page"], s["tokens"]
    table, counts = s["block_tables"].tolist(), s["page_counts"].tolist()
    W = len(table[0])
    stack, top = s["free_pages"].tolist(), int(s["num_free"])
    cu = [min(c, T) for c in s["cu"]]
    lens = [c + cu[b + 1] - cu[b] for b, c in enumerate(s["ctx"])]
    target = [min(W, -(-n // page)) for n in lens]
    for b, row in enumerate(table):
        for i in range(target[b], counts[b]):
            stack[top] = row[i]
            row[i] = -1
            top += 1
        counts[b] = min(counts[b], target[b])
    short = 0
    for b, row in enumerate(table):
        for i in range(counts[b], target[b]):
            if top:
                top -= 1
                row[i] = stack[top]
                counts[b] += 1
            else:
                row[i] = -1
                short += 1
    slots, positions = [-1] * T, [0] * T
    for b, c in enumerate(s["ctx"]):
        for i in range(cu[b + 1] - cu[b]):
            at = c + i
            if at // page < counts[b]:
                slots[cu[b] + i] = table[b][at // page] * page + at % page
            depth = i
            if s["tree_mask"] is not None:
                word = s["masks"][cu[b] + i] & ((1 << 64) - 1)
                depth = bin(word & ~(1 << i)).count("1")
            positions[cu[b] + i] = c + depth
    return [torch.tensor(x) for x in (cu, lens, slots, positions, [short], table, counts, stack, [top])]


def _exact_write(s):
    case = s["case"]
    out = []
    for x, i in ((s["k"], 0), (s["v"], 1)):
        cache = torch.zeros(s["k_cache"].shape, dtype=torch.float64, device="cuda").view(-1, case["hkv"], case["dim"])
        x = x.double()
        if case["fp8"]:
            # the nearest e4m3 value: a step of 2^-3 of the leading power of two, 2^-9 below 2^-6; ties to even
            x = x / s["kv_scales"][i]
            power = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
            step = torch.exp2(power - 3)
            x = (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)
        cache.index_copy_(0, s["slots"], x)
        out.append(cache.view(s["k_cache"].shape))
    return out


def _exact_attend(s):
    """Head by head and request by request; the pattern by its rule, the drafts' ancestors by walking the masks."""
    case = s["case"]
    page, bs, hkv = case["page"], case["block"], case["hkv"]
    group = case["hq"] // hkv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    ks, vs = s["kv_scales"] or (1.0, 1.0)
    for b, (L, n) in enumerate(zip(s["ctx"], s["new"])):
        t0, S = s["cu"][b], L + n
        place = torch.arange(S, device="cuda")
        slot = s["block_tables"][b].long()[place // page] * page + place % page
        sees, depth = [], []
        for i in range(n):
            if s["tree_mask"] is None:
                mine = list(range(i + 1))
            else:
                word = s["masks"][t0 + i] & ((1 << 64) - 1)
                mine = [j for j in range(n) if word >> j & 1]
            sees.append(mine)
            depth.append(len(set(mine) - {i}))
        allowed = torch.zeros((n, n), dtype=torch.bool)
        for i, mine in enumerate(sees):
            allowed[i, mine] = True
        where = place.clone()
        where[L:] = L + torch.tensor(depth, device="cuda")
        col, row = where // bs, where[L:, None] // bs
        legal = torch.ones((n, S), dtype=torch.bool, device="cuda")
        legal[:, L:] = allowed.cuda()
        caches = [c.view(torch.uint8) if case["fp8"] else c for c in (s["k_cache"], s["v_cache"])]
        for h in range(hkv):
            k, v = (c.view(-1, hkv, case["dim"])[:, h][slot] for c in caches)
            if case["fp8"]:
                k, v = k.view(E4M3), v.view(E4M3)
            k, v = k.double() * ks, v.double() * vs
            see = legal & (col <= row) & ((col > row - case["local"]) | ((col + h + 1) % case["stride"] == 0))
            q = s["q"][t0:t0 + n, h * group:(h + 1) * group].double().reshape(n * group, -1)
            x = (q @ k.T).view(n, group, S) / math.sqrt(case["dim"])
            x.masked_fill_(~see[:, None], -math.inf)
            w = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
            out[t0:t0 + n, h * group:(h + 1) * group] = (w.view(n * group, S) @ v).view(n, group, -1)
    return out


def _exact_commit(s):
    case = s["case"]
    page = case["page"]
    caches = [c.double() for c in (s["k_cache"], s["v_cache"])]
    table = s["block_tables"].tolist()
    lens = []
    src, dst = [], []
    for b, path in enumerate(s["paths"]):
        L = s["ctx"][b]
        for r, j in enumerate(path):
            for at, to in ((L + j, src), (L + r, dst)):
                to.append(table[b][at // page] * page + at % page)
        lens.append(L + len(path))
    src, dst = torch.tensor(src, device="cuda"), torch.tensor(dst, device="cuda")
    for c in caches:
        flat = c.view(-1, case["hkv"], case["dim"])
        flat.index_copy_(0, dst, flat.index_select(0, src))
    return caches + [torch.tensor(lens)]


def exact(case, seed):
    s = _inputs(case, seed)
    return {"step": _exact_step, "write": _exact_write, "attend": _exact_attend, "commit": _exact_commit}[case["kind"]](s)
