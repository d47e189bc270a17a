"""Seeded inputs for the paged-cache tests."""
import random

import numpy as np
import torch

from oracle import paged_oracle as P

E4M3 = torch.float8_e4m3fn


def local_stride(heads, blocks, local, stride):
    i, j, h = np.arange(blocks)[None, :, None], np.arange(blocks)[None, None, :], np.arange(heads)[:, None, None]
    return (j <= i) & ((i - j < local) | ((j + h + 1) % stride == 0))


def random_pattern(heads, blocks, density, seed):
    g = np.random.RandomState(seed)
    p = g.rand(heads, blocks, blocks) < density
    return p & np.tril(np.ones((blocks, blocks), bool))[None]


def random_trees(rng, sizes):
    """Per request the parents of its drafts (-1 = none); mixes chains, stars and bushes."""
    out = []
    for n in sizes:
        kind = rng.choice(["chain", "star", "any", "recent"])
        par = []
        for j in range(n):
            par.append(j - 1 if kind == "chain" else -1 if kind == "star" else
                       rng.randint(max(-1, j - 4), j - 1) if kind == "recent" else rng.randint(-1, j - 1))
        out.append(par)
    return out


def words_of(trees):
    return [P.tree_word(par, j) for par in trees for j in range(len(par))]


def paged_inputs(seed, hq, hkv, d, ctx, new, page, dtype, *, fp8=False, seq_dim=1, tree=True, spare=3, combined=False,
                 width=None):
    """CPU tensors of one attention call, and what the oracle needs beside them."""
    rng = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    total = [a + b for a, b in zip(ctx, new)]
    counts = [-(-n // page) for n in total]
    pages = sum(counts) + spare
    order = list(range(pages))
    rng.shuffle(order)
    width = max(counts + [1]) + 1 if width is None else width
    rows, at = [], 0
    for c in counts:
        rows.append(order[at:at + c] + [-1] * (width - c))
        at += c
    shape = (pages, page, hkv, d) if seq_dim == 1 else (pages, hkv, page, d)
    if combined:          # both caches in one allocation, K and V of a page side by side
        both = torch.randn((shape[0], 2) + shape[1:], generator=g).to(dtype)
        k, v = both[:, 0], both[:, 1]
    else:
        both = None
        k, v = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)
    kv_scales = None
    if fp8:
        k, v, kv_scales = (k.float() * 16).to(E4M3), (v.float() * 16).to(E4M3), (0.0625, 0.05)
    T = sum(new)
    q = torch.randn((T, hq, d), generator=g).to(dtype)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    trees = random_trees(rng, new) if tree else None
    return dict(q=q, k=k, v=v, both=both, table=torch.tensor(rows, dtype=torch.int32), seqlens=total, cu=cu,
                words=words_of(trees) if tree else None, trees=trees, kv_scales=kv_scales, ctx=list(ctx), new=list(new),
                page=page, seq_dim=seq_dim)


def logit_error(x, d, scale):
    """Bound on a logit's error in fp32: d products and sums, 2^-24 each, of at most |q||k|."""
    kc = P.dequant(x["k"], (x["kv_scales"] or (1.0, 1.0))[0])
    finite = torch.where(torch.isfinite(kc), kc, 0.0)
    qf = x["q"].double()
    qn, kn = qf.norm(dim=-1).max().item() if qf.numel() else 0.0, finite.norm(dim=-1).max().item() if finite.numel() else 0.0
    return (d + 4) * 2.0 ** -24 * qn * kn * abs(scale)


def check_attention(got, lse, ref, ref_lse, x, d, scale):
    """Rounding of the output to its type (half a step), the logits' error, and 2^-15 for weights that are kept as
    two 16-bit terms and for the approximate exponential (2^-22 each)."""
    e = logit_error(x, d, scale)
    vf = P.dequant(x["v"], (x["kv_scales"] or (1.0, 1.0))[1])
    vmax = torch.where(torch.isfinite(vf), vf, 0.0).abs().max().item() if vf.numel() else 0.0
    eps = torch.finfo(got.dtype).eps
    tiny = torch.finfo(got.dtype).tiny * eps          # half a step among subnormals
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    bound = eps / 2 * ref.abs() * (1 + 2.0 ** -7) + (4 * e + 2.0 ** -15) * vmax + tiny
    over = (got - ref).abs() - bound
    assert over.max().item() <= 0 if over.numel() else True, f"off by {(got - ref).abs().max().item():.3e}"
    if lse is not None:
        lse = lse.double().cpu()
        gone = torch.isinf(ref_lse)
        assert torch.equal(torch.isinf(lse) & (lse < 0), gone)
        d_lse = (lse - ref_lse)[~gone].abs()
        # 2^-22 of the LSE itself, for its rounding and the logarithm
        lim = 2 * e + 2.0 ** -20 + 2.0 ** -22 * ref_lse[~gone].abs()
        assert (d_lse <= lim).all() if d_lse.numel() else True, f"LSE off by {d_lse.max().item():.3e}"
