"""Contiguous forward where logits are NaN: a row that attends one is NaN, with a NaN LSE; every other row keeps its bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
bf16, f16 = torch.bfloat16, torch.float16


def _module(hq, hkv, S, bs, **kw):
    from dkernel_b200 import LocalStrideSparseAttention
    return LocalStrideSparseAttention.__wrapped__(hq, S, bs, 2, 3, num_kv_heads=hkv, seq_dim=1, impl="sm100", **kw)


@pytest.mark.parametrize("dtype", [bf16, f16])
@pytest.mark.parametrize("bs", [64, 32, 16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_query_rows_and_key_blocks(dtype, bs, D):
    if bs < 64 and D > 128:
        pytest.skip("fine blocks are served for head dims up to 128")
    B, S, hq, hkv = 2, 500, 4, 2
    mod = _module(hq, hkv, 512, bs)
    g = torch.Generator().manual_seed(7)
    q, k, v = (torch.randn((B, S, h, D), generator=g).to(dtype).cuda() for h in (hq, hkv, hkv))
    with torch.no_grad():
        clean, clean_lse = mod(q, k, v, return_lse=True)
        hit = torch.zeros((B, S, hq), dtype=torch.bool, device="cuda")
        q2 = q.clone()
        for b, s, h in ((0, 0, 1), (0, 499, 3), (1, 130, 0), (1, 64, 2)):
            q2[b, s, h, 5] = float("nan")
            hit[b, s, h] = True
        out, lse = mod(q2, k, v, return_lse=True)
    lse, clean_lse = lse.transpose(1, 2), clean_lse.transpose(1, 2)
    assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all()
    assert torch.equal(out[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])
    # a block of NaN keys: whoever attends it, first in its list or not
    from dkernel_b200 import get_sparse_attn_mask
    n = 512 // bs
    dense = get_sparse_attn_mask(hq, 512, block_size=bs, local_blocks=2, vert_stride=3, num_kv_heads=hkv)[1].bool().cuda()
    if dense.size(0) != hq:
        dense = dense.repeat_interleave(hq // dense.size(0), 0)
    for block in (0, 1, 2, n // 2, n - 2):
        k2 = k.clone()
        k2[0, block * bs:(block + 1) * bs] = float("nan")
        with torch.no_grad():
            out, lse = mod(q, k2, v, return_lse=True)
        lse = lse.transpose(1, 2)
        pos = torch.arange(S, device="cuda")
        hit = torch.zeros((B, S, hq), dtype=torch.bool, device="cuda")
        hit[0] = (dense[:, pos // bs, block] & (pos >= block * bs)[None]).T
        assert hit.any() and not hit[0].all()
        assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all()
        assert torch.equal(out[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])
