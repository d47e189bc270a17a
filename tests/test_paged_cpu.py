"""Paged cache, what needs no GPU: the oracle against dense attention, the C ABI's checks."""
import ctypes as C
import math
import os

import numpy as np
import pytest
import torch

from oracle import paged_oracle as P
from paged_cases import local_stride, paged_inputs

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_oracle_chain_is_causal_attention():
    hq, hkv, d, bs = 4, 2, 16, 16
    pat = local_stride(hkv, 8, 2, 3)
    x = paged_inputs(1, hq, hkv, d, [37, 0], [20, 50], 8, torch.float32, tree=False)
    out, lse, _ = P.attend(x["q"], x["k"], x["v"], x["table"], x["seqlens"], pat, bs, cu=x["cu"])
    for b in range(2):
        S, n, t0 = x["seqlens"][b], x["new"][b], x["cu"][b]
        s = np.arange(S)
        slot = [(int(x["table"][b, i // 8]), i % 8) for i in s]
        k, v = (torch.stack([c[p, o] for p, o in slot]).double().repeat_interleave(2, 1) for c in (x["k"], x["v"]))
        q = x["q"][t0:t0 + n].double()
        qpos = np.arange(S - n, S)
        ok = (s[None] <= qpos[:, None])[None] & np.repeat(pat, 2, 0)[:, qpos // bs][:, :, s // bs]
        y = torch.einsum("thd,shd->hts", q, k) / math.sqrt(d)
        y = y.masked_fill(~torch.from_numpy(ok), -math.inf)
        torch.testing.assert_close(out[t0:t0 + n], torch.einsum("hts,shd->thd", y.softmax(-1), v))
        torch.testing.assert_close(lse[:, t0:t0 + n], y.logsumexp(-1))


def test_oracle_branches_are_sequences():
    """A branch of a tree gives what the sequence that it spells gives at its last token."""
    hq, hkv, d, bs = 2, 1, 16, 16
    pat = local_stride(hkv, 8, 2, 3)
    x = paged_inputs(2, hq, hkv, d, [37], [30], 8, torch.float32)
    out, lse, _ = P.attend(x["q"], x["k"], x["v"], x["table"], x["seqlens"], pat, bs, cu=x["cu"], words=x["words"])
    for leaf in (0, 7, 29):
        k, lens = P.commit(x["k"], x["table"], [37], x["cu"], [leaf], x["words"])
        v, _ = P.commit(x["v"], x["table"], [37], x["cu"], [leaf], x["words"])
        one, one_lse, _ = P.attend(x["q"][leaf:leaf + 1], k, v, x["table"], lens, pat, bs)
        torch.testing.assert_close(one[0], out[leaf])
        torch.testing.assert_close(one_lse[:, 0], lse[:, leaf])


def test_struct_layouts_match_the_header(tmp_path):
    import subprocess
    from dkernel_b200 import _lib
    names = {"bsa_paged_step_params": _lib.PagedStepParams, "bsa_paged_write_params": _lib.PagedWriteParams,
             "bsa_paged_params": _lib.PagedParams, "bsa_paged_commit_params": _lib.PagedCommitParams}
    src, body = tmp_path / "sz.c", []
    for c, py in names.items():
        body.append(f'printf("%zu ", sizeof({c}));')
        body += [f'printf("%zu ", offsetof({c}, {f}));' for f, _ in py._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "bsa.h"\nint main(void){' + "".join(body) + "return 0;}\n")
    exe = tmp_path / "sz"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    want = []
    for py in names.values():
        want += [C.sizeof(py)] + [getattr(py, f).offset for f, _ in py._fields_]
    assert got == want


def test_argument_validation_needs_no_device():
    from dkernel_b200 import _lib
    lib = _lib.lib()
    for fn, cls in ((lib.bsa_paged_fwd, _lib.PagedParams), (lib.bsa_paged_step, _lib.PagedStepParams),
                    (lib.bsa_paged_write, _lib.PagedWriteParams), (lib.bsa_paged_commit, _lib.PagedCommitParams)):
        assert fn(None, None) == -1 and b"null params" in lib.bsa_last_error()
        assert fn(C.byref(cls()), None) == -1            # all zeros
    p = _lib.PagedParams()
    p.q = p.o = p.k_cache = p.v_cache = p.crow = p.col = p.block_tables = p.seqlens = 16
    p.batch, p.hq, p.hkv, p.d, p.total_q, p.max_pages, p.page_size, p.num_pages = 1, 3, 2, 64, 1, 4, 16, 8

    def refused(text):
        assert lib.bsa_paged_fwd(C.byref(p), None) == -1
        assert text in lib.bsa_last_error(), lib.bsa_last_error()
        assert lib.bsa_paged_workspace_bytes(C.byref(p)) == 0
        assert text in lib.bsa_paged_why_not_sm100(C.byref(p))

    refused(b"multiple of hkv")
    p.hq, p.h_pat = 4, 3
    refused(b"pattern has 3 heads")
    p.h_pat, p.block_size = 2, 48
    refused(b"power of two")
    p.block_size, p.dtype, p.kv_dtype = 64, 7, 7
    refused(b"unknown dtype")
    p.dtype, p.kv_dtype = _lib.BSA_BF16, _lib.BSA_F16
    refused(b"cache has q's type")
    p.dtype, p.kv_dtype = _lib.BSA_F32, _lib.BSA_F8E4M3
    refused(b"cache has q's type")
    p.dtype, p.kv_dtype, p.total_q = _lib.BSA_BF16, _lib.BSA_BF16, 2
    refused(b"one query token per request")
    p.page_size = 0
    refused(b"bad shape")
    s = _lib.PagedStepParams()
    s.cu_seqlen_q = s.num_free = s.short_pages = s.block_tables = s.page_counts = s.context_lens = s.new_lens = s.seqlens = 16
    s.page_size, s.batch, s.max_pages = 16, 9000, 4
    assert lib.bsa_paged_step(C.byref(s), None) == -4 and b"8192" in lib.bsa_last_error()
    s.batch, s.max_pages = 8000, 1 << 20
    assert lib.bsa_paged_step(C.byref(s), None) == -4
    w = _lib.PagedWriteParams()
    w.hkv, w.d, w.page_size, w.num_pages, w.tokens, w.dtype, w.cache_dtype = 1, 8, 16, 4, 3, _lib.BSA_BF16, _lib.BSA_F8E4M3
    assert lib.bsa_paged_write(C.byref(w), None) == -1 and b"positive scales" in lib.bsa_last_error()
    w.cache_dtype = _lib.BSA_F16
    assert lib.bsa_paged_write(C.byref(w), None) == -1 and b"k's type" in lib.bsa_last_error()
    w.cache_dtype = _lib.BSA_BF16
    assert lib.bsa_paged_write(C.byref(w), None) == -1 and b"null" in lib.bsa_last_error()
    c = _lib.PagedCommitParams()
    c.hkv, c.d, c.page_size, c.batch, c.cache_dtype = 1, 8, 16, 70000, _lib.BSA_BF16
    assert lib.bsa_paged_commit(C.byref(c), None) == -1 and b"null" in lib.bsa_last_error()
    for n in ("k_cache", "v_cache", "block_tables", "context_lens", "cu_q", "accepted", "new_context_lens"):
        setattr(c, n, 16)
    assert lib.bsa_paged_commit(C.byref(c), None) == -4


def test_functions_refuse_cpu_tensors():
    from dkernel_b200 import commit_paged_draft, plan_paged_step, write_paged_kv
    t, z = torch.zeros((2, 4), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        plan_paged_step(t, z, z, z[:1], z, z, page_size=16, max_new_tokens=4)
    k = torch.zeros((2, 16, 1, 8))
    with pytest.raises(RuntimeError, match="no CPU path"):
        write_paged_kv(k[0, :2], k[0, :2], k, k, z.long())
    with pytest.raises(RuntimeError, match="no CPU path"):
        commit_paged_draft(k, k, t, z, z, z)


def test_modules_on_another_device_are_refused():
    """The layouts' pointers are read on q's device."""
    from dkernel_b200 import _lib
    from dkernel_b200.ops import _Plan, _paged_statics
    t = torch.zeros((1, 3), dtype=torch.int32)
    q = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    assert len(_paged_statics(_Plan(t, t, t, t, 64, 1), q, 2, 2, _lib.IMPL_AUTO)) == 8
    m = t.to("meta")
    with pytest.raises(AssertionError, match="the module is on meta"):
        _paged_statics(_Plan(m, m, m, m, 64, 1), q, 2, 2, _lib.IMPL_AUTO)
