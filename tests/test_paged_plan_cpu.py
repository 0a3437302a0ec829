"""The paged prefill's plan on the CPU: every (token, head, key tile) that is needed is
in exactly one item, the items stay within their limits, and the merge lists every
state of every token that has several; arguments refused before a GPU is touched."""
import ctypes
import random

import numpy as np
import pytest
import torch

from test_serving_cpu import _lib

PACKED, SPLIT = 1, 2


def _plan(reqs, hq, hkv, page, causal=1, sms=148):
    ffi, lib = _lib()
    cq = np.array([0] + list(np.cumsum([a for a, _ in reqs])), dtype=np.int32)
    npg = [-(-k // page) for _, k in reqs]
    ck = np.array([0] + list(np.cumsum(npg)), dtype=np.int32)
    last = np.array([(k - 1) % page + 1 if k else 0 for _, k in reqs], dtype=np.int32)
    p = ffi.AtfPrefillPagedPlanParams(len(reqs), hq, hkv, page, cq.ctypes.data, ck.ctypes.data, last.ctypes.data, causal, sms)
    out = ffi.AtfPrefillPagedPlan()
    assert lib.atf_prefill_paged_plan(ctypes.byref(p), None, 0, None, 0, ctypes.byref(out)) == 0
    items, rows = np.zeros((out.num_items + 1, 12), np.int32), np.zeros((out.num_rows + 1, 4), np.int32)
    i32 = ctypes.POINTER(ctypes.c_int32)
    args = (items.ctypes.data_as(i32), out.num_items, rows.ctypes.data_as(i32), out.num_rows, ctypes.byref(out))
    assert lib.atf_prefill_paged_plan(ctypes.byref(p), *args) == 0
    if out.num_items:
        short = (args[0], out.num_items - 1, *args[2:])
        assert lib.atf_prefill_paged_plan(ctypes.byref(p), *short) == -5
    return out, items[:-1], rows[:-1], cq, ck


def _check(reqs, hq, hkv, page, causal=1, sms=148):
    out, items, rows, cq, ck = _plan(reqs, hq, hkv, page, causal, sms)
    g = hq // hkv
    seen, slots = {}, {}
    for n, it in enumerate(items):
        q_tok, q_len, k_len, page_beg, row, n0, n1, flags, kt0, kt1, part, parts = (int(x) for x in it)
        b = int(np.searchsorted(cq, q_tok, side="right")) - 1
        while reqs[b][0] == 0 or cq[b] != q_tok:
            b -= 1
        nq, nk = reqs[b]
        assert (q_len, k_len, page_beg) == (nq, nk, ck[b])
        assert bool(flags & PACKED) == (n >= out.num_wide)
        top = 128 // g if flags & PACKED else 128
        assert 1 <= n0 <= top and 0 <= n1 <= top and row + n0 + n1 <= nq
        assert bool(flags & SPLIT) == (n1 == 0)
        for first, m in ((row, n0), (row + n0, n1)):
            if m:
                assert first // 128 == (first + m - 1) // 128
                end = min(nk, nk - nq + first + m) if causal else nk
                want = -(-max(0, end) // 128)
                for tok in (first, first + m - 1):
                    key = (b, tok)
                    covered = seen.setdefault(key, [])
                    covered.append((min(kt0, want), min(kt1, want)))
        for tok in range(row, row + n0 + n1):
            slot = part + (tok - row) * parts if part >= 0 else None
            slots.setdefault(cq[b] + tok, []).append(slot)
            if part >= 0:
                assert 0 <= slot < out.num_parts
    for (b, tok), cover in seen.items():
        nq, nk = reqs[b]
        at = 0
        for lo, hi in sorted(cover):
            assert lo <= at or lo == hi
            at = max(at, hi)
    assert sorted(slots) == list(range(cq[-1]))
    merged = {int(t): list(range(int(s), int(s + n))) for t, s, n, _ in rows}
    assert len(merged) == out.num_rows
    used = []
    for tok, s in slots.items():
        if s == [None]:
            assert tok not in merged
        else:
            assert sorted(s) == merged[tok] and len(s) > 1
            used += s
    assert len(set(used)) == len(used) == out.num_parts
    assert out.partial_o_floats == out.num_parts * hq * 128 and out.partial_lse_floats == out.num_parts * hq
    return out


def test_random_batches():
    rng = random.Random(0)
    for _ in range(60):
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 3, 7, 8, 16, 130])
        reqs = []
        for _ in range(rng.randint(1, 12)):
            nk = rng.choice([0, rng.randint(1, 300), rng.randint(1, 20000)])
            nq = rng.choice([0, 1, rng.randint(1, 40), rng.randint(1, 700)])
            reqs.append((nq, nk))
        _check(reqs, hq, hkv, rng.choice([16, 32, 64, 128, 256]), rng.randint(0, 1), rng.choice([0, 1, 7, 148]))


def test_long_keys_are_shared_out_and_full_machines_are_not():
    assert _check([(1, 131072)], 28, 4, 16).num_parts > 4
    assert _check([(5, 16001)] * 4, 28, 4, 16).num_parts > 0
    assert _check([(2048, 8192)] * 8, 28, 4, 16).num_parts == 0
    assert _check([(1, 100)] * 64, 24, 8, 16).num_parts == 0


def test_c_abi_refuses_bad_arguments():
    ffi, lib = _lib()
    a = (ctypes.c_int32 * 2)(0, 1)
    last = (ctypes.c_int32 * 1)(16)
    out = ffi.AtfPrefillPagedPlan()
    p = ffi.AtfPrefillPagedPlanParams(1, 4, 2, 16, ctypes.addressof(a), ctypes.addressof(a), ctypes.addressof(last), 1, 0)
    call = lambda: lib.atf_prefill_paged_plan(ctypes.byref(p), None, 0, None, 0, ctypes.byref(out))
    assert lib.atf_prefill_paged_plan(None, None, 0, None, 0, ctypes.byref(out)) == -1
    assert call() == 0
    p.page_size = 24
    assert call() == -2
    p.page_size, p.num_qo_heads = 16, 3
    assert call() == -1
    p.num_qo_heads, last[0] = 4, 17
    assert call() == -1
    last[0] = 16
    a[1] = -1
    assert call() == -1
    a[1] = 1
    assert lib.atf_prefill_paged_plan(ctypes.byref(p), None, 1, None, 0, ctypes.byref(out)) == -1
    f = ffi.AtfPrefillPagedParams()
    assert lib.atf_prefill_paged_fwd(None, None) == -1
    assert lib.atf_prefill_paged_fwd(ctypes.byref(f), None) == -1
    f.q = f.k_cache = f.v_cache = f.out = f.items = f.indices = 256
    f.total_q = f.num_pages = f.num_heads_q = f.num_heads_kv = 1
    f.head_dim, f.page_size, f.softmax_scale = 64, 16, 1.0
    assert lib.atf_prefill_paged_fwd(ctypes.byref(f), None) == -2
    f.head_dim, f.page_size = 128, 8
    assert lib.atf_prefill_paged_fwd(ctypes.byref(f), None) == -2
    f.page_size, f.softmax_scale = 16, 0.0
    assert lib.atf_prefill_paged_fwd(ctypes.byref(f), None) == -1
    f.softmax_scale, f.k_stride_token = 1.0, 3
    assert lib.atf_prefill_paged_fwd(ctypes.byref(f), None) == -3
    f.k_stride_token, f.num_parts = 8, 1  # no workspace
    assert lib.atf_prefill_paged_fwd(ctypes.byref(f), None) == -1
    f.num_parts, f.num_rows = 0, 1  # no rows
    assert lib.atf_prefill_paged_fwd(ctypes.byref(f), None) == -1
    f.num_rows, f.num_wide = 0, 1
    assert lib.atf_prefill_paged_fwd(ctypes.byref(f), None) == -1
    f.num_wide, f.window = 0, ffi.ATF_WINDOW_SNAP16
    f.zhi[0], f.zhi[1] = 1, 2  # rising levels
    assert lib.atf_prefill_paged_fwd(ctypes.byref(f), None) == -1
    f.window = ffi.ATF_WINDOW_VEC8
    assert lib.atf_prefill_paged_fwd(ctypes.byref(f), None) == -2


def test_python_refuses_cpu_tensors():
    _lib()
    import atflash
    with pytest.raises(ValueError):
        atflash.BatchPrefillWithPagedKVCacheWrapper(torch.zeros(16))
