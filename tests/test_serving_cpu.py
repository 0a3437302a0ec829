"""CPU checks of the serving-step entry points: arguments refused before a GPU is
touched, and the host schedules (units of the e4m3 decode, items of the packed
prefill) cover every key and row once within their limits."""
import ctypes
import random

import numpy as np
import pytest
import torch


def _lib():
    from atflash import _ffi
    try:
        return _ffi, _ffi.load()
    except (ImportError, OSError) as e:
        pytest.skip(f"library not built: {e}")


def test_python_refuses_cpu_tensors():
    _lib()
    import atflash
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        atflash.build_page_tables(i, i, torch.zeros((2, 2), dtype=torch.int32), 16, num_tokens=0, max_pages=0)
    k = torch.zeros((2, 1, 128), dtype=torch.bfloat16)
    c = torch.zeros((2, 16, 1, 128), dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.ones((2, 1))
    with pytest.raises(ValueError):
        atflash.append_paged_kv_cache(k, k, i, i, (c, c), i, i, kv_scales=(s, s))
    with pytest.raises(ValueError):
        atflash.BatchPrefillWithRaggedKVCacheWrapper("cpu")


def test_c_abi_refuses_bad_arguments():
    ffi, lib = _lib()
    assert lib.atf_build_page_tables(None, None) == -1
    p = ffi.AtfPageTablesParams()
    assert lib.atf_build_page_tables(ctypes.byref(p), None) == -1
    for f in ("kv_lens", "append_lens", "req_pages", "indptr", "last_page_len", "append_indptr"):
        setattr(p, f, 16)
    p.batch, p.page_size, p.num_rows, p.max_req_pages, p.req_stride = 1, 16, 1, 4, 4
    p.max_pages = 3  # without indices
    assert lib.atf_build_page_tables(ctypes.byref(p), None) == -1
    p.indices, p.req_stride = 16, 3  # rows overlap
    assert lib.atf_build_page_tables(ctypes.byref(p), None) == -1
    p.req_stride = 4
    p.free_pages = p.free_head = p.free_head_out = 16  # the head in place
    assert lib.atf_build_page_tables(ctypes.byref(p), None) == -1
    p.free_head_out, p.batch = 32, ffi.ATF_TABLES_MAX_BATCH + 1
    assert lib.atf_build_page_tables(ctypes.byref(p), None) == -2

    a, s = ffi.AtfAppendParams(), ffi.AtfKvScales()
    assert lib.atf_paged_kv_append_e4m3(None, None, None) == -1
    assert lib.atf_paged_kv_append_e4m3(ctypes.byref(a), ctypes.byref(s), None) == -1
    for f in ("append_k", "append_v", "batch_indices", "positions", "k_cache", "v_cache", "kv_indptr", "kv_indices"):
        setattr(a, f, 16)
    s.k_scale = s.v_scale = 16
    a.head_dim = 64
    assert lib.atf_paged_kv_append_e4m3(ctypes.byref(a), ctypes.byref(s), None) == -2
    a.head_dim, a.num_kv_heads, a.page_size, a.batch_size, a.num_pages, a.nnz = 128, 1, 16, 1, 1, 1
    a.k_level_major = 1
    assert lib.atf_paged_kv_append_e4m3(ctypes.byref(a), ctypes.byref(s), None) == -2
    a.k_level_major, a.cos = 0, 16  # sin missing
    assert lib.atf_paged_kv_append_e4m3(ctypes.byref(a), ctypes.byref(s), None) == -1
    a.cos, a.kv_stride_token = None, 136
    assert lib.atf_paged_kv_append_e4m3(ctypes.byref(a), ctypes.byref(s), None) == -3
    a.kv_stride_token, a.nnz = 128, 0
    assert lib.atf_paged_kv_append_e4m3(ctypes.byref(a), ctypes.byref(s), None) == 0

    d = ffi.AtfDecodeParams()
    assert lib.atf_decode_run_e4m3(ctypes.byref(d), ctypes.byref(s), None) == -1
    for f in ("q", "k_cache", "v_cache", "indptr", "indices", "last_page_len", "items", "item_indptr", "partial_o",
              "partial_lse", "out"):
        setattr(d, f, 16)
    d.head_dim, d.batch_size, d.num_qo_heads, d.num_kv_heads, d.page_size, d.num_pages = 128, 1, 2, 1, 24, 1
    assert lib.atf_decode_run_e4m3(ctypes.byref(d), ctypes.byref(s), None) == -2  # page size
    d.page_size, d.num_qo_heads = 16, 17
    assert lib.atf_decode_run_e4m3(ctypes.byref(d), ctypes.byref(s), None) == -2  # group
    d.num_qo_heads, d.window, d.qk_layout = 2, 1, 1
    assert lib.atf_decode_run_e4m3(ctypes.byref(d), ctypes.byref(s), None) == -2  # window over rotate_half
    d.qk_layout, d.window = 0, 2
    assert lib.atf_decode_run_e4m3(ctypes.byref(d), ctypes.byref(s), None) == -2  # vec8
    d.window, d.kv_stride_head = 0, 8
    assert lib.atf_decode_run_e4m3(ctypes.byref(d), ctypes.byref(s), None) == -3

    r = ffi.AtfPrefillRaggedParams()
    assert lib.atf_prefill_ragged_fwd(ctypes.byref(r), None) == -1
    for f in ("q", "k", "v", "out", "items"):
        setattr(r, f, 16)
    r.head_dim = 64
    assert lib.atf_prefill_ragged_fwd(ctypes.byref(r), None) == -2
    r.head_dim, r.total_q, r.total_k, r.num_heads_q, r.num_heads_kv = 128, 4, 4, 3, 2
    assert lib.atf_prefill_ragged_fwd(ctypes.byref(r), None) == -1
    r.num_heads_kv, r.softmax_scale, r.q_stride_s = 1, 0.1, 4
    assert lib.atf_prefill_ragged_fwd(ctypes.byref(r), None) == -3


def _units(ffi, lib, lens, page, hkv, max_chunk=0, min_chunk=0):
    B = len(lens)
    ip = np.concatenate([[0], np.cumsum([-(-n // page) for n in lens])]).astype(np.int32)
    last = np.array([(n - 1) % page + 1 if n else 0 for n in lens], dtype=np.int32)
    p = ffi.AtfDecodePlanParams()
    p.batch_size, p.num_qo_heads, p.num_kv_heads, p.head_dim, p.page_size = B, hkv, hkv, 128, page
    p.indptr_host, p.last_page_len_host, p.num_sms, p.units = ip.ctypes.data, last.ctypes.data, 148, 1
    p.max_chunk_keys, p.min_chunk_keys = max_chunk, min_chunk
    out = ffi.AtfDecodePlan()
    assert lib.atf_decode_plan(ctypes.byref(p), None, 0, None, ctypes.byref(out)) == 0
    items = np.zeros((max(1, out.num_items), 4), dtype=np.int32)
    iptr = np.zeros(B + 1, dtype=np.int32)
    i32p = ctypes.POINTER(ctypes.c_int32)
    assert lib.atf_decode_plan(ctypes.byref(p), items.ctypes.data_as(i32p), len(items), iptr.ctypes.data_as(i32p),
                               ctypes.byref(out)) == 0
    if out.num_items > 1:
        assert lib.atf_decode_plan(ctypes.byref(p), items.ctypes.data_as(i32p), out.num_items - 1,
                                   iptr.ctypes.data_as(i32p), ctypes.byref(out)) == -5
        lib.atf_decode_plan(ctypes.byref(p), items.ctypes.data_as(i32p), len(items), iptr.ctypes.data_as(i32p),
                            ctypes.byref(out))
    return items[:out.num_items], iptr


@pytest.mark.parametrize("seed", range(40))
def test_units_cover_every_key_once(seed):
    ffi, lib = _lib()
    g = random.Random(seed)
    page, hkv = g.choice([16, 32, 64, 128, 256]), g.choice([1, 2, 8, 40, 400])
    top = g.choice([1, 20, 300, 5000, 200000])
    lens = [0 if g.random() < 0.1 else g.randint(1, top) for _ in range(g.choice([1, 2, 5, 40, 300]))]
    items, iptr = _units(ffi, lib, lens, page, hkv, g.choice([0, 0, 64, 1000]), g.choice([0, 0, 500]))
    for b, n in enumerate(lens):
        at = 0
        for r in items[iptr[b]:iptr[b + 1]]:
            assert r[0] == b and r[1] == at and r[2] > r[1] and r[1] % 64 == 0
            at = r[2]
        assert at == n
    if len(items) == 0:
        return
    units = int((items[:, 3] > 0).sum())
    first = items[:units, 3] - 1
    assert first[0] == 0 and np.all(np.diff(first) > 0) and np.all(items[units:, 3] == -1)
    for lo, hi in zip(first, np.append(first[1:], len(items))):
        rows = items[lo:hi]
        assert 1 <= len(rows) <= 32
        assert sum((r[2] - 1) // page - r[1] // page + 1 for r in rows) <= 1024


def test_units_share_ragged_requests_evenly():
    ffi, lib = _lib()
    g = random.Random(1)
    lens = [20011] + [g.randint(1, 20011) for _ in range(36)]
    items, _ = _units(ffi, lib, lens, 64, 4)
    units = int((items[:, 3] > 0).sum())
    first = items[:units, 3] - 1
    assert units == 74
    cost = [sum(r[2] - r[1] + (288 if r[1] == 0 else 0) for r in items[lo:hi])
            for lo, hi in zip(first, np.append(first[1:], len(items)))]
    assert max(cost) <= sum(cost) / units + 64 + 288 and min(cost[:-1]) >= sum(cost) / units - 64 - 288


@pytest.mark.parametrize("lens,hkv", [([3] * 30, 2), ([1], 1), ([300, 64, 1], 8), ([0, 65, 0, 1000], 4)])
def test_units_of_few_keys_hold_one_item(lens, hkv):
    """What fits one wave runs side by side, not one item after another."""
    ffi, lib = _lib()
    items, _ = _units(ffi, lib, lens, 32, hkv)
    assert np.array_equal(items[:, 3], np.arange(1, len(items) + 1))
    assert len(items) <= 2 * 148 // hkv and max(items[:, 2] - items[:, 1]) <= 64


def test_units_do_not_begin_a_request_for_its_first_keys_only():
    ffi, lib = _lib()
    items, _ = _units(ffi, lib, [100] * 64, 16, 8)  # 37 units at once
    assert len(items) == 64


@pytest.mark.parametrize("seed", range(20))
def test_ragged_items_cover_every_row_once(seed):
    ffi, lib = _lib()
    g = np.random.default_rng(seed)
    nq = g.integers(0, [2, 40, 300, 3000][seed % 4], g.integers(1, 30))
    nk = nq + g.integers(-50, 500, len(nq)).clip(-nq)
    cq, ck = (np.concatenate([[0], np.cumsum(x)]).astype(np.int32) for x in (nq, nk))
    p = ffi.AtfPrefillRaggedPlanParams()
    p.batch_size, p.qo_indptr_host, p.kv_indptr_host, p.causal = len(nq), cq.ctypes.data, ck.ctypes.data, 1
    n = ctypes.c_int32(0)
    i32p = ctypes.POINTER(ctypes.c_int32)
    assert lib.atf_prefill_ragged_plan(ctypes.byref(p), None, 0, ctypes.byref(n)) == 0
    items = np.zeros((max(1, n.value), 8), dtype=np.int32)
    assert lib.atf_prefill_ragged_plan(ctypes.byref(p), items.ctypes.data_as(i32p), n.value, ctypes.byref(n)) == 0
    if n.value:
        assert lib.atf_prefill_ragged_plan(ctypes.byref(p), items.ctypes.data_as(i32p), n.value - 1, ctypes.byref(n)) in (-1, -5)
    seen = np.zeros(cq[-1], dtype=int)
    tiles = []
    for q_beg, q_len, k_beg, k_len, row, *_ in items[:n.value]:
        b = int(np.flatnonzero((cq[:-1] == q_beg) & (nq == q_len) & (ck[:-1] == k_beg) & (nk == k_len))[0])
        assert row % 256 == 0 and row < q_len and b >= 0
        seen[q_beg + row:q_beg + min(row + 256, q_len)] += 1
        tiles.append(-(-max(0, min(k_len, k_len - q_len + row + 256)) // 128))
    assert np.all(seen == 1) and tiles == sorted(tiles, reverse=True)
    bad = cq.copy()
    bad[-1] = -1
    p.qo_indptr_host = bad.ctypes.data
    assert lib.atf_prefill_ragged_plan(ctypes.byref(p), None, 0, ctypes.byref(n)) == -1
