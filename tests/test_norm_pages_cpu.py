"""CPU checks of the norms and of the shared pages: arguments refused before a GPU is
touched."""
import ctypes

import pytest
import torch

from test_serving_cpu import _lib


def test_python_refuses_cpu_tensors():
    _lib()
    import atflash
    i, t = torch.zeros(1, dtype=torch.int32), torch.zeros((1, 2), dtype=torch.int32)
    x, w, c = torch.zeros((1, 1, 128), dtype=torch.bfloat16), torch.ones(128), torch.zeros((2, 64))
    with pytest.raises(ValueError):
        atflash.qk_norm_rope(x, x, w, w, c, c)
    with pytest.raises(ValueError):
        atflash.fork_requests(i, i, i, t, 16, free_pages=i, free_head=i, shared=i)
    with pytest.raises(ValueError):
        atflash.free_requests(i, i, t, 16, free_pages=i, free_head=i)
    with pytest.raises(ValueError):
        atflash.compact_pages(i, t, 16, 1, max_moves=1, free_pages=i)
    with pytest.raises(ValueError):
        atflash.copy_pages([t], i, i)


def test_norm_refuses_bad_arguments():
    ffi, lib = _lib()
    assert lib.atf_qk_norm_rope(None, None) == -1
    p = ffi.AtfQkNormParams()
    assert lib.atf_qk_norm_rope(ctypes.byref(p), None) == -1
    p.q = p.q_out = p.q_weight = p.cos = p.sin = 256
    p.batch = p.seqlen = p.num_heads_q = p.n_pos = 1
    p.cs_stride_pos, p.head_dim, p.weight_dtype = 64, 64, ffi.ATF_DTYPE_F32
    assert lib.atf_qk_norm_rope(ctypes.byref(p), None) == -2  # head_dim 64
    p.head_dim = 128
    assert lib.atf_qk_norm_rope(ctypes.byref(p), None) == -1  # eps 0
    p.eps, p.q_stride_s = 1e-6, 3
    assert lib.atf_qk_norm_rope(ctypes.byref(p), None) == -3
    p.q_stride_s, p.q_out_stride_s = 256, 512
    assert lib.atf_qk_norm_rope(ctypes.byref(p), None) == -1  # over its input, other strides
    p.q_out_stride_s, p.cos = 256, 264
    assert lib.atf_qk_norm_rope(ctypes.byref(p), None) == -3
    p.cos, p.num_heads_k = 256, 1  # no k
    assert lib.atf_qk_norm_rope(ctypes.byref(p), None) == -1
    p.num_heads_k, p.seqlen = 0, 0
    assert lib.atf_qk_norm_rope(ctypes.byref(p), None) == 0


def test_append_norm_refuses_bad_arguments():
    ffi, lib = _lib()
    p, n, s = ffi.AtfAppendParams(), ffi.AtfKNorm(), ffi.AtfKvScales()
    p.append_k = p.append_v = p.batch_indices = p.positions = p.k_cache = p.v_cache = p.kv_indptr = p.kv_indices = 256
    p.head_dim, p.num_kv_heads, p.page_size, p.batch_size, p.num_pages = 128, 1, 16, 1, 1
    s.k_scale = s.v_scale = p.kv_stride_token = 256
    s.stride_page = s.stride_head = 1
    for scales in (None, ctypes.byref(s)):
        call = lambda: lib.atf_paged_kv_append_norm(ctypes.byref(p), scales, ctypes.byref(n), None)
        assert lib.atf_paged_kv_append_norm(ctypes.byref(p), scales, None, None) == -1
        n.weight, n.eps, n.weight_dtype = 256, 1e-6, ffi.ATF_DTYPE_F32
        p.cos = p.sin = None
        assert call() == -1  # no rotation
        p.cos = p.sin = 256
        p.cs_stride_pos, p.n_pos = 64, 1
        n.eps = 0.0
        assert call() == -1
        n.eps, n.weight_dtype = 1e-6, 7
        assert call() == -1
        n.weight_dtype, n.weight = ffi.ATF_DTYPE_BF16, 258
        assert call() == -3
        n.weight, p.cs_stride_pos = 256, 66
        assert call() == -3
        p.cs_stride_pos = 64
        assert call() == 0  # no tokens


def test_pages_refuse_bad_arguments():
    ffi, lib = _lib()
    for name, cls in (("atf_fork_requests", ffi.AtfForkParams), ("atf_free_requests", ffi.AtfFreeParams),
                      ("atf_compact_pages", ffi.AtfCompactParams)):
        fn, p = getattr(lib, name), cls()
        assert fn(None, None) == -1
        assert fn(ctypes.byref(p), None) == -1
        for f, _ in cls._fields_:
            if dict(cls._fields_)[f] is ctypes.c_void_p and f != "error_flag":
                setattr(p, f, 256)
        p.free_head_out = 512
        p.batch, p.page_size, p.num_rows, p.max_req_pages, p.req_stride = 1, 16, 1, 4, 3
        p.num_pages = p.num_free = 8
        assert fn(ctypes.byref(p), None) == -1  # rows overlap
        p.req_stride, p.page_size = 4, 0
        assert fn(ctypes.byref(p), None) == -1
        p.page_size, p.num_rows = 16, ffi.ATF_PAGES_MAX_ROWS + 1
        assert fn(ctypes.byref(p), None) == -2
        p.num_rows, p.batch = 1, ffi.ATF_TABLES_MAX_BATCH + 1
        assert fn(ctypes.byref(p), None) == -2
        p.batch, p.max_req_pages, p.req_stride = 1024, 1 << 20, 1 << 20  # 2^30 entries
        assert fn(ctypes.byref(p), None) == -2
        p.batch, p.max_req_pages, p.req_stride = 1, 4, 4
        if hasattr(p, "free_head"):
            p.free_head_out = 256  # the head in place
            assert fn(ctypes.byref(p), None) == -1
    p.num_free = 7  # the free list of a compaction holds every page
    assert lib.atf_compact_pages(ctypes.byref(p), None) == -1
    p.num_pages = p.num_free = ffi.ATF_COMPACT_MAX_PAGES + 1
    assert lib.atf_compact_pages(ctypes.byref(p), None) == -2


def test_copy_refuses_bad_arguments():
    ffi, lib = _lib()
    t = (ffi.AtfPageTensor * 1)(ffi.AtfPageTensor(256, 64, 65))
    p = ffi.AtfCopyPagesParams(ctypes.addressof(t), 1, 2, 256, 256, 1, None)
    assert lib.atf_copy_pages(None, None) == -1
    assert lib.atf_copy_pages(ctypes.byref(p), None) == -1  # pages overlap
    t[0].page_bytes, t[0].base = 64, None
    assert lib.atf_copy_pages(ctypes.byref(p), None) == -1
    t[0].base, p.src = 256, None
    assert lib.atf_copy_pages(ctypes.byref(p), None) == -1
    p.num_pairs = 0
    assert lib.atf_copy_pages(ctypes.byref(p), None) == 0
