"""A norm's eps over the C interface: positive and finite, where the norm stands alone and
at an append."""
import ctypes

import pytest

from test_serving_cpu import _lib

EPS = [(0.0, -1), (-1e-6, -1), (float("nan"), -1), (float("inf"), -1), (1e39, -1), (1e-6, 0), (3e38, 0)]  # (1e39 is inf in fp32)


@pytest.mark.parametrize("eps,want", EPS)
def test_norm(eps, want):
    ffi, lib = _lib()
    p = ffi.AtfQkNormParams()
    p.q = p.q_out = p.q_weight = p.cos = p.sin = 256
    p.batch = p.num_heads_q = p.n_pos = 1  # (no tokens: nothing is launched)
    p.cs_stride_pos, p.head_dim, p.weight_dtype = 64, 128, ffi.ATF_DTYPE_F32
    p.eps = eps
    assert lib.atf_qk_norm_rope(ctypes.byref(p), None) == want


@pytest.mark.parametrize("eps,want", EPS)
@pytest.mark.parametrize("e4m3", [False, True])
def test_append(eps, want, e4m3):
    ffi, lib = _lib()
    p, n, s = ffi.AtfAppendParams(), ffi.AtfKNorm(), ffi.AtfKvScales()
    p.append_k = p.append_v = p.batch_indices = p.positions = p.k_cache = p.v_cache = p.kv_indptr = p.kv_indices = 256
    p.head_dim, p.num_kv_heads, p.page_size, p.batch_size, p.num_pages = 128, 1, 16, 1, 1
    s.k_scale = s.v_scale = p.kv_stride_token = p.cos = p.sin = n.weight = 256
    s.stride_page = s.stride_head = p.n_pos = 1
    p.cs_stride_pos, n.weight_dtype, n.eps = 64, ffi.ATF_DTYPE_F32, eps
    scales = ctypes.byref(s) if e4m3 else None
    assert lib.atf_paged_kv_append_norm(ctypes.byref(p), scales, ctypes.byref(n), None) == want
