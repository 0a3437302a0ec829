"""The append writes pages and scales: an axis that is broadcast (stride 0) is refused,
an axis of one entry may have any stride."""
import ctypes

import pytest

from test_serving_cpu import _lib


def _params(ffi):
    a, s = ffi.AtfAppendParams(), ffi.AtfKvScales()
    for f in ("append_k", "append_v", "batch_indices", "positions", "k_cache", "v_cache", "kv_indptr", "kv_indices"):
        setattr(a, f, 16)
    s.k_scale = s.v_scale = 16
    a.head_dim, a.num_kv_heads, a.page_size, a.batch_size, a.num_pages, a.nnz = 128, 2, 16, 1, 3, 0
    a.kv_stride_page, a.kv_stride_token, a.kv_stride_head = 4096, 256, 128
    s.stride_page, s.stride_head = 2, 1
    return a, s


@pytest.mark.parametrize("where,stride,axis", [
    ("s", "stride_page", "num_pages"), ("s", "stride_head", "num_kv_heads"), ("a", "kv_stride_page", "num_pages"),
    ("a", "kv_stride_head", "num_kv_heads"), ("a", "kv_stride_token", "page_size")])
def test_a_broadcast_axis_is_refused(where, stride, axis):
    ffi, lib = _lib()
    a, s = _params(ffi)
    assert lib.atf_paged_kv_append_e4m3(ctypes.byref(a), ctypes.byref(s), None) == 0
    setattr(s if where == "s" else a, stride, 0)
    assert lib.atf_paged_kv_append_e4m3(ctypes.byref(a), ctypes.byref(s), None) == -1
    setattr(a, axis, 1)
    assert lib.atf_paged_kv_append_e4m3(ctypes.byref(a), ctypes.byref(s), None) == 0
