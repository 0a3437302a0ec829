"""Paged-KV append: write new K/V tokens into a paged cache (FlashInfer's
``append_paged_kv_cache`` call shape), optionally applying RoPE to K and packing
it into the kernels' pair order on the way.

The reference's decode reads the KV cache that FlashInfer's append fills
(e2e_pipeline/atflash_e2e_fafi.py:219-223); this is that write side on the
library's own kernel (``atf_paged_kv_append``)."""
import ctypes
import warnings
from typing import Optional, Tuple

import torch

from . import _ffi, _runtime

_LAYOUTS = {"sorted_pair": _ffi.ATF_LAYOUT_SORTED_PAIR, "rotate_half": _ffi.ATF_LAYOUT_ROTATE_HALF}


def get_batch_indices_positions(append_indptr: torch.Tensor, seq_lens: torch.Tensor,
                                nnz: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Request index and KV position of each appended token. Request b appends
    append_indptr[b+1] - append_indptr[b] tokens that end its sequence of
    seq_lens[b] tokens (lengths after the append)."""
    dev = append_indptr.device
    indptr = append_indptr.to(torch.int64)
    counts = indptr[1:] - indptr[:-1]
    batch = torch.repeat_interleave(torch.arange(counts.numel(), device=dev), counts)
    offs = torch.arange(nnz, device=dev) - indptr[batch]
    pos = seq_lens.to(dev, torch.int64)[batch] - counts[batch] + offs
    return batch.to(torch.int32), pos.to(torch.int32)


def check_e4m3_cache(kc: torch.Tensor, vc: torch.Tensor, kv_scales, kv_layout: str) -> Tuple[tuple, tuple, _ffi.AtfKvScales]:
    """Pages and scales of an e4m3 cache, the checks of the decode and of an append without
    the compiled binding. Returns (pages, page size, kv heads), the byte strides (page, token, head) and the scales
    for the C call. (Sizes and strides are read once: on a short step the checks'
    host time is the call's.)"""
    if kc.dtype != torch.float8_e4m3fn or vc.dtype != torch.float8_e4m3fn:
        raise ValueError("with kv_scales the cache pages must be float8_e4m3fn")
    shape, st = kc.shape, kc.stride()
    if len(shape) != 4 or shape != vc.shape or st != vc.stride():
        raise ValueError("k and v pages must have the same 4-d shape and strides")
    if shape[3] != 128 or st[3] != 1:
        raise ValueError("the cache pages must have a contiguous head_dim of 128")
    if kv_layout == "NHD":
        size, strides = (shape[0], shape[1], shape[2]), st[:3]
    elif kv_layout == "HND":
        size, strides = (shape[0], shape[2], shape[1]), (st[0], st[2], st[1])
    else:
        raise ValueError("kv_layout must be NHD or HND")
    if not isinstance(kv_scales, (tuple, list)) or len(kv_scales) != 2:
        raise ValueError("kv_scales is (k_scales, v_scales)")
    ks, vs = kv_scales
    want, dev, ss = (size[0], size[2]), kc.device, ks.stride()
    if (ks.shape != want or vs.shape != want or ks.dtype != torch.float32 or vs.dtype != torch.float32
            or ks.device != dev or vs.device != dev):
        raise ValueError(f"k_scales and v_scales must be float32 {want} tensors (pages, kv heads) on {dev}")
    if ss != vs.stride():
        raise ValueError("k_scales and v_scales must have the same strides")
    return size, strides, _ffi.AtfKvScales(ks.data_ptr(), vs.data_ptr(), ss[0], ss[1])


def _dev_i32(t: torch.Tensor, dev: torch.device, top: int = 0x7fffffff) -> torch.Tensor:
    if t.dtype == torch.int32 and t.device == dev and t.is_contiguous():
        return t
    return _runtime.narrow_i32(t, dev, top)


def _append(k: torch.Tensor, v: torch.Tensor, batch_indices, positions, kc, vc, kv_indices, kv_indptr, kv_layout, cos, sin,
            rope_positions, out_layout, kv_scales) -> None:
    """The append over ctypes, which needs the library alone: for a Python or a torch that the
    compiled binding has not been built for. The same checks and the same kernels, but no norm."""
    if (cos is None) != (sin is None):
        raise ValueError("rope is (cos, sin)")
    dev = _runtime.require_cuda(k, v, kc, vc)
    level_major, scales = kv_scales is None and kc.dim() == 5, None
    if kv_scales is not None:
        (npages, page, hkv), strides, scales = check_e4m3_cache(kc, vc, kv_scales, kv_layout)
        if k.dim() != 3 or k.shape[2] != 128 or k.stride(2) != 1 or k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
            raise ValueError("keys and values must be (tokens, kv heads, 128) bf16 with a contiguous head_dim")
    else:
        if torch.float8_e4m3fn in (kc.dtype, vc.dtype):
            raise ValueError("float8_e4m3fn pages need kv_scales")
        for t in (k, v, vc) + (() if level_major else (kc,)):
            if t.dtype != torch.bfloat16 or t.dim() < 3 or t.stride(-1) != 1 or t.shape[-1] != 128:
                raise ValueError("keys, values and cache pages must be bf16 with a contiguous head_dim of 128")
        if k.dim() != 3:
            raise ValueError("keys and values must be (tokens, kv heads, 128)")
        if level_major:
            # (P, Hkv, 8 levels, page, 16) sorted-pair K pages (see BatchDecodeWithPagedKVCacheWrapper.run)
            if (kc.dtype != torch.bfloat16 or kc.shape[2] != 8 or kc.shape[4] != 16 or kc.stride(4) != 1
                    or kc.stride(3) != 16 or vc.dim() != 4 or kc.shape[0] != vc.shape[0]):
                raise ValueError("level-major k pages must be (P, Hkv, 8, page, 16) bf16 with 16-element rows")
            if cos is not None and out_layout != "sorted_pair":
                raise ValueError("level-major k pages hold sorted-pair K")
        elif kc.shape != vc.shape or kc.stride() != vc.stride() or kc.dim() != 4:
            raise ValueError("k and v pages must have the same 4-d shape and strides")
        if kv_layout not in ("NHD", "HND"):
            raise ValueError("kv_layout must be NHD or HND")
        tok, head = (1, 2) if kv_layout == "NHD" else (2, 1)
        npages, page, hkv = vc.shape[0], vc.shape[tok], vc.shape[head]
        strides = vc.stride(0), vc.stride(tok), vc.stride(head)
    if k.shape != v.shape or k.stride() != v.stride():
        raise ValueError("append_key and append_value must have the same shape and strides")
    nnz = k.shape[0]
    if k.shape[1] != hkv:
        raise ValueError("append_key heads do not match the cache")
    layout = _LAYOUTS[out_layout]
    if level_major and (kc.shape[1] != hkv or kc.shape[3] != page):
        raise ValueError("level-major k pages do not match the v pages")
    bi, ps = _dev_i32(batch_indices, dev), _dev_i32(positions, dev)
    ip, ix = _dev_i32(kv_indptr, dev, kv_indices.numel()), _dev_i32(kv_indices, dev)
    if bi.numel() != nnz or ps.numel() != nnz:
        raise ValueError("batch_indices and positions need one entry per appended token")
    if nnz == 0:
        return
    p = _ffi.AtfAppendParams(k.data_ptr(), v.data_ptr(), nnz, k.stride(0), k.stride(1), bi.data_ptr(), ps.data_ptr(),
                             kc.data_ptr(), vc.data_ptr(), npages, *strides, hkv, 128, page, ip.numel() - 1, ip.data_ptr(),
                             ix.data_ptr())
    p.out_layout = layout
    p.error_flag = _runtime.error_flag_ptr(dev)
    if cos is not None:
        if (cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.shape != sin.shape or cos.dim() != 2
                or cos.shape[0] < 1 or cos.shape[1] < 64 or cos.stride() != sin.stride() or cos.stride(1) != 1
                or cos.device != dev or sin.device != dev):
            raise ValueError("cos/sin must be matching fp32 (n_pos, >=64) tables")
        p.cos, p.sin, p.cs_stride_pos, p.n_pos = cos.data_ptr(), sin.data_ptr(), cos.stride(0), cos.shape[0]
        if rope_positions is not None:
            rp = rope_positions.to(device=dev, dtype=torch.int64).contiguous()
            if rp.numel() != nnz:
                raise ValueError("rope_positions needs one entry per appended token")
            p.rope_positions = rp.data_ptr()
    if level_major:
        p.k_level_major = 1
        p.k_stride_page, p.k_stride_head, p.k_stride_level = kc.stride(0), kc.stride(1), kc.stride(2)
    lib = _ffi.load()
    if scales is not None:
        _runtime.launch("atf_paged_kv_append_e4m3", lib.atf_paged_kv_append_e4m3, dev, ctypes.byref(p), ctypes.byref(scales))
    else:
        _runtime.launch("atf_paged_kv_append", lib.atf_paged_kv_append, dev, ctypes.byref(p))


def append_paged_kv_cache(append_key: torch.Tensor, append_value: torch.Tensor, batch_indices: torch.Tensor,
                          positions: torch.Tensor, paged_kv_cache, kv_indices: torch.Tensor,
                          kv_indptr: torch.Tensor, kv_last_page_len: Optional[torch.Tensor] = None,
                          kv_layout: str = "NHD", *, rope: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                          rope_positions: Optional[torch.Tensor] = None, out_layout: str = "sorted_pair",
                          kv_scales: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                          k_norm: Optional[Tuple[torch.Tensor, float]] = None) -> None:
    """append_key / append_value (nnz, Hkv, 128) bf16; token i goes to request
    batch_indices[i] at KV position positions[i]. paged_kv_cache = (k_pages,
    v_pages) or one tensor with a k/v axis at dim 1; kv_layout "NHD" or "HND".
    rope = (cos, sin) fp32 (n_pos, >=64): K is pre-RoPE in HF rotate_half order
    and is rotated at rope_positions[i] (default positions[i]) and written in
    out_layout order. Out-of-range page indices are skipped and reported by
    ``atflash.check_device_errors()`` (code 2). kv_last_page_len is accepted for
    call compatibility; positions fully determine the slots.

    kv_scales = (k_scales, v_scales), fp32 (num_pages, Hkv): the cache pages are
    float8_e4m3fn (not level-major) and each (page, kv head) has one scale, which
    the call sets for pages it begins and raises for pages it goes on filling
    (``atf_paged_kv_append_e4m3``; expanded pages or scales are refused). The tokens of
    a request are then adjacent and in position order, as ``build_page_tables`` and
    ``get_batch_indices_positions`` list them; a batch index of -1 is padding.

    k_norm = (weight, eps), with rope: each K row is RMS-normed before it is rotated, with
    128 bf16 or fp32 weights, in fp32 and rounded once to bf16, as by ``qk_norm_rope``; e4m3
    pages hold the rounding of that bf16 row. There is no backward pass.

    Without the compiled binding the call goes through ctypes, with a RuntimeWarning; k_norm
    needs the binding."""
    if isinstance(paged_kv_cache, (tuple, list)):
        kc, vc = paged_kv_cache
    else:
        kc, vc = paged_kv_cache[:, 0], paged_kv_cache[:, 1]
    cos = sin = None
    if rope is not None:
        cos, sin = rope
    try:
        binding = _ffi.binding()
    except ImportError as e:
        _ffi.load()  # (raises where it is the library that is missing)
        if k_norm is not None:
            raise
        warnings.warn(f"append_paged_kv_cache goes through ctypes, which takes longer: {e}", RuntimeWarning, stacklevel=2)
        _append(append_key, append_value, batch_indices, positions, kc, vc, kv_indices, kv_indptr, kv_layout, cos, sin,
                rope_positions, out_layout, kv_scales)
        return
    binding.append(append_key, append_value, batch_indices, positions, kc, vc, kv_indices, kv_indptr, kv_layout, cos, sin,
                   rope_positions, out_layout, kv_scales, k_norm)
