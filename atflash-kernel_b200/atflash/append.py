"""Paged-KV append: write new K/V tokens into a paged cache (FlashInfer's
``append_paged_kv_cache`` call shape), optionally applying RoPE to K and packing
it into the kernels' pair order on the way.

The reference's decode reads the KV cache that FlashInfer's append fills
(e2e_pipeline/atflash_e2e_fafi.py:219-223); this is that write side on the
library's own kernel (``atf_paged_kv_append``)."""
from typing import Optional, Tuple

import torch

from . import _ffi


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
    """Pages and scales of an e4m3 cache, the decode's checks (the append's are in the compiled
    binding). Returns
    (pages, page size, kv heads), the byte strides (page, token, head) and the scales
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
    pages hold the rounding of that bf16 row. There is no backward pass."""
    if isinstance(paged_kv_cache, (tuple, list)):
        kc, vc = paged_kv_cache
    else:
        kc, vc = paged_kv_cache[:, 0], paged_kv_cache[:, 1]
    cos = sin = None
    if rope is not None:
        cos, sin = rope
    _ffi.binding().append(append_key, append_value, batch_indices, positions, kc, vc, kv_indices, kv_indptr, kv_layout,
                          cos, sin, rope_positions, out_layout, kv_scales, k_norm)
