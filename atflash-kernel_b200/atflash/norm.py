"""RMS norms of the query and key heads with the RoPE rotation in the same pass
(``atf_qk_norm_rope``), for models that norm each head between projection and rotation.
``append_paged_kv_cache(k_norm=...)`` does the same to K on its way into a cache.

The reference's models have no such norms."""
import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _ffi, _runtime

_LAYOUTS = {"sorted_pair": _ffi.ATF_LAYOUT_SORTED_PAIR, "rotate_half": _ffi.ATF_LAYOUT_ROTATE_HALF}
_WEIGHTS = {torch.bfloat16: _ffi.ATF_DTYPE_BF16, torch.float32: _ffi.ATF_DTYPE_F32}


def check_norm(weight: torch.Tensor, eps: float, dev: torch.device, name: str) -> int:
    """Checks a norm's weights and eps; returns the weights' ATF_DTYPE."""
    dtype = _WEIGHTS.get(weight.dtype)
    if dtype is None or weight.shape != (128,) or weight.stride(0) != 1 or weight.device != dev:
        raise ValueError(f"{name} must be 128 contiguous bf16 or fp32 weights on {dev}")
    if not (eps > 0.0 and math.isfinite(eps) and ctypes.c_float(eps).value > 0.0):
        raise ValueError("the norm's eps must be a positive number")
    return dtype


def refuse_gradients(*tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("atflash has no backward pass: call it under torch.no_grad() or with detached tensors")


def _heads(x: torch.Tensor, name: str) -> Tuple[int, int, int, Tuple[int, int, int]]:
    """(batch, seqlen, heads) and the strides of a (B, S, H, 128) or (T, H, 128) tensor."""
    shape, st = x.shape, x.stride()
    if x.dtype != torch.bfloat16 or len(shape) not in (3, 4) or shape[-1] != 128 or st[-1] != 1:
        raise ValueError(f"{name} must be (B, S, H, 128) or (T, H, 128) bf16 with a contiguous last axis")
    if len(shape) == 3:
        return 1, shape[0], shape[1], (0, st[0], st[1])
    return shape[0], shape[1], shape[2], st[:3]


def _output(out: Optional[torch.Tensor], x: torch.Tensor, name: str) -> torch.Tensor:
    if out is None:
        return torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    if out.shape != x.shape or out.dtype != torch.bfloat16 or out.device != x.device or out.stride(-1) != 1:
        raise ValueError(f"{name} must be a bf16 {tuple(x.shape)} tensor on {x.device} with a contiguous last axis")
    if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
        raise ValueError(f"{name} must not be expanded: its rows are written")
    if out.data_ptr() == x.data_ptr() and out.stride() != x.stride() and out.numel() > 0:
        raise ValueError(f"{name} over its own input needs the input's strides")
    return out


def qk_norm_rope(q: torch.Tensor, k: Optional[torch.Tensor], q_weight: torch.Tensor, k_weight: Optional[torch.Tensor],
                 cos: torch.Tensor, sin: torch.Tensor, *, eps: float = 1e-6, pos_offset: int = 0,
                 positions: Optional[torch.Tensor] = None, out_layout: str = "rotate_half",
                 q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None):
    """Norm each head of q and k and rotate it: y = x w / sqrt(mean(x^2) + eps) over the 128
    elements, then RoPE of y in HF rotate_half order, in fp32 and rounded once to bf16,
    written in `out_layout` order ("rotate_half" or "sorted_pair"). Returns (q_out, k_out).

    q (B, S, Hq, 128) and k (B, S, Hk, 128), or packed tokens (T, H, 128); any strides that
    are multiples of 8 elements, so slices of one qkv projection are read in place. k and
    k_weight may be None (the append norms K itself, with ``k_norm``): k_out is then
    None. Weights: 128 bf16 or fp32, both of one type. positions: integers (S,) or (B, S), or
    (T,); default pos_offset + s; positions outside the tables are clamped into them, as
    by ``rope_pack``. q_out may be q and k_out may be k (in place); otherwise outputs overlap
    no input. There is no backward pass."""
    if (k is None) != (k_weight is None) or (k is None and k_out is not None):
        raise ValueError("k and k_weight go together")
    refuse_gradients(q, k, q_weight, k_weight)
    dev = _runtime.require_cuda(q, cos, sin)
    B, S, hq, qst = _heads(q, "q")
    wt = check_norm(q_weight, eps, dev, "q_weight")
    if out_layout not in _LAYOUTS:
        raise ValueError(f"out_layout must be one of {sorted(_LAYOUTS)}")
    csh, cst = cos.shape, cos.stride()
    if (cos.dtype != torch.float32 or sin.dtype != torch.float32 or len(csh) != 2 or csh != sin.shape or csh[0] < 1
            or csh[1] < 64 or cst != sin.stride() or cst[1] != 1):
        raise ValueError("cos/sin must be matching fp32 (n_pos, >=64) tables with a contiguous last axis")
    q_out = _output(q_out, q, "q_out")
    p = _ffi.AtfQkNormParams()
    p.q, p.q_out, p.q_weight = q.data_ptr(), q_out.data_ptr(), q_weight.data_ptr()
    p.batch, p.seqlen, p.num_heads_q, p.head_dim = B, S, hq, 128
    p.q_stride_b, p.q_stride_s, p.q_stride_h = qst
    _, _, _, ost = _heads(q_out, "q_out")
    p.q_out_stride_b, p.q_out_stride_s, p.q_out_stride_h = ost
    if k is not None:
        if k.device != dev:
            raise ValueError("all tensors must be on the same device")
        kb, ks, hk, kst = _heads(k, "k")
        if (kb, ks) != (B, S) or k.dim() != q.dim():
            raise ValueError("q and k must hold the same tokens")
        if check_norm(k_weight, eps, dev, "k_weight") != wt:
            raise ValueError("q_weight and k_weight must have the same type")
        k_out = _output(k_out, k, "k_out")
        p.k, p.k_out, p.k_weight, p.num_heads_k = k.data_ptr(), k_out.data_ptr(), k_weight.data_ptr(), hk
        p.k_stride_b, p.k_stride_s, p.k_stride_h = kst
        _, _, _, ost = _heads(k_out, "k_out")
        p.k_out_stride_b, p.k_out_stride_s, p.k_out_stride_h = ost
    p.weight_dtype, p.eps, p.out_layout = wt, eps, _LAYOUTS[out_layout]
    p.cos, p.sin, p.cs_stride_pos, p.n_pos = cos.data_ptr(), sin.data_ptr(), cst[0], csh[0]
    p.pos_offset = int(pos_offset)
    if positions is not None:
        ps = positions.shape
        if (positions.dtype not in (torch.int32, torch.int64) or positions.device != dev
                or (ps != (S,) and (q.dim() == 3 or ps != (B, S)))):
            raise ValueError(f"positions must be int32 or int64 on {dev}, one per token")
        st = positions.stride()
        p.positions, p.positions_64 = positions.data_ptr(), 1 if positions.dtype == torch.int64 else 0
        p.pos_stride_b, p.pos_stride_s = (0, st[0]) if len(ps) == 1 else st
    if csh[0] == 1:
        p.cs_stride_pos = max(64, cst[0] & ~3)  # the only row's stride is any
    if B * S > 0:  # (tensors without tokens have no address)
        _runtime.launch("atf_qk_norm_rope", _ffi.load().atf_qk_norm_rope, dev, ctypes.byref(p))
    return q_out, k_out
