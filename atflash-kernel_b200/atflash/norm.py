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
_ROW, _ONE = (128,), (1,)
_WEIGHTS = {torch.bfloat16: _ffi.ATF_DTYPE_BF16, torch.float32: _ffi.ATF_DTYPE_F32}


def check_norm(weight: torch.Tensor, eps: float, dev: torch.device, name: str) -> int:
    """Checks a norm's weights and eps; returns the weights' ATF_DTYPE."""
    dtype = _WEIGHTS.get(weight.dtype)
    if dtype is None or weight.shape != _ROW or weight.stride() != _ONE or weight.device != dev:
        raise ValueError(f"{name} must be 128 contiguous bf16 or fp32 weights on {dev}")
    if not 1e-38 <= eps < math.inf:  # (a normal fp32 number)
        raise ValueError("the norm's eps must be a positive number")
    return dtype


def refuse_gradients(*tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("atflash has no backward pass: call it under torch.no_grad() or with detached tensors")


def _heads(x: torch.Tensor, name: str) -> Tuple[torch.Size, Tuple[int, int, int]]:
    """The shape of a (B, S, H, 128) or (T, H, 128) tensor and its strides (batch, token, head)."""
    shape, st = x.shape, x.stride()
    n = len(shape)
    if x.dtype != torch.bfloat16 or (n != 3 and n != 4) or shape[-1] != 128 or st[-1] != 1:
        raise ValueError(f"{name} must be (B, S, H, 128) or (T, H, 128) bf16 with a contiguous last axis")
    return shape, ((0, st[0], st[1]) if n == 3 else st[:3])


def _output(out: torch.Tensor, x: torch.Tensor, name: str) -> Tuple[int, int, int]:
    """Checks a caller's output; returns its strides (batch, token, head)."""
    shape, st = out.shape, out.stride()
    if shape != x.shape or out.dtype != torch.bfloat16 or out.device != x.device or st[-1] != 1:
        raise ValueError(f"{name} must be a bf16 {tuple(x.shape)} tensor on {x.device} with a contiguous last axis")
    if any(n > 1 and s == 0 for n, s in zip(shape, st)):
        raise ValueError(f"{name} must not be expanded: its rows are written")
    if out.data_ptr() == x.data_ptr() and st != x.stride() and out.numel() > 0:
        raise ValueError(f"{name} over its own input needs the input's strides")
    return (0, st[0], st[1]) if len(shape) == 3 else st[:3]


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
    shape, qst = _heads(q, "q")
    tokens = shape[:-2]
    B, S = tokens if len(tokens) == 2 else (1, tokens[0])
    wt = check_norm(q_weight, eps, dev, "q_weight")
    layout = _LAYOUTS.get(out_layout)
    if layout is None:
        raise ValueError(f"out_layout must be one of {sorted(_LAYOUTS)}")
    csh, cst = cos.shape, cos.stride()
    if (cos.dtype != torch.float32 or sin.dtype != torch.float32 or len(csh) != 2 or csh != sin.shape or csh[0] < 1
            or csh[1] < 64 or cst != sin.stride() or cst[1] != 1):
        raise ValueError("cos/sin must be matching fp32 (n_pos, >=64) tables with a contiguous last axis")
    if q_out is None:
        q_out = torch.empty_like(q)
        st = q_out.stride()
        ost = (0, st[0], st[1]) if len(st) == 3 else st[:3]
    else:
        ost = _output(q_out, q, "q_out")
    k_ptr = k_out_ptr = k_w = hk = 0
    kst = kost = (0, 0, 0)
    if k is not None:
        if k.device != dev:
            raise ValueError("all tensors must be on the same device")
        kshape, kst = _heads(k, "k")
        if kshape[:-2] != tokens:
            raise ValueError("q and k must hold the same tokens")
        if check_norm(k_weight, eps, dev, "k_weight") != wt:
            raise ValueError("q_weight and k_weight must have the same type")
        if k_out is None:
            k_out = torch.empty_like(k)
            st = k_out.stride()
            kost = (0, st[0], st[1]) if len(st) == 3 else st[:3]
        else:
            kost = _output(k_out, k, "k_out")
        k_ptr, k_out_ptr, k_w, hk = k.data_ptr(), k_out.data_ptr(), k_weight.data_ptr(), kshape[-2]
    pos, pos64, pst = 0, 0, (0, 0)
    if positions is not None:
        ps = positions.shape
        if (positions.dtype not in (torch.int32, torch.int64) or positions.device != dev
                or (ps != tokens and ps != (S,))):
            raise ValueError(f"positions must be int32 or int64 on {dev}, one per token")
        st = positions.stride()
        pos, pos64 = positions.data_ptr(), 1 if positions.dtype == torch.int64 else 0
        pst = (0, st[0]) if len(ps) == 1 else st
    if B * S > 0:  # (tensors without tokens have no address)
        p = _ffi.AtfQkNormParams(
            q.data_ptr(), k_ptr, q_out.data_ptr(), k_out_ptr, B, S, shape[-2], hk, 128, *qst, *kst, *ost, *kost,
            q_weight.data_ptr(), k_w, wt, eps, cos.data_ptr(), sin.data_ptr(),
            # (the only row's stride is any)
            cst[0] if csh[0] > 1 else max(64, cst[0] & ~3), csh[0], pos, pos64, *pst, int(pos_offset), layout)
        _runtime.launch("atf_qk_norm_rope", _ffi.load().atf_qk_norm_rope, dev, ctypes.byref(p))
    return q_out, k_out
