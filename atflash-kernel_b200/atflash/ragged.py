"""Prefill over packed sequences of different lengths: a plan()/run() wrapper with
the names of FlashInfer's ``BatchPrefillWithRaggedKVCacheWrapper`` (its constructor
takes the device, since the kernel needs no workspace, and ``causal`` is on unless
turned off) and the ``flash_attn_varlen_func`` signature, on the windowed prefill
kernel.

The reference runs its windowed forward on one sequence at a time
(e2e_pipeline/atflash_e2e_fafi.py:119)."""
import ctypes
import math
from typing import Optional

import numpy as np
import torch

from . import _ffi, _runtime
from .prefill import WindowSpec, resolve_zhi

_LAYOUTS = {"sorted_pair": _ffi.ATF_LAYOUT_SORTED_PAIR, "rotate_half": _ffi.ATF_LAYOUT_ROTATE_HALF}


def _host_indptr(x, name: str) -> np.ndarray:
    a = x.detach().cpu().numpy() if isinstance(x, torch.Tensor) else np.asarray(x)
    if a.ndim != 1 or a.shape[0] < 2 or a.dtype.kind not in "iu":
        raise ValueError(f"{name} must be batch+1 integers")
    if a[0] != 0 or np.any(np.diff(a.astype(np.int64)) < 0) or a[-1] > 0x7fffffff:
        raise ValueError(f"{name} must start at 0, not decrease and fit 32 bits")
    return np.ascontiguousarray(a, dtype=np.int32)


class BatchPrefillWithRaggedKVCacheWrapper:
    """plan() once per batch of sequences, run() for each layer, on any stream. Sequence
    b holds the rows [qo_indptr[b], qo_indptr[b+1]) of q and [kv_indptr[b],
    kv_indptr[b+1]) of k and v; its queries are the last of its keys."""

    def __init__(self, device="cuda"):
        self._dev = torch.device(device)
        if self._dev.type != "cuda":
            raise ValueError("atflash kernels take CUDA tensors (there is no CPU path)")
        if self._dev.index is None:
            self._dev = torch.device("cuda", torch.cuda.current_device())
        self._plan = None

    def plan(self, qo_indptr, kv_indptr, num_qo_heads: int, num_kv_heads: int, head_dim: int = 128, *,
             causal: bool = True, sm_scale: Optional[float] = None, window_table: WindowSpec = None,
             qk_layout: str = "sorted_pair"):
        """Lay out the work items. The indptrs are read on the host (tensors on the
        GPU are copied, which waits for the stream)."""
        if head_dim != 128:
            raise NotImplementedError("head_dim must be 128")
        if num_kv_heads < 1 or num_qo_heads < 1 or num_qo_heads % num_kv_heads != 0:
            raise ValueError("num_qo_heads must be a multiple of num_kv_heads")
        if qk_layout not in _LAYOUTS:
            raise ValueError(f"qk_layout must be one of {sorted(_LAYOUTS)}")
        cq, ck = _host_indptr(qo_indptr, "qo_indptr"), _host_indptr(kv_indptr, "kv_indptr")
        if cq.shape != ck.shape:
            raise ValueError("qo_indptr and kv_indptr must have the same length")
        longest = int(np.diff(ck.astype(np.int64)).max())
        zhi = resolve_zhi(window_table, head_dim, longest)
        if zhi is not None and min(zhi) < 0:
            raise ValueError("zhi levels must be non-negative")
        pp = _ffi.AtfPrefillRaggedPlanParams()
        pp.batch_size, pp.causal = len(cq) - 1, 1 if causal else 0
        pp.qo_indptr_host, pp.kv_indptr_host = cq.ctypes.data, ck.ctypes.data
        n = ctypes.c_int32(0)
        lib = _ffi.load()
        _ffi.check("atf_prefill_ragged_plan", lib.atf_prefill_ragged_plan(ctypes.byref(pp), None, 0, ctypes.byref(n)))
        items = np.zeros((max(1, n.value), 8), dtype=np.int32)
        _ffi.check("atf_prefill_ragged_plan", lib.atf_prefill_ragged_plan(
            ctypes.byref(pp), items.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)), items.shape[0], ctypes.byref(n)))
        self._items = torch.from_numpy(items).to(self._dev)
        self._held = _runtime.PlanTensors(self._dev, self._items)
        t = _ffi.AtfPrefillRaggedParams()
        t.total_q, t.total_k = int(cq[-1]), int(ck[-1])
        t.num_heads_q, t.num_heads_kv, t.head_dim = num_qo_heads, num_kv_heads, head_dim
        t.items, t.num_items = self._items.data_ptr(), n.value
        t.softmax_scale = float(sm_scale) if sm_scale is not None else 1.0 / math.sqrt(head_dim)
        t.causal, t.qk_layout = pp.causal, _LAYOUTS[qk_layout]
        t.window = _ffi.ATF_WINDOW_SNAP16 if zhi is not None else _ffi.ATF_WINDOW_OFF
        for i, z in enumerate(zhi or ()):
            t.zhi[i] = z
        t.error_flag = _runtime.error_flag(self._dev).data_ptr()
        self._plan = t

    begin_forward = plan

    def run(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, out: Optional[torch.Tensor] = None,
            lse: Optional[torch.Tensor] = None, return_lse: bool = False):
        """q (total_q, Hq, 128), k / v (total_k, Hkv, 128) bf16. Returns out (total_q,
        Hq, 128) [, lse (total_q, Hq), natural log]; a row that sees no key is 0
        with an lse of -inf."""
        if self._plan is None:
            raise RuntimeError("plan() must be called before run()")
        t = self._plan
        nq, nk, hq, hkv = t.total_q, t.total_k, t.num_heads_q, t.num_heads_kv
        dev = _runtime.require_cuda(q, k, v)
        if dev != self._dev:
            raise ValueError(f"the plan is on {self._dev}, the tensors are on {dev}")
        if q.dtype != torch.bfloat16 or k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
            raise TypeError("q, k, v must be bfloat16")
        shape = (nq, hq, 128)
        if q.shape != shape or k.shape != (nk, hkv, 128) or k.shape != v.shape:
            raise ValueError(f"planned for q ({nq}, {hq}, 128) and k, v ({nk}, {hkv}, 128)")
        qst, kst, vst = q.stride(), k.stride(), v.stride()
        if qst[2] != 1 or kst[2] != 1 or vst[2] != 1:
            raise ValueError("the head_dim axis must be contiguous")
        if out is None:
            out = torch.empty(shape, dtype=torch.bfloat16, device=dev)
        elif (out.shape != shape or out.dtype != torch.bfloat16 or out.device != dev
              or out.stride(-1) != 1):
            raise ValueError(f"out must be a bf16 ({nq}, {hq}, 128) tensor on {dev} with a contiguous head_dim axis")
        if return_lse and lse is None:
            lse = torch.empty((nq, hq), dtype=torch.float32, device=dev)
        if lse is not None and (lse.shape != (nq, hq) or lse.dtype != torch.float32 or lse.device != dev
                                or not lse.is_contiguous()):
            raise ValueError(f"lse must be a contiguous float32 ({nq}, {hq}) tensor on {dev}")
        if nk == 0:  # no keys at all
            out.zero_()
            if lse is not None:
                lse.fill_(-math.inf)
        elif nq > 0:
            p = _ffi.AtfPrefillRaggedParams.from_buffer_copy(t)
            p.q, p.k, p.v, p.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
            if lse is not None:
                p.lse = lse.data_ptr()
            p.q_stride_s, p.q_stride_h, _ = qst
            p.k_stride_s, p.k_stride_h, _ = kst
            p.v_stride_s, p.v_stride_h, _ = vst
            p.o_stride_s, p.o_stride_h, _ = out.stride()
            self._held.use()
            _runtime.launch("atf_prefill_ragged_fwd", _ffi.load().atf_prefill_ragged_fwd, dev, ctypes.byref(p))
        return (out, lse) if return_lse else out

    forward = run


def flash_attn_varlen_func(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q=None, max_seqlen_k=None, dropout_p=0.0,
                           softmax_scale=None, causal=False, window_size=(-1, -1), softcap=0.0, alibi_slopes=None,
                           deterministic=False, return_attn_probs=False, block_table=None, *,
                           window_table: WindowSpec = None, qk_layout: str = "sorted_pair"):
    """flash_attn_varlen_func(q, k, v, cu_seqlens_q, cu_seqlens_k, ...) with an
    optional ATFlash window table: a plan and a run of
    ``BatchPrefillWithRaggedKVCacheWrapper`` (keep the wrapper to plan once for all
    layers: the plan reads the cu_seqlens on the host, and cost 0.05 to 0.14 ms of each
    call with 4 to 16 sequences). max_seqlen_* are accepted for call compatibility.
    Returns out, or (out, softmax_lse (Hq, total_q), None) when return_attn_probs."""
    if dropout_p != 0.0:
        raise NotImplementedError("dropout is not supported")
    if tuple(window_size) != (-1, -1):
        raise NotImplementedError("sliding-window (window_size) is not supported; use window_table")
    if softcap != 0.0 or alibi_slopes is not None or block_table is not None:
        raise NotImplementedError("softcap / alibi / block_table are not supported")
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q, k, v must be (total, heads, head_dim)")
    w = BatchPrefillWithRaggedKVCacheWrapper(_runtime.require_cuda(q, k, v))
    w.plan(cu_seqlens_q, cu_seqlens_k, q.shape[1], k.shape[1], q.shape[2], causal=causal, sm_scale=softmax_scale,
           window_table=window_table, qk_layout=qk_layout)
    res = w.run(q, k, v, return_lse=return_attn_probs)
    return (res[0], res[1].t(), None) if return_attn_probs else res
