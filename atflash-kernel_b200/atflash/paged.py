"""Attention of new tokens over a paged cache: a plan()/run() wrapper whose plan takes the
arguments of the decode's and the packed prefill's together, with ATFlash windows. One batch may hold decodes (one token), drafted tokens to verify (a few)
and chunks of prompts behind what their requests, or the requests they were forked
from, have in the cache.

The reference prefills over contiguous K and V (e2e_pipeline/atflash_e2e_fafi.py:119)."""
import ctypes
import math
from typing import Optional

import numpy as np
import torch

from . import _ffi, _runtime
from .prefill import WindowSpec, resolve_zhi
from .ragged import _host_indptr

_LAYOUTS = ("sorted_pair", "rotate_half")


class BatchPrefillWithPagedKVCacheWrapper:
    """plan() once per step, run() for each layer, on any stream (runs share the workspace, so
    those of one wrapper, and its captured graphs, follow one another). Request b's new tokens are the rows
    [qo_indptr[b], qo_indptr[b+1]) of q; they are the last of its tokens, whose K and V are
    all in its pages (append them first).

    A window is quantised as in the packed prefill, per tile of 128 queries, counted from the
    request's first new token, and 128 keys: a level counts where any pair of the tile is within
    its reach. So the scores of a token depend on where its chunk begins, and a request of one
    token keeps levels of some keys that ``BatchDecodeWithPagedKVCacheWrapper``, which goes by each
    key's own distance, drops (never the other way round). Chunks that begin on multiples of 128
    tokens keep what the whole prompt in one chunk keeps."""

    def __init__(self, float_workspace_buffer: torch.Tensor, kv_layout: str = "NHD"):
        if kv_layout not in ("NHD", "HND"):
            raise ValueError("kv_layout must be NHD or HND")
        if not float_workspace_buffer.is_cuda:
            raise ValueError("the workspace buffer must be a CUDA tensor")
        if not float_workspace_buffer.is_contiguous():
            raise ValueError("the workspace buffer must be contiguous")
        self._ws = float_workspace_buffer
        self._dev = float_workspace_buffer.device
        self._kv_layout = kv_layout
        self._plan = self._planned = None

    def plan(self, qo_indptr, paged_kv_indptr, paged_kv_indices, paged_kv_last_page_len, num_qo_heads: int,
             num_kv_heads: int, head_dim: int, page_size: int, *, causal: bool = True, sm_scale: Optional[float] = None,
             window_table: WindowSpec = None, qk_layout: str = "sorted_pair"):
        """Lay out the work items. qo_indptr, paged_kv_indptr and paged_kv_last_page_len are read on
        the host (tensors on the GPU are copied, which waits for the stream);
        paged_kv_indices may be a GPU tensor or a list, and is kept with the plan. Pages of 16, 32,
        64, 128 or 256 tokens. A window needs sorted pairs; without one, q and the cached K
        may have either pair order. `causal` is on unless turned off. The states of tokens
        whose keys are shared out over several SMs lie in the workspace buffer; a
        ValueError says how much a plan needs."""
        if head_dim != 128:
            raise NotImplementedError("head_dim must be 128")
        if num_kv_heads < 1 or num_qo_heads < 1 or num_qo_heads % num_kv_heads != 0:
            raise ValueError("num_qo_heads must be a multiple of num_kv_heads")
        if page_size not in (16, 32, 64, 128, 256):
            raise NotImplementedError("pages of 16, 32, 64, 128 or 256 tokens")
        if qk_layout not in _LAYOUTS:
            raise ValueError(f"qk_layout must be one of {sorted(_LAYOUTS)}")
        if window_table is not None and qk_layout != "sorted_pair":
            raise NotImplementedError("a window needs sorted pairs")
        cq, ck = _host_indptr(qo_indptr, "qo_indptr"), _host_indptr(paged_kv_indptr, "paged_kv_indptr")
        if cq.shape != ck.shape:
            raise ValueError("qo_indptr and paged_kv_indptr must have the same length")
        last = paged_kv_last_page_len
        last = np.asarray(last.detach().cpu().numpy() if isinstance(last, torch.Tensor) else last)
        pages = np.diff(ck.astype(np.int64))
        if last.shape != pages.shape or last.dtype.kind not in "iu":
            raise ValueError("paged_kv_last_page_len must be one integer per request")
        if np.any((pages > 0) & ((last < 1) | (last > page_size))):
            raise ValueError("last_page_len must be between 1 and page_size")
        last = np.ascontiguousarray(np.where(pages > 0, last, 0), dtype=np.int32)
        longest = int(((pages - 1) * page_size + last).max()) if pages.max() > 0 else 1
        if longest >= 1 << 30:
            raise NotImplementedError("fewer than 2^30 tokens per request")
        idx = paged_kv_indices if isinstance(paged_kv_indices, torch.Tensor) else torch.tensor(paged_kv_indices,
                                                                                              dtype=torch.int64)
        if idx.dim() != 1 or idx.dtype not in (torch.int32, torch.int64) or idx.numel() < int(ck[-1]):
            raise ValueError("paged_kv_indices must be a 1-d integer tensor of indptr[-1] entries or more")
        scale = float(sm_scale) if sm_scale is not None else 1.0 / math.sqrt(head_dim)
        if not (scale > 0.0 and math.isfinite(scale)):
            raise ValueError("sm_scale must be a positive number")
        zhi = resolve_zhi(window_table, head_dim, longest)
        if zhi is not None and min(zhi) < 0:
            raise ValueError("zhi levels must be non-negative")
        pp = _ffi.AtfPrefillPagedPlanParams(len(cq) - 1, num_qo_heads, num_kv_heads, page_size, cq.ctypes.data,
                                            ck.ctypes.data, last.ctypes.data, 1 if causal else 0,
                                            torch.cuda.get_device_properties(self._dev).multi_processor_count)
        lib, P, i32p = _ffi.load(), _ffi.AtfPrefillPagedPlan(), ctypes.POINTER(ctypes.c_int32)
        _ffi.check("atf_prefill_paged_plan", lib.atf_prefill_paged_plan(ctypes.byref(pp), None, 0, None, 0, ctypes.byref(P)))
        n, m = P.num_items * _ffi.ATF_PAGED_ITEM_INTS, 4 * P.num_rows
        buf = np.zeros(max(4, n + m), dtype=np.int32)  # the items, then the rows: one copy
        _ffi.check("atf_prefill_paged_plan", lib.atf_prefill_paged_plan(
            ctypes.byref(pp), buf.ctypes.data_as(i32p), P.num_items, buf[n:].ctypes.data_as(i32p) if m else None,
            P.num_rows, ctypes.byref(P)))
        need = 4 * (P.partial_o_floats + P.partial_lse_floats) + 256
        if P.num_parts > 0 and self._ws.numel() * self._ws.element_size() < need:
            raise ValueError(f"workspace too small: need {need} bytes")
        # the indices first: what converts them on this stream is done when the copy of the
        # items, which waits for the stream, returns, so that runs on any stream may read them
        indices = _runtime.narrow_i32(idx, self._dev)
        if indices.numel() == 0:
            indices = torch.full((1,), -1, dtype=torch.int32, device=self._dev)
        items = torch.from_numpy(buf).to(self._dev)
        held = _runtime.PlanTensors(self._dev, items, indices)
        t = _ffi.AtfPrefillPagedParams()
        t.total_q, t.num_heads_q, t.num_heads_kv, t.head_dim = int(cq[-1]), num_qo_heads, num_kv_heads, head_dim
        t.page_size, t.num_indices, t.indices = page_size, int(ck[-1]), indices.data_ptr()
        t.items, t.rows = items.data_ptr(), items.data_ptr() + 4 * n if m else None
        t.num_items, t.num_wide, t.num_rows, t.num_parts = P.num_items, P.num_wide, P.num_rows, P.num_parts
        if P.num_parts > 0:
            base = (self._ws.data_ptr() + 255) // 256 * 256
            t.partial_o, t.partial_lse = base, base + 4 * P.partial_o_floats
        t.softmax_scale, t.causal = scale, pp.causal
        t.window = _ffi.ATF_WINDOW_SNAP16 if zhi is not None else _ffi.ATF_WINDOW_OFF
        for i, z in enumerate(zhi or ()):
            t.zhi[i] = z
        t.error_flag = _runtime.error_flag(self._dev).data_ptr()
        # in one piece: a run of another thread takes all of the old plan or all of this one
        self._planned = t, ctypes.addressof(t), held
        self._plan = t

    begin_forward = plan

    def run(self, q: torch.Tensor, paged_kv_cache, *, out: Optional[torch.Tensor] = None,
            lse: Optional[torch.Tensor] = None, return_lse: bool = False):
        """q (total_q, Hq, 128) bf16; paged_kv_cache = (k_pages, v_pages) or one tensor with a
        k/v axis at dim 1, bf16 pages in the wrapper's kv_layout (K neither level-major nor e4m3).
        Returns out (total_q, Hq, 128) [, lse (total_q, Hq), natural log]; a row that sees no key
        is 0 with an lse of -inf. A NaN key makes the rows that see it NaN and no others. A NaN
        or an infinity in V of a key reaches all rows of every tile (up to 128 rows of a
        request) that loads the key's tile of 128 keys, those that do not see it too: there
        it meets a probability of 0, whose product with it is NaN. A page id outside the cache is reported by
        ``atflash.check_device_errors()`` (code 2); its request's outputs are not valid then."""
        if self._planned is None:
            raise RuntimeError("plan() must be called before run()")
        params, address, held = self._planned  # (held on to until the call has returned)
        if isinstance(paged_kv_cache, (tuple, list)):
            kc, vc = paged_kv_cache
        else:
            kc, vc = paged_kv_cache[:, 0], paged_kv_cache[:, 1]
        held.use()
        return _ffi.binding().paged_run(address, self._dev.index, self._kv_layout == "NHD", q, kc, vc, out, lse,
                                        return_lse)

    forward = run
