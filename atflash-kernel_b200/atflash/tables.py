"""Page tables and slot maps of a serving step, built on the GPU from the
requests' lengths (``atf_build_page_tables``). The paged append takes them without a
host round trip; the plans of the decode and of the packed prefill read their offsets
on the host, which waits for the stream.

The reference decodes one request over a contiguous cache
(e2e_pipeline/atflash_e2e_fafi.py:219-223) and has no counterpart."""
import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from . import _ffi, _runtime


@dataclass
class PageTables:
    """indptr (B+1) / indices / last_page_len (B): the CSR page table;
    append_indptr (B+1), batch_indices, positions, slot_mapping (int64): request,
    position and cache slot (page * page_size + slot) of each new token. Entries
    past the end are -1. free_head (1): the next free list position, or None."""
    indptr: torch.Tensor
    indices: torch.Tensor
    last_page_len: torch.Tensor
    append_indptr: torch.Tensor
    batch_indices: torch.Tensor
    positions: torch.Tensor
    slot_mapping: torch.Tensor
    free_head: Optional[torch.Tensor]


def _i32(t: torch.Tensor, name: str, n: Optional[int] = None) -> torch.Tensor:
    if t.dim() != 1 or t.dtype not in (torch.int32, torch.int64) or (n is not None and t.numel() != n):
        raise ValueError(f"{name} must be a 1-d integer tensor" + (f" of {n} entries" if n is not None else ""))
    if t.dtype != torch.int32 or not t.is_contiguous():
        t = _runtime.narrow_i32(t, t.device)
    return t


def build_page_tables(kv_lens: torch.Tensor, append_lens: torch.Tensor, req_pages: torch.Tensor, page_size: int, *,
                      num_tokens: int, max_pages: int, req_rows: Optional[torch.Tensor] = None,
                      free_pages: Optional[torch.Tensor] = None,
                      free_head: Optional[torch.Tensor] = None) -> PageTables:
    """Build a step's tables in one launch.

    kv_lens (B): tokens of each request after the step; append_lens (B): how many
    of them are new. req_pages int32 (rows, pages): the engine's table of page ids,
    row req_rows[b] (default b) for request b. With free_pages (int32, 1-d) and
    free_head (int32, 1 entry) the pages that a request lacks are taken from
    free_pages[free_head:] in request order and written into req_pages, in place;
    the next head is in the result (free_head itself stays). Without them req_pages
    holds every page already.

    num_tokens and max_pages are the sizes of the token outputs and of indices: the
    step's totals, or capacities (a fixed shape for a CUDA graph): entries past the
    end are -1. Bad lengths or rows, an exhausted free list, pages that req_pages should
    hold but does not (negative entries) and exceeded capacities are reported by
    ``atflash.check_device_errors()`` (code 2). A capacity cuts the lists only: req_pages
    gets, and free_head counts, every new page of the step, so that the same call with
    the same free_head and larger capacities completes it."""
    dev = _runtime.require_cuda(kv_lens, append_lens, req_pages)
    B = kv_lens.numel()
    if B < 1 or B > _ffi.ATF_TABLES_MAX_BATCH:
        raise ValueError(f"between 1 and {_ffi.ATF_TABLES_MAX_BATCH} requests")
    kv_lens, append_lens = _i32(kv_lens, "kv_lens"), _i32(append_lens, "append_lens", B)
    num_tokens, max_pages = int(num_tokens), int(max_pages)
    shape, st = req_pages.shape, req_pages.stride()
    if len(shape) != 2 or req_pages.dtype != torch.int32 or (shape[1] > 1 and st[1] != 1):
        raise ValueError("req_pages must be an int32 (rows, pages) tensor with contiguous rows")
    R, M = shape
    if R < 1 or (req_rows is None and R < B):
        raise ValueError("req_pages needs a row for each request")
    if R > 1 and st[0] < M:
        raise ValueError("the rows of req_pages must not overlap")
    if page_size < 1 or num_tokens < 0 or max_pages < 0:
        raise ValueError("page_size must be positive, num_tokens and max_pages not negative")
    if max(num_tokens, max_pages) >= 1 << 30:
        raise ValueError("num_tokens and max_pages must be under 2^30")
    if (free_pages is None) != (free_head is None):
        raise ValueError("free_pages and free_head go together")
    rows_ptr = free_ptr = head_ptr = num_free = 0
    if req_rows is not None:
        _runtime.require_cuda(kv_lens, req_rows)
        req_rows = _i32(req_rows, "req_rows", B)
        rows_ptr = req_rows.data_ptr()
    if free_pages is not None:
        _runtime.require_cuda(kv_lens, free_pages, free_head)
        free_pages = _i32(free_pages, "free_pages")
        free_head = _i32(free_head, "free_head", 1)
        # an empty list still has a head: any valid address will do for its pages
        head_ptr, num_free = free_head.data_ptr(), free_pages.numel()
        free_ptr = free_pages.data_ptr() or head_ptr
    # one allocation for the 32-bit outputs, in the order of PageTables
    buf = torch.empty(3 * B + 3 + max_pages + 2 * num_tokens, dtype=torch.int32, device=dev)
    slots = torch.empty(num_tokens, dtype=torch.int64, device=dev)
    indptr = buf.data_ptr()
    indices = indptr + 4 * (B + 1)
    last = indices + 4 * max_pages
    aptr = last + 4 * B
    bidx = aptr + 4 * (B + 1)
    pos = bidx + 4 * num_tokens
    lens_ptr = kv_lens.data_ptr()
    # (req_pages without columns is never read: any valid address will do)
    p = _ffi.AtfPageTablesParams(
        lens_ptr, append_lens.data_ptr(), B, int(page_size), req_pages.data_ptr() or lens_ptr, st[0] if R > 1 else max(1, M),
        R, M, rows_ptr, free_ptr, head_ptr, pos + 4 * num_tokens if head_ptr else 0, num_free, max_pages, num_tokens,
        indptr, indices, last, aptr, bidx, pos, slots.data_ptr(), _runtime.error_flag_ptr(dev))
    _runtime.launch("atf_build_page_tables", _ffi.load().atf_build_page_tables, dev, ctypes.byref(p))
    out = buf.split_with_sizes((B + 1, max_pages, B, B + 1, num_tokens, num_tokens, 1))
    return PageTables(*out[:6], slots, out[6] if head_ptr else None)
