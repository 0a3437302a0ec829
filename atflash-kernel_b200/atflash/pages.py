"""Cache pages that requests share: fork requests, free them, compact the pool and copy
pages, over the tables of ``build_page_tables`` (req_pages, free_pages, free_head).

``shared`` (int32, one entry per page, zeros to begin with) counts the holders of a page
beyond the first. It is 0 for a free page and for a page of one request, so pages that
``build_page_tables`` takes from the free list need no entry. A request that only grows
writes into its last page and new ones, and a fork gives the child a copy of a last page
that is partly filled, so a page with several holders is never written. (A request whose
length is cut back into pages that it shares would write into them: fork it at that length
instead, and free the old row.)

Index reports of these calls go to ``atflash.check_device_errors()`` (code 2). The
reference serves one request and has no counterpart."""
import ctypes
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import _ffi, _runtime


@dataclass
class PageMoves:
    """src, dst int32: pages to copy (-1 on both sides: none), for ``PageCopier.copy``;
    free_head (1): the next free list position."""
    src: torch.Tensor
    dst: torch.Tensor
    free_head: torch.Tensor


def fork_requests(parents: torch.Tensor, children: torch.Tensor, kv_lens: torch.Tensor, req_pages: torch.Tensor,
                  page_size: int, *, free_pages: torch.Tensor, free_head: torch.Tensor,
                  shared: torch.Tensor) -> PageMoves:
    """Fork requests in one launch: row children[i] of req_pages gets the pages that hold
    the first kv_lens[i] tokens of row parents[i]. Full pages are shared (one holder more in
    `shared`, in place); a last page that is partly filled becomes a page of the child's
    own from free_pages[free_head:], in the order of the children, and a pair (src, dst)
    to copy in every layer's cache before the child is read. A row may be the parent of
    many. kv_lens[i] may be less than the parent's length (a shared prefix).

    The child's row must hold no pages yet (free it first); entries past its pages stay.
    A row is a child at most once and no child is a parent: entries against that, rows or
    lengths out of range are left out. A page that the free list cannot give is -1 in the
    row, and its pair is -1. Each is reported (code 2). src and dst have one entry per
    child, -1 where there is nothing to copy; free_head itself stays."""
    return PageMoves(*_ffi.binding().fork_requests(parents, children, kv_lens, req_pages, page_size, free_pages, free_head,
                                                   shared))


def free_requests(req_rows: Optional[torch.Tensor], kv_lens: torch.Tensor, req_pages: torch.Tensor, page_size: int, *,
                  free_pages: torch.Tensor, free_head: torch.Tensor,
                  shared: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Free requests in one launch: row req_rows[i] (default i) of req_pages gives up the
    ceil(kv_lens[i] / page_size) pages of its kv_lens[i] tokens, and its entries become -1.
    Each page loses one holder; the n that have none left go back to the free list,
    free_pages[free_head - n : free_head], in place, in the order of the requests (a page
    that several of them held at its last one). Returns the next free_head; free_head
    itself stays. Without `shared` every page has one holder.

    A row that is named twice (its first entry counts), rows and lengths out of range,
    page ids outside the cache, a page given up more often than it was held and a list
    without room are reported (code 2) and left out. (Without `shared` the call knows
    neither the cache's size nor the holders: it reports negative ids, and lists any other id
    as often as the rows hold it.)"""
    return _ffi.binding().free_requests(req_rows, kv_lens, req_pages, page_size, free_pages, free_head, shared)


def compact_pages(kv_lens: torch.Tensor, req_pages: torch.Tensor, page_size: int, num_pages: int, *, max_moves: int,
                  free_pages: torch.Tensor, req_rows: Optional[torch.Tensor] = None,
                  shared: Optional[torch.Tensor] = None) -> PageMoves:
    """Move pages in use towards the start of the cache, in one launch. kv_lens (and
    req_rows, default i) name every request that holds pages; the L pages that they hold
    out of num_pages end up as pages 0 .. L-1: the highest page at or above L moves to the
    lowest free one, the next to the next, at most max_moves of them (a later call goes
    on). req_pages and `shared` follow, in place; src and dst (max_moves) are the pairs
    to copy in every layer's cache, -1 past the last; free_pages (num_pages entries or
    more) becomes the list of all other pages, rising, at its end, and free_head in the
    result points to its first.

    Pages that no named request holds count as free, and their entries of `shared` become 0.
    A page that named and other requests held together keeps its count of holders: free a
    request, rather than leave it out, when others share its pages. Rows, lengths and page ids out of
    range are reported (code 2) and left out. At most 2^20 pages."""
    return PageMoves(*_ffi.binding().compact_pages(kv_lens, req_pages, page_size, num_pages, max_moves, free_pages, req_rows,
                                                   shared))


class PageCopier:
    """Copies pages in every tensor of a cache at once: the K and V pages of all layers
    and, for e4m3 pages, their scales. Made once for a cache (it keeps the tensors, whose
    first axis is the page); copy() is one launch per 256 tensors."""

    def __init__(self, caches: Sequence[torch.Tensor]):
        caches = list(caches)
        if not caches:
            raise ValueError("at least one cache tensor")
        self._dev = _runtime.require_cuda(*caches)
        self._pages = caches[0].shape[0] if caches[0].dim() > 0 else 0
        desc = (_ffi.AtfPageTensor * len(caches))()
        for d, t in zip(desc, caches):
            if t.dim() < 1 or t.shape[0] != self._pages or t.numel() == 0:
                raise ValueError("the first axis of every cache tensor is the page, of the same number")
            dense = 1  # a page's own elements lie together, in any order of the axes
            for size, stride in sorted(zip(t.shape[1:], t.stride()[1:]), key=lambda x: (x[1], x[0])):
                if size > 1:
                    if stride != dense:
                        raise ValueError("a page's elements must lie together in memory")
                    dense *= size
            if self._pages > 1 and t.stride(0) < dense:
                raise ValueError("the pages of a cache tensor must not overlap")
            es = t.element_size()
            d.base, d.page_stride_bytes, d.page_bytes = t.data_ptr(), t.stride(0) * es, dense * es
        self._caches, self._desc, self._desc_ptr = caches, desc, ctypes.addressof(desc)

    def copy(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Page src[i] of every tensor to page dst[i]; -1 on both sides is no copy, and
        other ids outside the cache are reported by ``atflash.check_device_errors()`` (code 2)
        and left out. The pages of dst differ from one another and are none of src's, as in
        the lists of ``fork_requests`` and ``compact_pages``; src may name a page twice."""
        _ffi.binding().copy_pages(self._desc_ptr, len(self._desc), self._pages, self._dev.index, src, dst)


def copy_pages(caches: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor) -> None:
    """``PageCopier(caches).copy(src, dst)``, for a single copy."""
    PageCopier(caches).copy(src, dst)
