// Page tables and slot maps of one serving step, from the requests' lengths.
//
// n_b = ceil(len_b / page) pages and a_b new tokens per request; the CSR offsets
// are the exclusive sums of n and a, and the pages a request lacks
// (n_b - ceil((len_b - a_b) / page)) come from the free list in request order, at
// the exclusive sum of those counts. Entry e of the page list belongs to the
// request whose offsets bracket it, and so does token t; each is found by a
// binary search.
//
// What bounds it: the launch and the scan's dependent steps; the data is 8 bytes
// per page and 16 per token. So everything is one launch: each CTA repeats the
// whole scan over the requests into its shared memory (8 bytes per request, from
// L2 after the first CTA) instead of waiting for another kernel or CTA, and then
// writes its own part of the entries. No CTA reads what another writes: the new
// pages go into req_pages by the thread that lists them, slots of new pages are
// taken from the free list again, and the next free head is a word of its own.
#include "atf_internal.h"

namespace atf {
namespace tables {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int ENTRIES_PER_CTA = THREADS * 4;

struct Args {
  const int32_t* kv_lens;
  const int32_t* append_lens;
  int B, page;
  int32_t* req_pages;
  long long req_stride;
  int R, M;
  const int32_t* req_rows;
  const int32_t* free_pages;
  const int32_t* free_head;
  int32_t* free_head_out;
  int F, cap_pages, cap_tokens;
  int32_t *indptr, *indices, *last, *aptr, *bidx, *pos;
  int64_t* slots;
  int* err;
};

__device__ __forceinline__ int pages_of(int len, int page) {
  return static_cast<int>((static_cast<unsigned>(len) + static_cast<unsigned>(page) - 1u) /
                          static_cast<unsigned>(page));
}

struct Req {
  int len, app, n, have;
  bool bad;
};
__device__ __forceinline__ Req load_req(const Args& a, int b) {
  Req r;
  r.len = a.kv_lens[b];
  r.app = a.append_lens[b];
  const int row = a.req_rows != nullptr ? a.req_rows[b] : b;
  r.bad = r.len < 0 || r.app < 0 || r.app > r.len || row < 0 || row >= a.R || pages_of(max(r.len, 0), a.page) > a.M;
  if (r.bad) r.len = r.app = 0;
  r.n = pages_of(r.len, a.page);
  // without a free list every page is in the table already
  r.have = a.free_pages != nullptr ? pages_of(r.len - r.app, a.page) : r.n;
  return r;
}

// largest i in [0, n) with off[i] <= x (off[0] = 0, non-decreasing)
__device__ __forceinline__ int bracket(const int* off, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(THREADS) tables_kernel(const Args a) {
  // offsets of pages, tokens and new pages, and the first new page of a request
  extern __shared__ int sm[];
  int* s_page = sm;
  int* s_tok = s_page + a.B + 1;
  int* s_new = s_tok + a.B + 1;
  int* s_have = s_new + a.B + 1;
  __shared__ long long w_sum[3][WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool first_cta = blockIdx.x == 0;

  // each thread sums a run of requests; the runs' sums are scanned over the CTA.
  // 64-bit sums: the offsets are cut at the capacities, the sums need not fit.
  const int per = (a.B + THREADS - 1) / THREADS;
  const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
  long long sum[3] = {0, 0, 0};
  bool bad = false;
  for (int b = b0; b < b1; ++b) {
    const Req r = load_req(a, b);
    bad |= r.bad;
    sum[0] += r.n;
    sum[1] += r.app;
    sum[2] += r.n - r.have;
  }
  long long incl[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    long long x = sum[k];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, off);
      if (lane >= off) x += y;
    }
    incl[k] = x;
    if (lane == 31) w_sum[k][warp] = x;
  }
  __syncthreads();
  long long total[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before += w_sum[k][w];
      all += w_sum[k][w];
    }
    incl[k] += before - sum[k];  // exclusive
    total[k] = all;
  }
  for (int b = b0; b < b1; ++b) {
    const Req r = load_req(a, b);
    const int p = static_cast<int>(min(incl[0], static_cast<long long>(a.cap_pages)));
    const int t = static_cast<int>(min(incl[1], static_cast<long long>(a.cap_tokens)));
    s_page[b] = p;
    s_tok[b] = t;
    // past the free list's end every index is refused, so a cut keeps its meaning
    s_new[b] = static_cast<int>(min(incl[2], static_cast<long long>(0x3fffffff)));
    s_have[b] = r.have;
    if (first_cta) {
      a.indptr[b] = p;
      a.aptr[b] = t;
      a.last[b] = r.n > 0 ? r.len - (r.n - 1) * a.page : 0;
    }
    incl[0] += r.n;
    incl[1] += r.app;
    incl[2] += r.n - r.have;
  }
  const int n_pages = static_cast<int>(min(total[0], static_cast<long long>(a.cap_pages)));
  const int n_tok = static_cast<int>(min(total[1], static_cast<long long>(a.cap_tokens)));
  const long long head = a.free_pages != nullptr ? *a.free_head : 0;
  if (first_cta) {
    if (tid == 0) {
      a.indptr[a.B] = n_pages;
      a.aptr[a.B] = n_tok;
      const bool short_of = a.free_pages != nullptr && (head < 0 || head + total[2] > a.F);
      if (a.free_pages != nullptr)
        *a.free_head_out = static_cast<int>(min(max(head, 0ll) + total[2], max(static_cast<long long>(a.F), head)));
      if (a.err != nullptr && (short_of || total[0] > a.cap_pages || total[1] > a.cap_tokens))
        atomicCAS(a.err, 0, kDevErrIndex);
    }
    if (bad && a.err != nullptr) atomicCAS(a.err, 0, kDevErrIndex);
  }
  __syncthreads();

  // page j of request b: its table's, or a new one
  auto new_page = [&](int b, int j) -> int {
    const long long at = head + s_new[b] + (j - s_have[b]);
    return at >= 0 && head >= 0 && at < a.F ? a.free_pages[at] : -1;
  };
  const long long stride = static_cast<long long>(gridDim.x) * THREADS;
  for (long long e = static_cast<long long>(blockIdx.x) * THREADS + tid; e < a.cap_pages; e += stride) {
    int id = -1;
    if (e < n_pages) {
      const int b = bracket(s_page, a.B, static_cast<int>(e));
      const int j = static_cast<int>(e) - s_page[b];
      const long long row = a.req_rows != nullptr ? a.req_rows[b] : b;
      int32_t* at = a.req_pages + row * a.req_stride + j;
      if (j < s_have[b]) {
        id = *at;
      } else {
        id = new_page(b, j);
        *at = id;
      }
    }
    a.indices[e] = id;
  }
  for (long long t = static_cast<long long>(blockIdx.x) * THREADS + tid; t < a.cap_tokens; t += stride) {
    int b = -1, pos = -1;
    int64_t slot = -1;
    if (t < n_tok) {
      b = bracket(s_tok, a.B, static_cast<int>(t));
      pos = a.kv_lens[b] - a.append_lens[b] + (static_cast<int>(t) - s_tok[b]);
      const int j = pos / a.page;
      const long long row = a.req_rows != nullptr ? a.req_rows[b] : b;
      const int id = j < s_have[b] ? a.req_pages[row * a.req_stride + j] : new_page(b, j);
      if (id >= 0) slot = static_cast<int64_t>(id) * a.page + pos % a.page;
    }
    a.bidx[t] = b;
    a.pos[t] = pos;
    a.slots[t] = slot;
  }
}

}  // namespace tables
}  // namespace atf

using namespace atf;

extern "C" int atf_build_page_tables(const AtfPageTablesParams* p, atf_stream_t stream) {
  if (p == nullptr || p->kv_lens == nullptr || p->append_lens == nullptr || p->req_pages == nullptr ||
      p->indptr == nullptr || p->last_page_len == nullptr || p->append_indptr == nullptr)
    return ATF_ERR_INVALID_ARG;
  if (p->batch < 1 || p->page_size < 1 || p->num_rows < 1 || p->max_req_pages < 0 || p->max_pages < 0 ||
      p->max_tokens < 0 || p->req_stride < p->max_req_pages || p->num_free < 0)
    return ATF_ERR_INVALID_ARG;
  if ((p->max_pages > 0 && p->indices == nullptr) ||
      (p->max_tokens > 0 && (p->batch_indices == nullptr || p->positions == nullptr || p->slot_mapping == nullptr)))
    return ATF_ERR_INVALID_ARG;
  if (p->free_pages != nullptr &&
      (p->free_head == nullptr || p->free_head_out == nullptr || p->free_head == p->free_head_out))
    return ATF_ERR_INVALID_ARG;
  if (p->batch > ATF_TABLES_MAX_BATCH) return ATF_ERR_UNSUPPORTED;
  int dev = 0;
  int rc = check_device(&dev);
  if (rc != ATF_OK) return rc;
  tables::Args a;
  a.kv_lens = p->kv_lens;
  a.append_lens = p->append_lens;
  a.B = p->batch;
  a.page = p->page_size;
  a.req_pages = p->req_pages;
  a.req_stride = p->req_stride;
  a.R = p->num_rows;
  a.M = p->max_req_pages;
  a.req_rows = p->req_rows;
  a.free_pages = p->free_pages;
  a.free_head = p->free_head;
  a.free_head_out = p->free_head_out;
  a.F = p->num_free;
  a.cap_pages = p->max_pages;
  a.cap_tokens = p->max_tokens;
  a.indptr = p->indptr;
  a.indices = p->indices;
  a.last = p->last_page_len;
  a.aptr = p->append_indptr;
  a.bidx = p->batch_indices;
  a.pos = p->positions;
  a.slots = p->slot_mapping;
  a.err = p->error_flag;
  const size_t smem = (4 * static_cast<size_t>(a.B) + 3) * sizeof(int);
  if (smem > 47 * 1024 && cudaFuncSetAttribute(tables::tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(smem)) != cudaSuccess)
    return ATF_ERR_CUDA;
  const long long most = a.cap_pages > a.cap_tokens ? a.cap_pages : a.cap_tokens;
  long long grid = (most + tables::ENTRIES_PER_CTA - 1) / tables::ENTRIES_PER_CTA;
  if (grid < 1) grid = 1;
  if (grid > 148) grid = 148;
  tables::tables_kernel<<<static_cast<unsigned>(grid), tables::THREADS, smem,
                          reinterpret_cast<cudaStream_t>(stream)>>>(a);
  return cudaGetLastError() == cudaSuccess ? ATF_OK : ATF_ERR_CUDA;
}
