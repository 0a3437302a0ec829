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
constexpr int PER_LANE = 4;  // entries of a lane in one step
constexpr int CHUNK = 32 * PER_LANE;

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

  // The requests, read side by side into shared memory (n, new tokens, owned
  // pages), then summed run by run: each thread a run of `per`, the runs' sums
  // scanned over the CTA. 64-bit sums: the offsets are cut at the capacities, the
  // sums need not fit.
  bool bad = false;
  for (int b = tid; b < a.B; b += THREADS) {
    const Req r = load_req(a, b);
    bad |= r.bad;
    s_page[b] = r.n;
    s_tok[b] = r.app;
    s_have[b] = r.have;
    if (first_cta) a.last[b] = r.n > 0 ? r.len - (r.n - 1) * a.page : 0;
  }
  __syncthreads();
  const int per = (a.B + THREADS - 1) / THREADS;
  const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
  long long sum[3] = {0, 0, 0};
  for (int b = b0; b < b1; ++b) {
    sum[0] += s_page[b];
    sum[1] += s_tok[b];
    sum[2] += s_page[b] - s_have[b];
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
  for (int b = b0; b < b1; ++b) {  // each thread turns its own run into offsets
    const int n = s_page[b], app = s_tok[b];
    s_page[b] = static_cast<int>(min(incl[0], static_cast<long long>(a.cap_pages)));
    s_tok[b] = static_cast<int>(min(incl[1], static_cast<long long>(a.cap_tokens)));
    // past the free list's end every index is refused, so a cut keeps its meaning
    s_new[b] = static_cast<int>(min(incl[2], static_cast<long long>(0x3fffffff)));
    incl[0] += n;
    incl[1] += app;
    incl[2] += n - s_have[b];
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
  if (tid == 0) {  // the ends, for the walk below
    s_page[a.B] = 0x7fffffff;
    s_tok[a.B] = 0x7fffffff;
  }
  __syncthreads();
  if (first_cta)
    for (int b = tid; b < a.B; b += THREADS) {
      a.indptr[b] = s_page[b];
      a.aptr[b] = s_tok[b];
    }

  // page j of request b: its table's, or a new one
  auto new_page = [&](int b, int j) -> int {
    const long long at = head + s_new[b] + (j - s_have[b]);
    return at >= 0 && head >= 0 && at < a.F ? a.free_pages[at] : -1;
  };
  // A warp takes chunks of 128 entries: one search for the chunk's first entry, and
  // from there each lane walks to the requests of its four (a chunk meets few).
  const int gw = static_cast<int>(blockIdx.x) * WARPS + warp, nw = static_cast<int>(gridDim.x) * WARPS;
  for (long long e0 = static_cast<long long>(gw) * CHUNK; e0 < a.cap_pages; e0 += static_cast<long long>(nw) * CHUNK) {
    int b = e0 < n_pages ? bracket(s_page, a.B, static_cast<int>(e0)) : 0;
    int id[PER_LANE];
    int32_t* put[PER_LANE];
#pragma unroll
    for (int k = 0; k < PER_LANE; ++k) {
      const long long e = e0 + 32 * k + lane;
      id[k] = -1;
      put[k] = nullptr;
      if (e < n_pages) {
        while (s_page[b + 1] <= e) ++b;
        const int j = static_cast<int>(e) - s_page[b];
        const long long row = a.req_rows != nullptr ? a.req_rows[b] : b;
        int32_t* at = a.req_pages + row * a.req_stride + j;
        if (j < s_have[b]) {
          id[k] = *at;
        } else {
          id[k] = new_page(b, j);
          put[k] = at;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < PER_LANE; ++k) {
      const long long e = e0 + 32 * k + lane;
      if (put[k] != nullptr) *put[k] = id[k];
      if (e < a.cap_pages) a.indices[e] = id[k];
    }
  }
  for (long long t0 = static_cast<long long>(gw) * CHUNK; t0 < a.cap_tokens; t0 += static_cast<long long>(nw) * CHUNK) {
    int b = t0 < n_tok ? bracket(s_tok, a.B, static_cast<int>(t0)) : 0;
    int bi[PER_LANE], pos[PER_LANE];
    int64_t slot[PER_LANE];
#pragma unroll
    for (int k = 0; k < PER_LANE; ++k) {
      const long long t = t0 + 32 * k + lane;
      bi[k] = pos[k] = -1;
      slot[k] = -1;
      if (t < n_tok) {
        while (s_tok[b + 1] <= t) ++b;
        bi[k] = b;
        pos[k] = a.kv_lens[b] - a.append_lens[b] + (static_cast<int>(t) - s_tok[b]);
        const int j = pos[k] / a.page;
        const long long row = a.req_rows != nullptr ? a.req_rows[b] : b;
        const int id = j < s_have[b] ? a.req_pages[row * a.req_stride + j] : new_page(b, j);
        if (id >= 0) slot[k] = static_cast<int64_t>(id) * a.page + pos[k] % a.page;
      }
    }
#pragma unroll
    for (int k = 0; k < PER_LANE; ++k) {
      const long long t = t0 + 32 * k + lane;
      if (t < a.cap_tokens) {
        a.bidx[t] = bi[k];
        a.pos[t] = pos[k];
        a.slots[t] = slot[k];
      }
    }
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
  long long grid = (most + tables::WARPS * tables::CHUNK - 1) / (tables::WARPS * tables::CHUNK);
  if (grid < 1) grid = 1;
  if (grid > 148) grid = 148;
  tables::tables_kernel<<<static_cast<unsigned>(grid), tables::THREADS, smem,
                          reinterpret_cast<cudaStream_t>(stream)>>>(a);
  return cudaGetLastError() == cudaSuccess ? ATF_OK : ATF_ERR_CUDA;
}
