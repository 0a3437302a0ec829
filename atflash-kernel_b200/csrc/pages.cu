// Pages that requests share: forking, freeing, compacting and copying them.
//
// shared[p] counts the holders of page p beyond the first, so that a page of one
// request, or of none, is 0 and the page tables (tables.cu) take pages without touching
// it. Entry e = (request i of the call, page j of its row).
//
// Fork: a child's full pages are its parent's, each with one holder more; a last page
// that is only partly filled is one of its own from the free list, and goes on the list
// of copies. Which entry gets which new page is an exclusive sum over the children.
// One launch; as in tables.cu every CTA repeats the scan and then writes its part.
//
// Free: every entry takes one holder from its page; a page left without any goes back to
// the free list, listed at its last entry of the call. So the order does not depend on
// the atomics': all entries subtract, then (-1: nobody is left) race with atomicMin for
// the largest e, whose place is an exclusive sum over entries. The three steps are
// phases of one thread-block cluster, with cluster barriers between them.
//
// Compact: live pages are marked in a bitmap (each CTA of the cluster its part of the
// entries, merged over distributed shared memory), with the number of live pages before
// each group of words. That gives every page's place in closed form: of L live pages
// the i-th highest at or above L moves to the i-th lowest free page below L, and
// the free list is the rising list of what is free afterwards. Then the tables and the
// counts follow. One launch.
//
// Copy: 16 KB pieces of (pair, tensor) over the grid, 16 bytes per lane and load, eight
// loads in flight. HBM-bound: 2144 pairs x 4 tensors x 64 KB 174 us (floor 173); with four
// loads and eight CTAs of 256 an SM, each going through its pieces, 209 (191 with eight
// loads). Up to 128 CTAs an SM wait their turn; more bring nothing, and lists that are
// mostly padding want few.
//
// What bounds the first three: the launch and a few dependent reads of the tables. 96
// children of up to 128 pages: fork 7 us, free 7.4 (10.7 with the page ids read again in
// each phase, 7.7 with the marks read twice); compaction of a pool of 8703 pages 8.5.
#include <cooperative_groups.h>

#include "atf_internal.h"

namespace atf {
namespace pages {

namespace cg = cooperative_groups;

__device__ __forceinline__ void report(int* err) {
  if (err != nullptr) atomicCAS(err, 0, kDevErrIndex);
}
__device__ __forceinline__ int pages_of(int len, int page) {  // len >= 0
  return static_cast<int>((static_cast<unsigned>(len) + static_cast<unsigned>(page) - 1u) / static_cast<unsigned>(page));
}

// Exclusive sum of one value per thread over the CTA; *total gets the sum. Every thread
// calls it; s_warp holds a value per warp and one more.
__device__ __forceinline__ int cta_exclusive(int v, int* s_warp, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int x = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();  // a previous call's readers are done
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = lane < warps ? s_warp[lane] : 0, z = w;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, z, off);
      if (lane >= off) z += y;
    }
    if (lane < warps) s_warp[lane] = z - w;
    if (lane == 31) s_warp[32] = z;
  }
  __syncthreads();
  *total = s_warp[32];
  return s_warp[warp] + x - v;
}

// ------------------------------------------------------------------ fork

struct ForkArgs {
  const int32_t* parents;
  const int32_t* children;
  const int32_t* lens;
  int N, page;
  int32_t* rows;  // req_pages
  long long stride;
  int R, M;
  int32_t* shared;
  int P;
  const int32_t* free_pages;
  const int32_t* free_head;
  int32_t* free_head_out;
  int F;
  int32_t* src;
  int32_t* dst;
  int* err;
};

constexpr int FORK_THREADS = 512;

__global__ void __launch_bounds__(FORK_THREADS) fork_kernel(const ForkArgs a) {
  extern __shared__ int sm[];
  int* s_owner = sm;             // [R] first child entry of a row
  int* s_new = s_owner + a.R;    // [N] new pages of the children before
  int* s_len = s_new + a.N;      // [N] tokens, 0 for a child that is left out
  __shared__ int s_warp[33];
  const int tid = threadIdx.x;
  const bool first = blockIdx.x == 0;
  for (int r = tid; r < a.R; r += FORK_THREADS) s_owner[r] = 0x7fffffff;
  __syncthreads();
  for (int i = tid; i < a.N; i += FORK_THREADS) {
    const int c = a.children[i];
    if (c >= 0 && c < a.R) atomicMin(&s_owner[c], i);
  }
  __syncthreads();
  bool bad = false;
  for (int i = tid; i < a.N; i += FORK_THREADS) {
    const int c = a.children[i], p = a.parents[i], len = a.lens[i];
    const bool ok = c >= 0 && c < a.R && p >= 0 && p < a.R && len >= 0 && pages_of(max(len, 0), a.page) <= a.M &&
                    s_owner[c] == i && s_owner[p] == 0x7fffffff;
    bad |= !ok;
    s_len[i] = ok ? len : 0;
  }
  __syncthreads();
  // each thread a run of children
  const int per = (a.N + FORK_THREADS - 1) / FORK_THREADS;
  const int i0 = min(tid * per, a.N), i1 = min(i0 + per, a.N);
  int n = 0, total = 0;
  for (int i = i0; i < i1; ++i) n += s_len[i] % a.page != 0 ? 1 : 0;
  n = cta_exclusive(n, s_warp, &total);
  for (int i = i0; i < i1; ++i) {
    s_new[i] = n;
    n += s_len[i] % a.page != 0 ? 1 : 0;
  }
  __syncthreads();
  const int head = *a.free_head;
  auto new_page = [&](int i) -> int {
    const long long at = static_cast<long long>(head) + s_new[i];
    const int id = head >= 0 && at < a.F ? a.free_pages[at] : -1;
    return id >= 0 && id < a.P ? id : -1;
  };
  if (first) {
    for (int i = tid; i < a.N; i += FORK_THREADS) {
      int src = -1, dst = -1;
      const int len = s_len[i], full = len / a.page;
      if (len % a.page != 0) {
        src = a.rows[a.parents[i] * a.stride + full];
        dst = new_page(i);
        if (src < 0 || src >= a.P || dst < 0) {
          src = dst = -1;
          bad = true;
        }
      }
      a.src[i] = src;
      a.dst[i] = dst;
    }
    if (tid == 0) {
      const bool short_of = total > 0 && (head < 0 || total > a.F - head);
      *a.free_head_out = short_of ? max(a.F, head) : head + total;
      if (short_of) report(a.err);
    }
    if (bad) report(a.err);
  }
  // entries, four at a time per thread with their reads side by side
  const long long all = static_cast<long long>(a.N) * a.M, step = static_cast<long long>(gridDim.x) * FORK_THREADS;
  bool missing = false;
  for (long long e0 = static_cast<long long>(blockIdx.x) * FORK_THREADS + tid; e0 < all; e0 += 4 * step) {
    int id[4];
    long long put[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long long e = e0 + u * step;
      put[u] = -1;
      id[u] = -1;
      if (e >= all) continue;
      const int i = static_cast<int>(static_cast<unsigned>(e) / static_cast<unsigned>(a.M));
      const int j = static_cast<int>(e - static_cast<long long>(i) * a.M);
      const int len = s_len[i], full = len / a.page;
      if (j > full || (j == full && len % a.page == 0)) continue;
      put[u] = a.children[i] * a.stride + j;
      if (j == full) {
        id[u] = new_page(i);
        continue;
      }
      id[u] = a.rows[a.parents[i] * a.stride + j];
      if (id[u] >= 0 && id[u] < a.P)
        atomicAdd(a.shared + id[u], 1);
      else
        missing = true;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (put[u] >= 0) a.rows[put[u]] = id[u];
  }
  if (missing) report(a.err);
}

// ------------------------------------------------------------------ free

constexpr int CLUSTER = 8;
constexpr int THREADS = 1024;

struct FreeArgs {
  const int32_t* req_rows;
  const int32_t* lens;
  int N, page;
  int32_t* rows;
  long long stride;
  int R, M;
  int32_t* shared;  // or null: no page is shared
  int P;            // pages counted in shared (or the largest int)
  int32_t* free_pages;
  const int32_t* free_head;
  int32_t* free_head_out;
  int F;
  int* err;
};

// the reads of the counts between the phases come from L2, where the atomics are
__device__ __forceinline__ int fresh(const int* p) { return __ldcg(p); }

constexpr int KEPT = 4;  // entries of a lane whose pages stay in registers over the phases

__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(THREADS) free_kernel(const FreeArgs a) {
  extern __shared__ int sm[];
  int* s_owner = sm;            // [R] first entry of a row
  int* s_n = s_owner + a.R;     // [N] pages to free, 0 for a request that is left out
  int* s_row = s_n + a.N;       // [N]
  __shared__ int s_warp[33];
  __shared__ int s_count;       // pages that this CTA frees
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, rank = static_cast<int>(cluster.block_rank());
  for (int r = tid; r < a.R; r += THREADS) s_owner[r] = 0x7fffffff;
  __syncthreads();
  for (int i = tid; i < a.N; i += THREADS) {
    const int r = a.req_rows != nullptr ? a.req_rows[i] : i;
    s_row[i] = r;
    s_n[i] = a.lens[i];
    if (r >= 0 && r < a.R) atomicMin(&s_owner[r], i);
  }
  const int head = *a.free_head;
  __syncthreads();
  bool bad = false;
  for (int i = tid; i < a.N; i += THREADS) {
    const int r = s_row[i], len = s_n[i];
    const bool ok = r >= 0 && r < a.R && s_owner[r] == i && len >= 0 && pages_of(max(len, 0), a.page) <= a.M;
    bad |= !ok;
    s_n[i] = ok ? pages_of(len, a.page) : 0;
  }
  __syncthreads();
  // this thread's entries: CTA, warp and lane in the order of e, in steps of 32
  const int all = a.N * a.M;  // under 2^30
  const int warps = CLUSTER * THREADS / 32;
  const int per_warp = ((all + warps - 1) / warps + 31) / 32 * 32;
  const int gw = rank * (THREADS / 32) + (tid >> 5), lane = tid & 31;
  const int e0 = static_cast<int>(min(static_cast<long long>(gw) * per_warp, static_cast<long long>(all)));
  const int e1 = static_cast<int>(min(static_cast<long long>(e0) + per_warp, static_cast<long long>(all)));
  // where entry e's page id stands, null where there is no entry
  auto place_of = [&](int e) -> int32_t* {
    if (e >= e1) return nullptr;
    const int i = static_cast<int>(static_cast<unsigned>(e) / static_cast<unsigned>(a.M)), j = e - i * a.M;
    return j < s_n[i] ? a.rows + s_row[i] * a.stride + j : nullptr;
  };
  // page of entry e, -1 where there is none
  auto page_at = [&](int e) -> int {
    const int32_t* at = place_of(e);
    if (at == nullptr) return -1;
    const int id = *at;
    if (id < 0 || id >= a.P) {
      bad = true;
      return -1;
    }
    return id;
  };
  int kept[KEPT];  // pages of the lane's first entries, read side by side
#pragma unroll
  for (int k = 0; k < KEPT; ++k) kept[k] = page_at(e0 + lane + 32 * k);
  // f(e, page) for the lane's entries in order, every lane of the warp together
  auto entries = [&](auto&& f) {
#pragma unroll
    for (int k = 0; k < KEPT; ++k)
      if (e0 + 32 * k < e1) f(e0 + lane + 32 * k, kept[k], k);
    for (int e = e0 + lane + 32 * KEPT; e - lane < e1; e += 32) f(e, page_at(e), KEPT);
  };
  auto mark_of = [&](int e) { return static_cast<int>(0x80000000u) + (all - 1 - e); };
  if (a.shared != nullptr) {
    entries([&](int, int id, int) {
      if (id >= 0) atomicSub(a.shared + id, 1);
    });
    cluster.sync();
    entries([&](int e, int id, int) {
      if (id < 0) return;
      const int left = fresh(a.shared + id);
      if (left >= 0) return;
      // (marks are far below any count) more requests gave the page up than held it
      if (left < -1 && left > -(1 << 30)) bad = true;
      atomicMin(a.shared + id, mark_of(e));
    });
    cluster.sync();
  }
  auto freed = [&](int e, int id) {
    return id >= 0 && (a.shared == nullptr || fresh(a.shared + id) == mark_of(e));
  };
  int mine = 0;        // of this warp
  unsigned known = 0;  // whether the kept entries are freed
  entries([&](int e, int id, int k) {
    const bool is = freed(e, id);
    if (k < KEPT) known |= is ? 1u << k : 0u;
    mine += __popc(__ballot_sync(0xffffffffu, is));
  });
  int in_cta = 0;
  int before = cta_exclusive(lane == 0 ? mine : 0, s_warp, &in_cta);
  before = __shfl_sync(0xffffffffu, before, 0);
  if (tid == 0) s_count = in_cta;
  cluster.sync();
  int total = 0;
  for (int r = 0; r < CLUSTER; ++r) {
    const int n = *cluster.map_shared_rank(&s_count, r);
    if (r < rank) before += n;
    total += n;
  }
  const long long start = static_cast<long long>(head) - total;
  entries([&](int e, int id, int k) {
    const bool is = k < KEPT ? ((known >> k) & 1u) != 0 : freed(e, id);
    const unsigned who = __ballot_sync(0xffffffffu, is);
    if (is) {
      const long long to = start + before + __popc(who & ((1u << lane) - 1u));
      if (to >= 0 && to < a.F)
        a.free_pages[to] = id;
      else
        bad = true;  // the list has no room: a page was freed that was not taken from it
      if (a.shared != nullptr) a.shared[id] = 0;
    }
    before += __popc(who);
    if (int32_t* at = place_of(e)) *at = -1;
  });
  if (rank == 0 && tid == 0) *a.free_head_out = static_cast<int>(start < 0 ? 0 : start);
  if (bad) report(a.err);
  cluster.sync();  // no CTA leaves while another reads its count
}

// ------------------------------------------------------------------ compact

struct CompactArgs {
  const int32_t* req_rows;
  const int32_t* lens;
  int N, page;
  int32_t* rows;
  long long stride;
  int R, M;
  int32_t* shared;  // or null
  int P, max_moves;
  int32_t* free_pages;
  int32_t* free_head_out;
  int F;
  int32_t* src;
  int32_t* dst;
  int* err;
};

constexpr int GROUP = 8;  // words of the bitmap per entry of the sums

__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(THREADS) compact_kernel(const CompactArgs a) {
  extern __shared__ unsigned smu[];
  const int groups = (a.P + 32 * GROUP - 1) / (32 * GROUP), words = groups * GROUP;
  unsigned* s_live = smu;                                   // [words]
  int* s_rank = reinterpret_cast<int*>(s_live + words);     // [groups + 1] live pages before a group
  __shared__ int s_warp[33];
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, rank = static_cast<int>(cluster.block_rank());
  const int gt = rank * THREADS + tid, all_threads = CLUSTER * THREADS;
  for (int w = tid; w < words; w += THREADS) s_live[w] = 0;
  __syncthreads();
  bool bad = false;
  const long long all = static_cast<long long>(a.N) * a.M;
  // f(address, page) for this thread's entries
  auto entries = [&](auto&& f) {
    for (long long e = gt; e < all; e += all_threads) {
      const int i = static_cast<int>(static_cast<unsigned>(e) / static_cast<unsigned>(a.M));
      const int j = static_cast<int>(e - static_cast<long long>(i) * a.M);
      const int r = a.req_rows != nullptr ? a.req_rows[i] : i, len = a.lens[i];
      if (r < 0 || r >= a.R || len < 0 || pages_of(max(len, 0), a.page) > a.M) {
        bad = true;
        continue;
      }
      if (j >= pages_of(len, a.page)) continue;
      int32_t* at = a.rows + r * a.stride + j;
      const int id = *at;
      if (id < 0 || id >= a.P)
        bad = true;
      else
        f(at, id);
    }
  };
  entries([&](int32_t*, int id) { atomicOr(&s_live[id >> 5], 1u << (id & 31)); });
  cluster.sync();
  // the CTAs' bitmaps joined: each CTA a slice of the words, written to all
  for (int w = gt; w < words; w += all_threads) {
    unsigned v = 0;
    for (int r = 0; r < CLUSTER; ++r) v |= *cluster.map_shared_rank(&s_live[w], r);
    for (int r = 0; r < CLUSTER; ++r) *cluster.map_shared_rank(&s_live[w], r) = v;
  }
  cluster.sync();
  int live = 0;
  {
    const int per = (groups + THREADS - 1) / THREADS;
    const int g0 = min(tid * per, groups), g1 = min(g0 + per, groups);
    int n = 0;
    for (int g = g0; g < g1; ++g)
      for (int k = 0; k < GROUP; ++k) n += __popc(s_live[g * GROUP + k]);
    n = cta_exclusive(n, s_warp, &live);
    for (int g = g0; g < g1; ++g) {
      s_rank[g] = n;
      for (int k = 0; k < GROUP; ++k) n += __popc(s_live[g * GROUP + k]);
    }
  }
  __syncthreads();
  // live pages below p < P
  auto rank_of = [&](int p) -> int {
    const int w = p >> 5, g = w / GROUP;
    int n = s_rank[g] + __popc(s_live[w] & ((1u << (p & 31)) - 1u));
    for (int k = g * GROUP; k < w; ++k) n += __popc(s_live[k]);
    return n;
  };
  // live pages at or above `live`, as many as free ones below it
  const int movers = live < a.P ? live - rank_of(live) : 0;
  const int moves = min(movers, a.max_moves), n_free = a.P - live;
  for (int p = gt; p < a.P; p += all_threads) {
    const int r = rank_of(p), z = p - r;  // live and free pages below p
    const bool is_live = (s_live[p >> 5] >> (p & 31)) & 1u;
    const int from_top = live - 1 - r;    // live pages above, of a live one
    bool free_after = !is_live && z >= moves;
    if (is_live && p >= live && from_top < moves) {
      a.src[from_top] = p;
      free_after = true;
    }
    if (!is_live && z < moves) a.dst[z] = p;
    if (free_after) {
      const int live_before = r + min(moves, z) - max(0, r - (live - moves));
      a.free_pages[a.F - n_free + (p - live_before)] = p;
    }
    // Holders that were not named are gone: a free page has none. (A hole that a page moves
    // into takes that page's count below, and the page that leaves is 0 from then on.)
    if (!is_live && z >= moves && a.shared != nullptr) a.shared[p] = 0;
  }
  for (int i = gt; i < a.max_moves; i += all_threads)
    if (i >= moves) a.src[i] = a.dst[i] = -1;
  if (gt == 0) *a.free_head_out = a.F - n_free;
  cluster.sync();
  if (a.shared != nullptr)
    for (int i = gt; i < moves; i += all_threads) {
      const int from = __ldcg(a.src + i), to = __ldcg(a.dst + i);
      a.shared[to] = a.shared[from];
      a.shared[from] = 0;
    }
  entries([&](int32_t* at, int id) {
    if (id < live) return;
    const int i = live - 1 - rank_of(id);
    if (i < moves) *at = __ldcg(a.dst + i);
  });
  if (bad) report(a.err);
}

// ------------------------------------------------------------------ copy

constexpr int MAX_TENSORS = ATF_COPY_MAX_TENSORS;
constexpr int COPY_THREADS = 128;
constexpr int COPY_LOADS = 8;
constexpr int PIECE = COPY_THREADS * COPY_LOADS * 16;  // bytes

struct CopyArgs {
  const int32_t* src;
  const int32_t* dst;
  int n, P, tensors, pieces;  // pieces of a pair, over all tensors
  int* err;
  int first[MAX_TENSORS + 1];  // pieces before a tensor
  struct {
    uint8_t* base;
    long long stride, bytes;
  } t[MAX_TENSORS];
};

template <typename T>
__device__ __forceinline__ void copy_piece(const uint8_t* from, uint8_t* to, int bytes) {
  constexpr int U = COPY_LOADS;
  const T* f = reinterpret_cast<const T*>(from);
  T* d = reinterpret_cast<T*>(to);
  const int n = bytes / static_cast<int>(sizeof(T));
  for (int i0 = threadIdx.x; i0 < n; i0 += U * COPY_THREADS) {
    T v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * COPY_THREADS < n) v[u] = f[i0 + u * COPY_THREADS];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * COPY_THREADS < n) d[i0 + u * COPY_THREADS] = v[u];
  }
}

__global__ void __launch_bounds__(COPY_THREADS) copy_kernel(const __grid_constant__ CopyArgs a) {
  const long long all = static_cast<long long>(a.n) * a.pieces;
  for (long long w = blockIdx.x; w < all; w += gridDim.x) {
    const int i = static_cast<int>(w / a.pieces), x = static_cast<int>(w - static_cast<long long>(i) * a.pieces);
    const int from = __ldg(a.src + i), to = __ldg(a.dst + i);
    if (from < 0 || to < 0 || from >= a.P || to >= a.P) {
      // padding is -1 on both sides
      if (!(from == -1 && to == -1) && x == 0 && threadIdx.x == 0) report(a.err);
      continue;
    }
    if (from == to) continue;
    int lo = 0, hi = a.tensors;  // the tensor whose pieces bracket x
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.first[mid] <= x) lo = mid; else hi = mid;
    }
    const long long off = static_cast<long long>(x - a.first[lo]) * PIECE, left = a.t[lo].bytes - off;
    const int bytes = static_cast<int>(left < PIECE ? left : PIECE);
    const uint8_t* f = a.t[lo].base + from * a.t[lo].stride + off;
    uint8_t* d = a.t[lo].base + to * a.t[lo].stride + off;
    const unsigned long long low = reinterpret_cast<unsigned long long>(f) | reinterpret_cast<unsigned long long>(d) |
                                   static_cast<unsigned long long>(bytes);
    if ((low & 15) == 0)
      copy_piece<uint4>(f, d, bytes);
    else if ((low & 3) == 0)
      copy_piece<uint32_t>(f, d, bytes);
    else
      copy_piece<uint8_t>(f, d, bytes);
  }
}

}  // namespace pages
}  // namespace atf

using namespace atf;

namespace {
template <typename K>
int allow_smem(K kernel, size_t bytes) {
  return bytes > 47 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(bytes)) != cudaSuccess
             ? ATF_ERR_CUDA
             : ATF_OK;
}
// the request table, as all three calls take it
int table_ok(const int32_t* rows, int64_t stride, int32_t num_rows, int32_t max_pages, int32_t batch, int32_t page) {
  if (rows == nullptr || batch < 1 || page < 1 || num_rows < 1 || max_pages < 1 || stride < max_pages)
    return ATF_ERR_INVALID_ARG;
  if (batch > ATF_TABLES_MAX_BATCH || num_rows > ATF_PAGES_MAX_ROWS ||
      static_cast<long long>(batch) * max_pages >= (1ll << 30))
    return ATF_ERR_UNSUPPORTED;
  return ATF_OK;
}
}  // namespace

extern "C" int atf_fork_requests(const AtfForkParams* p, atf_stream_t stream) {
  if (p == nullptr || p->parents == nullptr || p->children == nullptr || p->kv_lens == nullptr ||
      p->shared == nullptr || p->free_pages == nullptr || p->free_head == nullptr || p->free_head_out == nullptr ||
      p->free_head == p->free_head_out || p->src == nullptr || p->dst == nullptr || p->num_pages < 1 ||
      p->num_free < 0)
    return ATF_ERR_INVALID_ARG;
  int rc = table_ok(p->req_pages, p->req_stride, p->num_rows, p->max_req_pages, p->batch, p->page_size);
  if (rc != ATF_OK) return rc;
  int dev = 0;
  if ((rc = check_device(&dev)) != ATF_OK) return rc;
  const pages::ForkArgs a = {p->parents,   p->children, p->kv_lens,    p->batch,     p->page_size,     p->req_pages,
                             p->req_stride, p->num_rows, p->max_req_pages, p->shared, p->num_pages,    p->free_pages,
                             p->free_head, p->free_head_out, p->num_free, p->src,    p->dst,           p->error_flag};
  const size_t smem = (static_cast<size_t>(a.R) + 2 * static_cast<size_t>(a.N)) * sizeof(int);
  if ((rc = allow_smem(pages::fork_kernel, smem)) != ATF_OK) return rc;
  const long long all = static_cast<long long>(a.N) * a.M, per = 4 * pages::FORK_THREADS;
  const long long grid = (all + per - 1) / per;
  pages::fork_kernel<<<static_cast<unsigned>(grid > 148 ? 148 : grid), pages::FORK_THREADS, smem,
                       reinterpret_cast<cudaStream_t>(stream)>>>(a);
  return cudaGetLastError() == cudaSuccess ? ATF_OK : ATF_ERR_CUDA;
}

extern "C" int atf_free_requests(const AtfFreeParams* p, atf_stream_t stream) {
  if (p == nullptr || p->kv_lens == nullptr || p->free_pages == nullptr || p->free_head == nullptr ||
      p->free_head_out == nullptr || p->free_head == p->free_head_out || p->num_free < 0 ||
      (p->shared != nullptr && p->num_pages < 1))
    return ATF_ERR_INVALID_ARG;
  int rc = table_ok(p->req_pages, p->req_stride, p->num_rows, p->max_req_pages, p->batch, p->page_size);
  if (rc != ATF_OK) return rc;
  int dev = 0;
  if ((rc = check_device(&dev)) != ATF_OK) return rc;
  const pages::FreeArgs a = {p->req_rows,      p->kv_lens,   p->batch,     p->page_size,     p->req_pages,
                             p->req_stride,    p->num_rows,  p->max_req_pages, p->shared,
                             p->shared != nullptr ? p->num_pages : 0x7fffffff, p->free_pages, p->free_head,
                             p->free_head_out, p->num_free,  p->error_flag};
  const size_t smem = (static_cast<size_t>(a.R) + 2 * static_cast<size_t>(a.N)) * sizeof(int);
  if ((rc = allow_smem(pages::free_kernel, smem)) != ATF_OK) return rc;
  pages::free_kernel<<<pages::CLUSTER, pages::THREADS, smem, reinterpret_cast<cudaStream_t>(stream)>>>(a);
  return cudaGetLastError() == cudaSuccess ? ATF_OK : ATF_ERR_CUDA;
}

extern "C" int atf_compact_pages(const AtfCompactParams* p, atf_stream_t stream) {
  if (p == nullptr || p->kv_lens == nullptr || p->free_pages == nullptr || p->free_head_out == nullptr ||
      p->num_pages < 1 || p->max_moves < 0 || p->num_free < p->num_pages ||
      (p->max_moves > 0 && (p->src == nullptr || p->dst == nullptr)))
    return ATF_ERR_INVALID_ARG;
  int rc = table_ok(p->req_pages, p->req_stride, p->num_rows, p->max_req_pages, p->batch, p->page_size);
  if (rc != ATF_OK) return rc;
  if (p->num_pages > ATF_COMPACT_MAX_PAGES) return ATF_ERR_UNSUPPORTED;
  int dev = 0;
  if ((rc = check_device(&dev)) != ATF_OK) return rc;
  const pages::CompactArgs a = {p->req_rows,  p->kv_lens,  p->batch,         p->page_size, p->req_pages,
                                p->req_stride, p->num_rows, p->max_req_pages, p->shared,    p->num_pages,
                                p->max_moves, p->free_pages, p->free_head_out, p->num_free, p->src,
                                p->dst,       p->error_flag};
  const size_t groups = (static_cast<size_t>(a.P) + 32 * pages::GROUP - 1) / (32 * pages::GROUP);
  const size_t smem = (groups * pages::GROUP + groups + 1) * sizeof(int);
  if ((rc = allow_smem(pages::compact_kernel, smem)) != ATF_OK) return rc;
  pages::compact_kernel<<<pages::CLUSTER, pages::THREADS, smem, reinterpret_cast<cudaStream_t>(stream)>>>(a);
  return cudaGetLastError() == cudaSuccess ? ATF_OK : ATF_ERR_CUDA;
}

extern "C" int atf_copy_pages(const AtfCopyPagesParams* p, atf_stream_t stream) {
  if (p == nullptr || p->tensors_host == nullptr || p->num_tensors < 1 || p->num_pairs < 0 || p->num_pages < 1 ||
      (p->num_pairs > 0 && (p->src == nullptr || p->dst == nullptr)))
    return ATF_ERR_INVALID_ARG;
  for (int i = 0; i < p->num_tensors; ++i) {
    const AtfPageTensor& t = p->tensors_host[i];
    if (t.base == nullptr || t.page_bytes < 1 || (p->num_pages > 1 && t.page_stride_bytes < t.page_bytes))
      return ATF_ERR_INVALID_ARG;
    if (t.page_bytes > (1ll << 40)) return ATF_ERR_UNSUPPORTED;
  }
  if (p->num_pairs == 0) return ATF_OK;
  int dev = 0;
  int rc = check_device(&dev);
  if (rc != ATF_OK) return rc;
  // MAX_TENSORS at a time: their descriptors are the kernel's parameters
  for (int i0 = 0; i0 < p->num_tensors; i0 += pages::MAX_TENSORS) {
    pages::CopyArgs a;
    a.src = p->src;
    a.dst = p->dst;
    a.n = p->num_pairs;
    a.P = p->num_pages;
    a.tensors = p->num_tensors - i0 < pages::MAX_TENSORS ? p->num_tensors - i0 : pages::MAX_TENSORS;
    a.err = p->error_flag;
    long long pieces = 0;
    for (int i = 0; i < a.tensors; ++i) {
      const AtfPageTensor& t = p->tensors_host[i0 + i];
      a.t[i].base = static_cast<uint8_t*>(t.base);
      a.t[i].stride = t.page_stride_bytes;
      a.t[i].bytes = t.page_bytes;
      a.first[i] = static_cast<int>(pieces);
      pieces += (t.page_bytes + pages::PIECE - 1) / pages::PIECE;
      if (pieces > 0x7fffffffLL) return ATF_ERR_UNSUPPORTED;
    }
    a.first[a.tensors] = static_cast<int>(pieces);
    a.pieces = static_cast<int>(pieces);
    const long long all = pieces * a.n, most = 148ll * 128;
    pages::copy_kernel<<<static_cast<unsigned>(all < most ? all : most), pages::COPY_THREADS, 0,
                         reinterpret_cast<cudaStream_t>(stream)>>>(a);
    if (cudaGetLastError() != cudaSuccess) return ATF_ERR_CUDA;
  }
  return ATF_OK;
}
