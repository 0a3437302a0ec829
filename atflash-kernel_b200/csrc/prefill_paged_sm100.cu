// Attention of a chunk of new tokens of each request over the pages of a cache, for
// sm_100a: one token (a decode), a few (drafted tokens to verify) or thousands (chunked
// prefill behind a cached prefix), in one batch.
//
// Mathematics and pipeline are the packed prefill's (prefill_ragged_sm100.cu): an online
// softmax in the log2 domain over 128-key tiles, S = Q K^T over the window's 16-dim levels
// and O += P V on the tensor cores with both accumulators in TMEM, P in bf16 (the tensor
// core's f16 kind has one type for both operands, and V is bf16), sums and statistics
// in fp32: off by 0.0021 to 0.0024 of the outputs' size from 64 bits, where the rounding of the
// bf16 outputs alone makes 0.0017. The window is quantised per tile of 128 queries and 128 keys of the request.
// Three things differ.
//
// Pages. A key tile is 128 / R slices of R = min(page, 128) rows. The K producer warp, and the
// V producer warp, read page ids 32 slices at a time, a batch ahead, and a lane per slice
// and half issues its box, {64 dims, R rows} with 128-byte swizzle, into the rows of the
// tile. So K lies as Q does: level i is 32 bytes into a row, and dims 64 and up are another
// 16 KB. Slices past the request's last page are not loaded; their keys are masked and their
// V rows cleared. (With ids read tile by tile the producers were what a step waited for: 2.2
// us for two tiles of rows against a key tile instead of 1.8, and long chunks 5.45 ms
// instead of 4.8.)
//
// Rows. A tile's 128 rows are 128 tokens of a query head, or, where that takes fewer
// tiles, 128 / G tokens with the G heads of a kv head side by side (row = token x G + head;
// one box of Q, since the heads of a token are G rows in memory): a chunk of 5 tokens
// with 7 heads a kv head reads K and V once instead of 7 times. No tile crosses a multiple of
// 128 tokens, so that its rows share the window's levels.
//
// Splits. A CTA has two tiles in flight (two softmax groups, 512 TMEM columns). Two
// tiles of rows against each key tile share K and V; a single tile of rows works on
// the even key tiles with one group and on the odd ones with the other, and the groups'
// states are joined in TMEM at the end (a row's lane is the same for both). Where
// there are fewer blocks than SMs, the plan also cuts the keys of a block over
// CTAs; their states go to a workspace (fp32) and merge_states_kernel joins them.
//
// What bounds it: HBM where rows are few (24 requests x 5 tokens over up to 16001 keys, 28 /
// 4 heads, pages of 16: 127 to 131 us replayed from a graph, 142 to 154 a call from cold memory;
// the floor is 113. A key tile takes
// 1.1 us from L2 and 1.5 with all SMs reading HBM, and a CTA's start and end 6 more); else
// the step of two tiles, as in the packed prefill (2 chunks of 8192 behind 24K keys, the
// window on: 4.9 to 5.0 ms, 61% of the burst rate; 4.3 in a few launches at a higher clock).
#include <math.h>

#include <algorithm>
#include <cstring>
#include <functional>
#include <queue>
#include <vector>

#include "atf_internal.h"
#include "atf_ptx.cuh"
#include "prefill_common.cuh"

namespace atf {
namespace paged {

using namespace prefill;

// The L (1..8) QK MMAs of a tile and the commit, both operands as two boxes of 64 dims in
// 128-byte rows (128-byte swizzle, 16 KB each): a level advances them by 32 bytes inside a
// row, and to the next box after four levels.
__device__ __forceinline__ void qk_rows_asm(uint32_t d_tmem, uint64_t qd, uint64_t kd, uint32_t idesc, int L,
                                            uint32_t bar_addr) {
  asm volatile(
      "{\n\t.reg .pred pe, p1, p2, p3, p4, p5, p6, p7;\n\t.reg .b64 a, b;\n\t"
      "elect.sync _|pe, 0xffffffff;\n\t"
      "setp.gt.and.s32 p1, %4, 1, pe;\n\tsetp.gt.and.s32 p2, %4, 2, pe;\n\tsetp.gt.and.s32 p3, %4, 3, pe;\n\t"
      "setp.gt.and.s32 p4, %4, 4, pe;\n\tsetp.gt.and.s32 p5, %4, 5, pe;\n\tsetp.gt.and.s32 p6, %4, 6, pe;\n\t"
      "setp.gt.and.s32 p7, %4, 7, pe;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, 0;\n\t"
      "add.u64 a, %1, 2;\n\tadd.u64 b, %2, 2;\n\t"
      "@p1 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 2;\n\tadd.u64 b, b, 2;\n\t"
      "@p2 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 2;\n\tadd.u64 b, b, 2;\n\t"
      "@p3 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 1018;\n\tadd.u64 b, b, 1018;\n\t"
      "@p4 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 2;\n\tadd.u64 b, b, 2;\n\t"
      "@p5 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 2;\n\tadd.u64 b, b, 2;\n\t"
      "@p6 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 2;\n\tadd.u64 b, b, 2;\n\t"
      "@p7 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "@pe tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t}"
      ::"r"(d_tmem), "l"(qd), "l"(kd), "r"(idesc), "r"(L), "r"(bar_addr)
      : "memory");
}

constexpr int WARP_V = 10;  // the producer of Q and V (WARP_LOAD: K)
constexpr uint32_t QBOX_BYTES = QTILE_BYTES / 2;
// Shared memory: seven slots of 32 KB. Two tiles of Q, two stages of K and three of V; or one
// tile of Q and three stages each where the groups share out the keys, where a step takes
// two of each.
constexpr int V_STAGES = 3;
template <bool SPLIT_KEYS>
constexpr int K_STAGES = SPLIT_KEYS ? 3 : 2;
constexpr uint32_t SLOT = 32 * 1024;
static_assert(QTILE_BYTES == SLOT && KSTAGE_BYTES == SLOT && VSTAGE_BYTES == SLOT, "one size for all");
constexpr uint32_t OFF_Q = 0;
template <bool SPLIT_KEYS>
constexpr uint32_t OFF_K = (SPLIT_KEYS ? 1 : 2) * SLOT;
constexpr uint32_t OFF_V = 4 * SLOT;
constexpr uint32_t OFF_STATE = 3 * SLOT;  // [t][128] of (max, sum), in K's place once all products are done
constexpr uint32_t OFF_BAR = 7 * SLOT;

enum {
  B_Q = 0,
  B_KFULL = 1,
  B_KEMPTY = B_KFULL + 3,
  B_VFULL = B_KEMPTY + 3,
  B_VEMPTY = B_VFULL + V_STAGES,
  B_SFULL = B_VEMPTY + V_STAGES,  // [t]
  B_PFULL = B_SFULL + NQ,     // [t]
  B_ODONE = B_PFULL + NQ,     // [t], one phase per O += P V
  B_OFINAL = B_ODONE + NQ,    // [t], single phase: the group's last O += P V done
  B_LOADED = B_OFINAL + NQ,   // [t], phase i: group t has read its i-th S into registers
  B_FINAL = B_LOADED + NQ,
  NUM_BARS
};
constexpr uint32_t OFF_PLACE = OFF_BAR + 8 * ((NUM_BARS + 1) / 2 * 2);  // Place
constexpr uint32_t OFF_ROWS = OFF_PLACE + 48;  // [t][128] of where a row goes
constexpr uint32_t OFF_ABORT = OFF_ROWS + NQ * BM * 4;
constexpr uint32_t OFF_TMEM = OFF_ABORT + 16;
constexpr uint32_t SMEM_BYTES = OFF_TMEM + 16 + 1024;  // slack for 1024-B alignment
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory of a CTA");

enum { PACKED = 1, SPLIT = 2 };
// One work item: the rows of one or two tiles of a request against the key tiles [kt0,
// kt1). Tokens are the request's own; tile 0 holds n0 from `row` on, tile 1 the n1 after
// them (0 in a SPLIT item, whose two groups share tile 0).
struct Item {
  int q_tok, q_len, k_len, page_beg;  // first packed query row, queries, keys, first entry of the page list
  int row, n0, n1, flags;
  int kt0, kt1, part, n_parts;        // part: workspace slot of the first token, -1: the outputs
};
static_assert(sizeof(Item) == 4 * ATF_PAGED_ITEM_INTS, "the header's item size");

struct Args {
  int Hq, Hkv, G, T;   // T = 128 / G tokens of a packed tile
  int walk;            // heads of an unpacked item that lie next to each other in the grid
  float scale_log2;
  int causal, window;
  int zhi[ATF_MAX_LEVELS];
  __nv_bfloat16* out;
  long long o_ss, o_sh;
  float* lse;
  float* part_o;
  float* part_lse;
  long long parts;     // slots in the workspace
  int* err;
  const int* items;
  int n_wide, n_items; // unpacked items come first
  long long total_q;
  const int* indices;
  int num_indices, num_pages, page_shift, row_shift;  // of the page size and of R
  int merge;           // a merge of states follows
};

// key tile j reads level i when j >= lim[i]
__device__ __forceinline__ void window_limits(const Args& a, int q_offset, int row0, int (&lim)[ATF_MAX_LEVELS]) {
  const long long base = static_cast<long long>(q_offset) + row0 / BM * BM - (BN - 1);
#pragma unroll
  for (int i = 0; i < ATF_MAX_LEVELS; ++i) {
    const long long x = base - a.zhi[i];
    lim[i] = (!a.window || i == 0 || x <= 0) ? 0 : static_cast<int>((x + BN - 1) / BN);
  }
}

// What the warps of a CTA share
struct Unit {
  uint32_t sb;      // aligned shared memory
  uint8_t* sp;
  uint32_t tmem;
  AbortCtl ab;
  int sk, q_offset, row0, n0, n1, kt0, page_beg;
  int nk[NQ];       // key tiles of each group
  int hk, P;        // heads side by side in a tile
  int lim[NQ][ATF_MAX_LEVELS];
  __device__ __forceinline__ uint32_t bar(int i) const { return sb + OFF_BAR + 8u * static_cast<uint32_t>(i); }
};

// Where the rows go, in shared memory: the softmax groups have no registers left for it
// until their loop is done.
struct Place {
  int q_tok, row0, part, n_parts, head0, P, n0, n1;
  int nk[NQ], pad[2];
};
static_assert(sizeof(Place) == 48, "its room in shared memory");

// The key tile of a group's i-th step, and its place in the order of all loads
template <bool SPLIT_KEYS>
__device__ __forceinline__ int nth(int t, int i) {
  return SPLIT_KEYS ? 2 * i + t : i;
}

// Page id of slice 32 batch + lane of the item's key tiles (-1: no such slice). A batch is 32
// slices, so 4 (pages of 16) to 32 key tiles; one is read while another is used.
__device__ __forceinline__ int slice_page(const Args& a, const Unit& u, int batch, int lane) {
  const int key = u.kt0 * BN + ((32 * batch + lane) << a.row_shift);
  const unsigned at = static_cast<unsigned>(u.page_beg + (key >> a.page_shift));
  return key < u.sk && at < static_cast<unsigned>(a.num_indices) ? __ldg(a.indices + at) : -1;
}

// The loads of K or V, tile by tile: lane = half x slices + slice issues the box of its
// slice and half. An id outside the cache is a coordinate outside the map, which reads
// zeros; it is reported.
template <bool SPLIT_KEYS>
__device__ __forceinline__ void produce(const Args& a, const Unit& u, const CUtensorMap* map, bool is_k, int ids, int lane) {
  const int tiles = SPLIT_KEYS ? u.nk[0] + u.nk[1] : max(u.nk[0], u.nk[1]);
  const int stages = is_k ? K_STAGES<SPLIT_KEYS> : V_STAGES;
  const int full = is_k ? B_KFULL : B_VFULL, empty = is_k ? B_KEMPTY : B_VEMPTY;
  const int slices_shift = 7 - a.row_shift, slices = 1 << slices_shift;
  const int slice = lane & (slices - 1), half = lane >> slices_shift, first_row = slice << a.row_shift;
  const uint32_t dst = u.sb + (is_k ? OFF_K<SPLIT_KEYS> : OFF_V) + half * (BN * 128) + first_row * 128;
  int issued = 0, later = slice_page(a, u, 1, lane);
  for (int g = 0; g < tiles; ++g) {
    const int s = g % stages, kt = u.kt0 + g, at = g << slices_shift;
    if (g > 0 && (at & 31) == 0) {  // the next batch of page ids
      ids = later;
      later = slice_page(a, u, (at >> 5) + 1, lane);
    }
    const int id = __shfl_sync(FULL, ids, (at + slice) & 31);
    int halves = 2;
    if (is_k && a.window) {  // the second 64 dims are levels 4 to 7
      int L = 0;
#pragma unroll
      for (int t = 0; t < NQ; ++t)
        if (SPLIT_KEYS ? t == 0 : g < u.nk[t]) L = max(L, levels_for(u.lim[t], kt));
      halves = L > 4 ? 2 : 1;
    }
    // slices of the tile before the request's last key
    const int live = min(slices, (u.sk - kt * BN + (1 << a.row_shift) - 1) >> a.row_shift);
    if (!__all_sync(FULL, mbar_wait_inl(u.bar(empty + s), ((g / stages) & 1) ^ 1, u.ab, kDevErrTimeout))) break;
    mbar_arrive_expect_tx_elect(u.bar(full + s), static_cast<uint32_t>(live * halves) << (a.row_shift + 7));
    __syncwarp();
    if (half < halves && slice < live) {
      if ((id < 0 || id >= a.num_pages) && a.err != nullptr) atomicCAS(a.err, 0, kDevErrIndex);
      tma_load_4d(dst + s * SLOT, map, u.bar(full + s), 64 * half, (kt * BN + first_row) & ((1 << a.page_shift) - 1), u.hk,
                  id);
    }
    __syncwarp();
    issued = g + 1;
  }
  // Every copy this warp issued lands before shared memory is released (no wait on the
  // normal path, where the MMA warp consumed them).
  for (int g = issued - stages; g < issued; ++g)
    if (g >= 0) drain_wait(u.bar(full + g % stages), (g / stages) & 1);
  __syncwarp();
}

template <bool SPLIT_KEYS>
__device__ __forceinline__ void issue_mmas(const Args& a, const Unit& u, int lane) {
  constexpr int KS = K_STAGES<SPLIT_KEYS>, VS = V_STAGES;
  const uint32_t tm = __shfl_sync(FULL, u.tmem, 0);
  const uint64_t qdesc0 = make_sdesc(u.sb + OFF_Q, 16, 1024, kLayoutSw128);
  const uint64_t kdesc0 = make_sdesc(u.sb + OFF_K<SPLIT_KEYS>, 16, 1024, kLayoutSw128);
  const uint64_t vdesc0 = make_sdesc(u.sb + OFF_V, VBOX_BYTES, 1024, kLayoutSw128);
  const int nk0 = u.nk[0], nk1 = u.nk[1], nk_max = max(nk0, nk1);
  // S_t(i) into group t's S columns
  auto issue_S = [&](int t, int i) {
    const int g = nth<SPLIT_KEYS>(t, i);
    const int L = levels_for(u.lim[SPLIT_KEYS ? 0 : t], u.kt0 + g);
    qk_rows_asm(tm + static_cast<uint32_t>(t * 128), qdesc0 + (SPLIT_KEYS ? 0 : (t * QTILE_BYTES) >> 4),
                kdesc0 + (((g % KS) * SLOT) >> 4), IDESC_QK, L, u.bar(B_SFULL + t));
  };
  // O_t += P_t(i) V; P_t sits in columns 64..127 of the other group's S
  auto issue_PV = [&](int t, int i) {
    const uint64_t vd = vdesc0 + (((nth<SPLIT_KEYS>(t, i) % VS) * SLOT) >> 4);
    pv_group_asm(tm + 256u + static_cast<uint32_t>(t * 128), tm + static_cast<uint32_t>((1 - t) * 128 + 64), vd, IDESC_PV,
                 i > 0 ? 1u : 0u, u.bar(B_ODONE + t));
  };
  // stages are waited for in order, once each
  int k_waited = -1;
  auto kwait = [&](int g) -> bool {
    while (k_waited < g) {
      ++k_waited;
      if (!__all_sync(FULL, mbar_wait_inl(u.bar(B_KFULL + k_waited % KS), (k_waited / KS) & 1, u.ab, kDevErrTimeout)))
        return false;
      tc_fence_after();
    }
    return true;
  };
  auto vwait = [&](int g) -> bool {
    if (!__all_sync(FULL, mbar_wait_inl(u.bar(B_VFULL + g % VS), (g / VS) & 1, u.ab, kDevErrTimeout))) return false;
    // V rows past the request's last key hold another time's bytes, or nothing
    const int live = u.sk - (u.kt0 + g) * BN;
    if (live < BN) {
      uint8_t* v0 = u.sp + OFF_V + (g % VS) * SLOT;
      for (int e = live * 8 + lane; e < BN * 8; e += 32) {
        *reinterpret_cast<uint4*>(v0 + 16 * e) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(v0 + VBOX_BYTES + 16 * e) = make_uint4(0, 0, 0, 0);
      }
      // the MMAs read V through the async proxy
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    }
    tc_fence_after();
    return true;
  };
  auto wait_for = [&](int which, int t, int i) -> bool {
    const bool w = __all_sync(FULL, mbar_wait_inl(u.bar(which + t), i & 1, u.ab, kDevErrTimeout));
    tc_fence_after();
    return w;
  };
  // A K stage is released after the last S that reads it: with split keys its only one,
  // else S_1(i) where tile 1 has key tile i, or S_0(i).
  bool ok = wait_for(B_Q, 0, 0);
  if (ok && nk_max > 0 && (ok = kwait(0))) {
    if (nk0 > 0) issue_S(0, 0);
    if (SPLIT_KEYS) tc_commit_elect(u.bar(B_KEMPTY + 0));
    if (nk1 > 0 && (!SPLIT_KEYS || (ok = kwait(1)))) issue_S(1, 0);
    if (!SPLIT_KEYS || nk1 > 0) tc_commit_elect(u.bar(B_KEMPTY + (SPLIT_KEYS ? 1 : 0)));
  }
  // S_0(1) once group 0 has read S_0(0)
  if (ok && nk0 > 1 && (ok = kwait(nth<SPLIT_KEYS>(0, 1)) && wait_for(B_LOADED, 0, 0))) {
    issue_S(0, 1);
    if (SPLIT_KEYS || 1 >= nk1) tc_commit_elect(u.bar(B_KEMPTY + nth<SPLIT_KEYS>(0, 1) % KS));
  }
  for (int i = 0; ok && i < nk_max; ++i) {
    if (!SPLIT_KEYS && !(ok = vwait(i))) break;
    if (i < nk0) {
      if (SPLIT_KEYS && !(ok = vwait(2 * i))) break;
      if (!(ok = wait_for(B_PFULL, 0, i))) break;
      issue_PV(0, i);
      if (i + 1 == nk0) tc_commit_elect(u.bar(B_OFINAL + 0));
      if (SPLIT_KEYS) tc_commit_elect(u.bar(B_VEMPTY + (2 * i) % VS));
    }
    // S_1(i+1) overwrites the columns P_0(i) occupies (O_0 += P_0(i) V was issued first;
    // tcgen05.mma ops of one thread run in order) and needs group 1 to have read S_1(i)
    if (i + 1 < nk1) {
      if (!(ok = kwait(nth<SPLIT_KEYS>(1, i + 1)) && wait_for(B_LOADED, 1, i))) break;
      issue_S(1, i + 1);
      tc_commit_elect(u.bar(B_KEMPTY + nth<SPLIT_KEYS>(1, i + 1) % KS));
    }
    if (i < nk1) {
      if (SPLIT_KEYS && !(ok = vwait(2 * i + 1))) break;
      if (!(ok = wait_for(B_PFULL, 1, i))) break;
      issue_PV(1, i);
      if (i + 1 == nk1) tc_commit_elect(u.bar(B_OFINAL + 1));
      if (SPLIT_KEYS) tc_commit_elect(u.bar(B_VEMPTY + (2 * i + 1) % VS));
    }
    // S_0(i+2): after O_1 += P_1(i) V (P_1(i) sits in S_0's columns) and group 0's read
    // of S_0(i+1)
    if (i + 2 < nk0) {
      if (!(ok = kwait(nth<SPLIT_KEYS>(0, i + 2)) && wait_for(B_LOADED, 0, i + 1))) break;
      issue_S(0, i + 2);
      if (SPLIT_KEYS || i + 2 >= nk1) tc_commit_elect(u.bar(B_KEMPTY + nth<SPLIT_KEYS>(0, i + 2) % KS));
    }
    if (!SPLIT_KEYS) tc_commit_elect(u.bar(B_VEMPTY + i % VS));
  }
  // Every MMA issued by this CTA completes before TMEM is released.
  tc_commit_elect(u.bar(B_FINAL));
  __syncwarp();
  drain_wait(u.bar(B_FINAL), 0);
  __syncwarp();
}

// Where row r of a tile goes, in steps of 16 bytes from the outputs' or the states' first
// (NO_ROW: it is not one of the tile's). Found by the softmax threads while the CTA is set
// up: divisions at its end cost 1 to 10 us.
constexpr uint32_t NO_ROW = 0xffffffffu;
__device__ __forceinline__ uint32_t row_place(const Args& a, const Place& to, int t, int r) {
  if (r >= (t ? to.n1 : to.n0) * to.P) return NO_ROW;
  const int k = r / to.P, tok = to.row0 + (t ? to.n0 : 0) + k, head = to.head0 + r - k * to.P;
  if (to.part < 0)
    return static_cast<uint32_t>(((to.q_tok + tok) * a.o_ss + head * a.o_sh) >> 3);
  return static_cast<uint32_t>(((to.part + static_cast<long long>(tok - to.row0) * to.n_parts) * a.Hq + head) * 32);
}

// 64 dims of a warp's 32 rows (v: this lane's row) from dim 64 half on, through `stage`
// (4 KB): rows of 128 bytes, 16-byte chunks XORed with the row, then eight lanes per row,
// so that whole 128-byte lines leave. place: of the warp's rows.
__device__ __forceinline__ void store_half(const Args& a, const uint32_t* place, bool out, int half, uint8_t* stage, int lane,
                                           const float (&v)[64]) {
  const int lr = lane >> 3, c = lane & 7;
  if (out) {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      *reinterpret_cast<uint4*>(stage + lane * 128 + 16 * (q ^ (lane & 7))) =
          make_uint4(pack_bf16x2(v[8 * q], v[8 * q + 1]), pack_bf16x2(v[8 * q + 2], v[8 * q + 3]),
                     pack_bf16x2(v[8 * q + 4], v[8 * q + 5]), pack_bf16x2(v[8 * q + 6], v[8 * q + 7]));
    __syncwarp();
    uint4* to = reinterpret_cast<uint4*>(a.out) + 8 * half + c;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + lr;
      const uint4 x = *reinterpret_cast<const uint4*>(stage + r * 128 + 16 * (c ^ (r & 7)));
      const uint32_t at = place[r];
      if (at != NO_ROW) to[at] = x;
    }
    __syncwarp();
    return;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      *reinterpret_cast<float4*>(stage + lane * 128 + 16 * (q ^ (lane & 7))) =
          make_float4(v[32 * k + 4 * q], v[32 * k + 4 * q + 1], v[32 * k + 4 * q + 2], v[32 * k + 4 * q + 3]);
    __syncwarp();
    float4* to = reinterpret_cast<float4*>(a.part_o) + 16 * half + 8 * k + c;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + lr;
      const float4 x = *reinterpret_cast<const float4*>(stage + r * 128 + 16 * (c ^ (r & 7)));
      const uint32_t at = place[r];
      if (at != NO_ROW) to[at] = x;
    }
    __syncwarp();
  }
}

template <bool SPLIT_KEYS>
__device__ __forceinline__ void softmax(const Args& a, const Unit& u, int warp, int lane) {
  const int t = warp >> 2, wq = warp & 3;
  const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
  const uint32_t tS = u.tmem + static_cast<uint32_t>(t * 128) + lane_off;
  const uint32_t tP = u.tmem + static_cast<uint32_t>((1 - t) * 128 + 64) + lane_off;
  const uint32_t tO = u.tmem + 256u + static_cast<uint32_t>(t * 128) + lane_off;
  const int my_nk = t ? u.nk[1] : u.nk[0], other_nk = t ? u.nk[0] : u.nk[1];
  const int tok0 = u.row0 + (!SPLIT_KEYS && t ? u.n0 : 0);      // the tile's first token
  // keys that this row still sees from the step's key tile on, and that the tile's first row
  // sees: under 128, some row of the tile does not see every key
  int left = (a.causal ? min(u.sk, u.q_offset + tok0 + (wq * 32 + lane) / u.P + 1) : u.sk) - (u.kt0 + nth<SPLIT_KEYS>(t, 0)) * BN;
  int left0 = (a.causal ? min(u.sk, u.q_offset + tok0 + 1) : u.sk) - (u.kt0 + nth<SPLIT_KEYS>(t, 0)) * BN;
  const float sl2 = a.scale_log2;
  float m2 = -INFINITY, l = 0.f;
  bool ok = true;
  for (int i = 0; i < my_nk; ++i) {
    ok = __all_sync(FULL, mbar_wait_inl(u.bar(B_SFULL + t), i & 1, u.ab, kDevErrTimeout));
    if (!ok) break;
    tc_fence_after();
    float s[BN];
    {
      uint32_t rr[BN];
      tmem_ld128(tS, rr);
#pragma unroll
      for (int e = 0; e < BN; ++e) s[e] = __uint_as_float(rr[e]);
    }
    // S_t's columns are free now: the MMA warp may compute the next S_t into them, and the
    // other group may store its P there
    tc_fence_before();
    mbar_arrive(u.bar(B_LOADED + t));
    if (left0 < BN) {
#pragma unroll
      for (int c = 0; c < BN; ++c) s[c] = c < left ? s[c] : -INFINITY;
    }
    left -= (SPLIT_KEYS ? 2 : 1) * BN;
    left0 -= (SPLIT_KEYS ? 2 : 1) * BN;
    // three-input max: 64 instructions for the 128 scores, 4 chains
    float mx0 = fmax3(s[0], s[1], s[2]), mx1 = fmax3(s[3], s[4], s[5]);
    float mx2 = fmax3(s[6], s[7], s[8]), mx3 = fmax3(s[9], s[10], s[11]);
#pragma unroll
    for (int c = 12; c < BN - 8; c += 8) {
      mx0 = fmax3(mx0, s[c], s[c + 1]);
      mx1 = fmax3(mx1, s[c + 2], s[c + 3]);
      mx2 = fmax3(mx2, s[c + 4], s[c + 5]);
      mx3 = fmax3(mx3, s[c + 6], s[c + 7]);
    }
    mx0 = fmax3(mx0, s[BN - 4], s[BN - 3]);
    mx1 = fmax3(mx1, s[BN - 2], s[BN - 1]);
    const float mnew = fmaxf(m2, fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * sl2);
    // Lazy rescale: the running max only moves when it grows by more than 8 (log2 units), so
    // P <= 2^8 stays exact enough in bf16 and O is rescaled rarely. The O update itself
    // happens after P is stored.
    float alpha = 1.0f;
    bool need = false;
    if (i == 0) {
      m2 = mnew;
    } else {
      need = mnew > m2 + 8.0f;
      if (need) {
        alpha = ex2_approx(m2 - mnew);
        l *= alpha;
        m2 = mnew;
      }
    }
    const float msub = (m2 == -INFINITY) ? 0.f : m2;
    // exponentials, the row sum and the bf16 packing of P, two columns at a time with packed
    // f32x2 arithmetic
    uint32_t pk[BN / 2];
    float2 ls0 = make_float2(0.f, 0.f), ls1 = make_float2(0.f, 0.f);
    const float2 sl2x2 = make_float2(sl2, sl2), negm = make_float2(-msub, -msub);
#pragma unroll
    for (int c = 0; c < BN / 2; ++c) {
      const float2 x = __ffma2_rn(make_float2(s[2 * c], s[2 * c + 1]), sl2x2, negm);
      const float2 p = make_float2(ex2_approx(x.x), ex2_approx(x.y));
      if (c & 1) ls1 = __fadd2_rn(ls1, p); else ls0 = __fadd2_rn(ls0, p);
      pk[c] = pack_bf16x2(p.x, p.y);
    }
    {
      const float2 ls = __fadd2_rn(ls0, ls1);
      l += ls.x + ls.y;
    }
    // P_t(i) goes into columns 64..127 of the other group's S once the scores there have
    // been read: S_1(i) for group 0, S_0(i+1) for group 1 (whose computation followed O_1 +=
    // P_1(i-1) V, the last reader of those columns). Past the other group's last step,
    // wait for its last read and for this group's previous O += P V instead.
    {
      const int want = i + t;
      bool w = true;
      if (want < other_nk) {
        w = mbar_wait_inl(u.bar(B_LOADED + (t ^ 1)), want & 1, u.ab, kDevErrTimeout);
      } else {
        if (other_nk > 0) w = mbar_wait_inl(u.bar(B_LOADED + (t ^ 1)), (other_nk - 1) & 1, u.ab, kDevErrTimeout);
        if (w && i > 0) w = mbar_wait_inl(u.bar(B_ODONE + t), (i - 1) & 1, u.ab, kDevErrTimeout);
      }
      ok = __all_sync(FULL, w);
      if (!ok) break;
      tc_fence_after();
    }
    tmem_st64(tP, pk);
    if (__any_sync(FULL, need)) {
      // O holds the sum up to step i-1 once that product has completed (S_t(i) was issued
      // after it, so at most that one is in flight); this step's is not issued before this
      // warpgroup arrives on PFULL below.
      ok = __all_sync(FULL, mbar_wait_inl(u.bar(B_ODONE + t), (i - 1) & 1, u.ab, kDevErrTimeout));
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int c4 = 0; c4 < HD / 32; ++c4) {
        uint32_t rr[32];
        tmem_ld32(tO + static_cast<uint32_t>(32 * c4), rr);
#pragma unroll
        for (int e = 0; e < 32; ++e) rr[e] = __float_as_uint(__uint_as_float(rr[e]) * alpha);
        tmem_st32(tO + static_cast<uint32_t>(32 * c4), rr);
      }
    }
    tc_fence_before();
    mbar_arrive(u.bar(B_PFULL + t));
  }

  float lse2;  // log2 of the row's sum
  const int r = wq * 32 + lane;
  const Place& to = *reinterpret_cast<const Place*>(u.sp + OFF_PLACE);
  const bool out = to.part < 0;
  const int tile = SPLIT_KEYS ? 0 : t;
  const uint32_t* place = reinterpret_cast<const uint32_t*>(u.sp + OFF_ROWS) + tile * BM + wq * 32;
  float v[64];
  if (SPLIT_KEYS) {
    // both groups' states of the row: (max, sum) through shared memory, O from TMEM, where
    // the row has the same lane in both. Group t stores half t of the dims.
    float2* state = reinterpret_cast<float2*>(u.sp + OFF_STATE);
#pragma unroll
    for (int k = 0; k < NQ; ++k)
      if (ok && to.nk[k] > 0) ok = __all_sync(FULL, mbar_wait_inl(u.bar(B_OFINAL + k), 0, u.ab, kDevErrTimeout));
    // (without keys nothing has read Q, whose place the outputs take)
    if (ok && to.nk[0] == 0) ok = __all_sync(FULL, mbar_wait_inl(u.bar(B_Q), 0, u.ab, kDevErrTimeout));
    tc_fence_after();
    if (ok) state[t * BM + r] = make_float2(m2, l);
    __syncwarp();
    asm volatile("bar.sync 1, 256;" ::: "memory");  // every softmax thread of the CTA comes here
    if (!ok) return;
    const float2 s0 = state[r], s1 = state[BM + r];
    const float m = fmaxf(s0.x, s1.x);
    const float w0 = s0.x == -INFINITY ? 0.f : ex2_approx(s0.x - m), w1 = s1.x == -INFINITY ? 0.f : ex2_approx(s1.x - m);
    l = s0.y * w0 + s1.y * w1;
    lse2 = m + log2f(l);
    const bool keyless = l == 0.f;  // no key, or none with weight: 0, whatever V holds
    const float inv = l > 0.f ? 1.0f / l : 0.f;
    const float f0 = w0 * inv, f1 = w1 * inv;
    const uint32_t tO0 = tO + static_cast<uint32_t>(64 * t - 128 * t);
    uint32_t rr[64];
    if (to.nk[0] > 0) {  // (the same for every thread of the CTA)
      tmem_ld64(tO0, rr);
#pragma unroll
      for (int e = 0; e < 64; ++e) v[e] = keyless ? 0.f : __uint_as_float(rr[e]) * f0;
    } else {
#pragma unroll
      for (int e = 0; e < 64; ++e) v[e] = 0.f;
    }
    if (to.nk[1] > 0) {
      tmem_ld64(tO0 + 128u, rr);
#pragma unroll
      for (int e = 0; e < 64; ++e) v[e] = keyless ? 0.f : fmaf(__uint_as_float(rr[e]), f1, v[e]);
    }
    store_half(a, place, out, t, u.sp + OFF_Q + warp * 4096, lane, v);
    if (t != 0) return;
  } else {
    if (!ok || (t ? to.n1 : to.n0) == 0) return;
    // through the tile's own Q in shared memory (its last product has read it; a tile without
    // keys has no products)
    if (!__all_sync(FULL, mbar_wait_inl(u.bar(my_nk > 0 ? B_OFINAL + t : B_Q), 0, u.ab, kDevErrTimeout))) return;
    tc_fence_after();
    const bool keyless = l == 0.f;  // no key, or none with weight: 0, whatever V holds
    const float inv = l > 0.f ? 1.0f / l : 0.f;
    lse2 = m2 + log2f(l);
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      if (my_nk > 0) {
        uint32_t rr[64];
        tmem_ld64(tO + static_cast<uint32_t>(64 * half), rr);
#pragma unroll
        for (int e = 0; e < 64; ++e) v[e] = keyless ? 0.f : __uint_as_float(rr[e]) * inv;
      } else {
#pragma unroll
        for (int e = 0; e < 64; ++e) v[e] = 0.f;
      }
      store_half(a, place, out, half, u.sp + OFF_Q + t * QTILE_BYTES + wq * 4096, lane, v);
    }
  }
  if (place[lane] != NO_ROW && (!out || a.lse != nullptr)) {
    const int k = r / to.P, tok = to.row0 + (tile ? to.n0 : 0) + k, head = to.head0 + r - k * to.P;
    if (!out)
      a.part_lse[(to.part + static_cast<long long>(tok - to.row0) * to.n_parts) * a.Hq + head] = lse2;
    else
      a.lse[static_cast<long long>(to.q_tok + tok) * a.Hq + head] = lse2 * 0.69314718055994531f;
  }
}

__global__ void __launch_bounds__(THREADS, 1)
    paged_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQP,
                 const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  Unit u;
  u.sb = (raw_u32 + 1023u) & ~1023u;
  u.sp = smem_raw + (u.sb - raw_u32);
  volatile int* s_abort = reinterpret_cast<volatile int*>(u.sp + OFF_ABORT);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(u.sp + OFF_TMEM);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  // This CTA's item and head: unpacked items go by query heads, packed ones by kv heads
  int item, h;
  const int bid = static_cast<int>(blockIdx.x), wide = a.n_wide * a.Hq;
  if (bid < wide) {
    const int per_walk = a.n_wide * a.walk, rem = bid % per_walk;
    h = bid / per_walk * a.walk + rem % a.walk;
    u.hk = h / a.G;
    item = rem / a.walk;
  } else {
    u.hk = (bid - wide) % a.Hkv;
    h = u.hk * a.G;
    item = a.n_wide + (bid - wide) / a.Hkv;
  }
  const int4* src = reinterpret_cast<const int4*>(a.items) + 3 * item;
  const int4 it0 = __ldg(src), it1 = __ldg(src + 1), it2 = __ldg(src + 2);
  const bool stop0 = threadIdx.x == 0 && stops(a.err);
  if (threadIdx.x == 0) {
    mbar_init(u.bar(B_Q), 1);
    for (int s = 0; s < 3; ++s) {
      mbar_init(u.bar(B_KFULL + s), 1);
      mbar_init(u.bar(B_KEMPTY + s), 1);
    }
    for (int s = 0; s < V_STAGES; ++s) {
      mbar_init(u.bar(B_VFULL + s), 1);
      mbar_init(u.bar(B_VEMPTY + s), 1);
    }
    for (int t = 0; t < NQ; ++t) {
      mbar_init(u.bar(B_SFULL + t), 1);
      mbar_init(u.bar(B_PFULL + t), 128);
      mbar_init(u.bar(B_ODONE + t), 1);
      mbar_init(u.bar(B_OFINAL + t), 1);
      mbar_init(u.bar(B_LOADED + t), 128);
    }
    mbar_init(u.bar(B_FINAL), 1);
    fence_mbar_init();
  }
  if (warp == WARP_LOAD && lane == 0) tma_prefetch_desc(&tmK);
  if (warp == WARP_V && lane == 0) {
    tma_prefetch_desc(bid < wide ? &tmQ : &tmQP);
    tma_prefetch_desc(&tmV);
  }
  if (warp == WARP_MMA) {
    tmem_alloc(smem_u32(s_tmem), 512);
    tmem_relinquish();
  }
  // the merge of the states may be launched: it waits for this grid before it reads them
  if (a.merge) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  u.sk = it0.z;
  u.q_offset = it0.z - it0.y;  // position of the request's query 0 among its keys (negative: rows without keys)
  u.page_beg = it0.w;
  u.row0 = it1.x;
  u.n0 = it1.y;
  u.n1 = it1.z;
  u.kt0 = it2.x;
  const bool packed = (it1.w & PACKED) != 0;
  u.P = packed ? a.G : 1;
  const bool split = (it1.w & SPLIT) != 0;
  const int tile_tokens = packed ? a.T : BM;
  // An item outside the query rows, the page list or the workspace (a plan made for
  // others) has no rows.
  const long long last_tok = static_cast<long long>(it1.x) + it1.y + it1.z;
  const bool bad = it0.x < 0 || it0.y < 0 || it0.z < 0 || it0.w < 0 || it1.x < 0 || it1.y < 1 || it1.z < 0 ||
                   it1.y > tile_tokens || it1.z > tile_tokens || (split && it1.z != 0) || last_tok > it0.y ||
                   it0.x + static_cast<long long>(it0.y) > a.total_q || it2.x < 0 || it2.y < it2.x ||
                   packed != (bid >= wide) ||
                   it0.w + ((static_cast<long long>(it0.z) + (1 << a.page_shift) - 1) >> a.page_shift) > a.num_indices ||
                   (it2.z >= 0 && (it2.w < 1 || it2.z + (static_cast<long long>(it1.y) + it1.z - 1) * it2.w >= a.parts));
  if (bad) u.n0 = u.n1 = 0;
  if (threadIdx.x == 0) {
    *s_abort = stop0 ? 1 : 0;
    if (bad && a.err != nullptr) atomicCAS(a.err, 0, kDevErrIndex);
  }
#pragma unroll
  for (int t = 0; t < NQ; ++t) {
    const int n = t ? u.n1 : u.n0, first = u.row0 + (t ? u.n0 : 0);
    // key tiles that the tile's last row sees, of those of the item
    const int kend = a.causal ? min(u.q_offset + first + n, u.sk) : u.sk;
    const int end = min(it2.y, kend > 0 ? (kend + BN - 1) / BN : 0);
    u.nk[t] = n > 0 ? max(0, end - u.kt0) : 0;
    window_limits(a, u.q_offset, first, u.lim[t]);
  }
  if (split) {
    u.nk[1] = u.nk[0] / 2;
    u.nk[0] -= u.nk[1];
  }
  if (warp < 8) {
    const Place to = {it0.x, u.row0, it2.z, it2.w, h, u.P, u.n0, u.n1, {u.nk[0], u.nk[1]}, {0, 0}};
    reinterpret_cast<uint32_t*>(u.sp + OFF_ROWS)[threadIdx.x] = row_place(a, to, warp >> 2, threadIdx.x & (BM - 1));
    if (threadIdx.x == 0) *reinterpret_cast<Place*>(u.sp + OFF_PLACE) = to;
  }

  // the producers' first page ids: on their way over the barrier
  const int first_id = warp == WARP_LOAD || warp == WARP_V ? slice_page(a, u, 0, lane) : -1;

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  u.tmem = *s_tmem;
  u.ab = AbortCtl{s_abort, a.err};
  const bool start_ok = (*s_abort == 0);
  if (warp >= 8) {
    reg_dealloc<REG_SMALL>();
    if (start_ok && warp == WARP_LOAD) {
      if (split)
        produce<true>(a, u, &tmK, true, first_id, lane);
      else
        produce<false>(a, u, &tmK, true, first_id, lane);
    } else if (start_ok && warp == WARP_V) {
      // Q (rows of 128 bytes, two boxes of 64 dims a tile), which the first S needs, then V
      const uint32_t qbytes = static_cast<uint32_t>(tile_tokens * u.P) * 256u;
      const int n_q = (u.n0 > 0 ? 1 : 0) + (u.n1 > 0 ? 1 : 0);
      mbar_arrive_expect_tx_elect(u.bar(B_Q), n_q * qbytes);
      for (int t = 0; t < n_q; ++t)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          tma_load_4d_elect(u.sb + OFF_Q + t * QTILE_BYTES + half * QBOX_BYTES, bid < wide ? &tmQ : &tmQP, u.bar(B_Q),
                            64 * half, h, it0.x + u.row0 + (t ? u.n0 : 0), 0);
      __syncwarp();
      if (split)
        produce<true>(a, u, &tmV, false, first_id, lane);
      else
        produce<false>(a, u, &tmV, false, first_id, lane);
      drain_wait(u.bar(B_Q), 0);
      __syncwarp();
    } else if (start_ok && warp == WARP_MMA) {
      if (split)
        issue_mmas<true>(a, u, lane);
      else
        issue_mmas<false>(a, u, lane);
    }
  } else {
    reg_alloc<REG_SOFTMAX>();
    if (start_ok) {
      if (split)
        softmax<true>(a, u, warp, lane);
      else
        softmax<false>(a, u, warp, lane);
    }
  }

  __syncthreads();
  if (warp == WARP_MMA) {
    tc_fence_after();
    tmem_dealloc(u.tmem, 512);
  }
}

// ------------------------------------------------------------------ merge

struct MergeArgs {
  const float* part_o;
  const float* part_lse;
  long long parts;
  const int* rows;  // {token, first slot, slots, -}
  int n_rows, Hq;
  long long total_q;
  __nv_bfloat16* out;
  long long o_ss, o_sh;
  float* lse;
  int* err;
};

// A warp per (token, head): LSE = log2 sum 2^LSE_i and O = sum 2^(LSE_i - LSE) O_i over
// the row's states; a lane holds 4 dims.
__global__ void __launch_bounds__(256) merge_states_kernel(const MergeArgs a) {
  const int lane = threadIdx.x & 31;
  const long long w = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const bool on = w < static_cast<long long>(a.n_rows) * a.Hq;
  const int h = static_cast<int>(w % a.Hq);
  int4 row = make_int4(0, 0, 0, 0);
  if (on) row = __ldg(reinterpret_cast<const int4*>(a.rows) + w / a.Hq);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!on || stops(a.err)) return;
  if (row.x < 0 || row.x >= a.total_q || row.y < 0 || row.z < 0 || row.y + static_cast<long long>(row.z) > a.parts) {
    if (a.err != nullptr && lane == 0) atomicCAS(a.err, 0, kDevErrIndex);
    return;
  }
  const float* pl = a.part_lse + static_cast<long long>(row.y) * a.Hq + h;
  const float* po = a.part_o + (static_cast<long long>(row.y) * a.Hq + h) * 128 + 4 * lane;
  const long long step = static_cast<long long>(a.Hq) * 128;
  // the first states on their way while the largest LSE is found
  constexpr int AHEAD = 4;
  float x0[AHEAD];
  float4 v0[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (i < row.z) {
      x0[i] = pl[static_cast<long long>(i) * a.Hq];
      v0[i] = *reinterpret_cast<const float4*>(po + i * step);
    }
  float m = -INFINITY;
  bool nan = false;  // (a maximum passes a NaN over)
  for (int i = lane; i < row.z; i += 32) {
    const float x = pl[static_cast<long long>(i) * a.Hq];
    nan |= x != x;
    m = fmaxf(m, x);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, off));
  nan = __any_sync(FULL, nan);
  const float base = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float x, const float4& v) {
    const float wgt = x == -INFINITY ? 0.f : exp2f(x - base);
    sum += wgt;
    if (wgt != 0.f) {  // a state without weight may hold anything
      acc.x = fmaf(wgt, v.x, acc.x);
      acc.y = fmaf(wgt, v.y, acc.y);
      acc.z = fmaf(wgt, v.z, acc.z);
      acc.w = fmaf(wgt, v.w, acc.w);
    }
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (i < row.z) add(x0[i], v0[i]);
#pragma unroll 4
  for (int i = AHEAD; i < row.z; ++i)
    add(pl[static_cast<long long>(i) * a.Hq], *reinterpret_cast<const float4*>(po + i * step));
  const float inv = sum > 0.f || nan ? 1.0f / sum : 0.f;
  uint2 pk;
  pk.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  pk.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(a.out + row.x * a.o_ss + h * a.o_sh + 4 * lane) = pk;
  if (a.lse != nullptr && lane == 0)
    a.lse[static_cast<long long>(row.x) * a.Hq + h] = (base + log2f(sum)) * 0.69314718055994531f;
}

// ------------------------------------------------------------------ plan

// A block: the rows of one or two tiles of a request, before its keys are cut
struct Block {
  Item it;
  int units;   // heads (or kv heads) that take it
  int tiles;   // key tiles
  float step;  // us a key tile
  float cost() const { return tiles * step; }
};

// Measured on the device: 1.8 us for a step of two tiles of rows against a key tile; 1.1 us
// per key tile where the groups share out the keys, with K and V in L2, and 1.5 with all
// SMs reading them from HBM; 6 us of a CTA's start and end; 4 more for writing states and
// merging them.
constexpr float STEP_US = 1.8f, SHARED_US = 1.3f, START_US = 6.f, STATES_US = 4.f;

// pieces of at most `most` us (or of one key tile)
inline int parts(const Block& b, float most) {
  return std::max(1, std::min(b.tiles, static_cast<int>(ceilf(b.cost() / most))));
}

// when the last CTA ends if the blocks are cut into pieces of at most `most` us: the
// hardware takes items in order, each for the first SM that is free
inline float makespan(const std::vector<Block>& blocks, float most, int sms) {
  std::priority_queue<float, std::vector<float>, std::greater<float>> ends;
  float last = 0.f;
  bool cut = false;
  for (const Block& b : blocks) {
    const int n = parts(b, most);
    cut |= n > 1;
    const float c = (b.tiles + n - 1) / n * b.step + START_US;
    for (int k = 0; k < n * b.units; ++k) {
      float at = 0.f;
      if (static_cast<int>(ends.size()) >= sms) {
        at = ends.top();
        ends.pop();
      }
      ends.push(at + c);
      last = std::max(last, at + c);
    }
  }
  return last + (cut ? STATES_US : 0.f);
}

// The same for more pieces than are worth going through one by one: the SMs are full until
// the work runs out, or until the longest piece ends. Unpacked blocks come first, so the
// longest packed one begins when these are under way everywhere.
inline float estimate(const std::vector<Block>& blocks, float most, int sms) {
  float load[2] = {0.f, 0.f}, longest[2] = {0.f, 0.f};  // unpacked, packed
  long long wide = 0;
  bool cut = false;
  for (const Block& b : blocks) {
    const int n = parts(b, most), packed = b.it.flags & PACKED ? 1 : 0;
    const float c = (b.tiles + n - 1) / n * b.step + START_US;
    cut |= n > 1;
    if (!packed) wide += static_cast<long long>(n) * b.units;
    load[packed] += c * static_cast<float>(n) * static_cast<float>(b.units) / static_cast<float>(sms);
    longest[packed] = std::max(longest[packed], c);
  }
  const float begins = wide < sms ? 0.f : load[0];
  return std::max({load[0] + load[1], longest[0], begins + longest[1]}) + (cut ? STATES_US : 0.f);
}

}  // namespace paged
}  // namespace atf

using namespace atf;

extern "C" int atf_prefill_paged_plan(const AtfPrefillPagedPlanParams* p, int32_t* items_host, int32_t items_capacity,
                                      int32_t* rows_host, int32_t rows_capacity, AtfPrefillPagedPlan* out) {
  using namespace atf::paged;
  if (p == nullptr || out == nullptr || p->qo_indptr_host == nullptr || p->kv_indptr_host == nullptr ||
      p->last_page_len_host == nullptr || p->batch_size < 1 || p->num_qo_heads < 1 || p->num_kv_heads < 1 ||
      p->num_qo_heads % p->num_kv_heads != 0 || (items_host == nullptr && items_capacity > 0) ||
      (rows_host == nullptr && rows_capacity > 0) || p->num_sms < 0)
    return ATF_ERR_INVALID_ARG;
  if (p->page_size != 16 && p->page_size != 32 && p->page_size != 64 && p->page_size != 128 && p->page_size != 256)
    return ATF_ERR_UNSUPPORTED;
  if (p->num_qo_heads > (1 << 20)) return ATF_ERR_UNSUPPORTED;
  const int G = p->num_qo_heads / p->num_kv_heads, T = BM / G;  // T = 0: too many heads to pack
  const int sms = p->num_sms > 0 ? p->num_sms : 148;
  std::vector<Block> blocks;
  try {
    for (int b = 0; b < p->batch_size; ++b) {
      const long long nq = static_cast<long long>(p->qo_indptr_host[b + 1]) - p->qo_indptr_host[b];
      const long long np = static_cast<long long>(p->kv_indptr_host[b + 1]) - p->kv_indptr_host[b];
      const int last = p->last_page_len_host[b];
      if (p->qo_indptr_host[b] < 0 || p->kv_indptr_host[b] < 0 || nq < 0 || np < 0 ||
          (np > 0 && (last < 1 || last > p->page_size)))
        return ATF_ERR_INVALID_ARG;
      const long long nk = np > 0 ? (np - 1) * p->page_size + last : 0;
      if (nq > (1ll << 30) || nk > (1ll << 30)) return ATF_ERR_UNSUPPORTED;
      // tiles of rows with and without the heads side by side, per kv head
      const long long tail = nq % BM;
      const long long plain = (nq + BM - 1) / BM * G;
      const long long packed = T > 0 ? nq / BM * ((BM + T - 1) / T) + (tail + T - 1) / T : plain;
      const bool pack = G > 1 && packed < plain;
      const int tt = pack ? T : BM;
      for (long long row = 0; row < nq;) {
        Block x = {};
        Item& it = x.it;
        it.q_tok = p->qo_indptr_host[b];
        it.q_len = static_cast<int>(nq);
        it.k_len = static_cast<int>(nk);
        it.page_beg = p->kv_indptr_host[b];
        it.row = static_cast<int>(row);
        // a tile ends at the next multiple of 128 tokens at the latest
        auto tokens = [&](long long from) -> int {
          return static_cast<int>(std::min<long long>(std::min<long long>(tt, BM - from % BM), nq - from));
        };
        it.n0 = tokens(row);
        it.n1 = row + it.n0 < nq ? tokens(row + it.n0) : 0;
        it.flags = (pack ? PACKED : 0) | (it.n1 == 0 ? SPLIT : 0);
        row += it.n0 + it.n1;
        long long kend = p->causal ? nk - nq + row : nk;
        kend = kend > nk ? nk : (kend < 0 ? 0 : kend);
        x.tiles = static_cast<int>((kend + BN - 1) / BN);
        x.units = pack ? p->num_kv_heads : p->num_qo_heads;
        x.step = it.n1 == 0 ? SHARED_US : STEP_US;
        it.part = -1;
        it.n_parts = 1;
        blocks.push_back(x);
      }
    }
    // unpacked blocks first, then by falling cost
    std::stable_sort(blocks.begin(), blocks.end(), [](const Block& x, const Block& y) {
      const int px = x.it.flags & PACKED, py = y.it.flags & PACKED;
      return px != py ? px < py : x.cost() > y.cost();
    });
    // Cut the keys where that ends sooner: tried are the longest block in 2, 3, 4, ... parts
    long long units = 0;
    float longest = 0.f, share = 0.f;  // share: an SM's part of all work
    for (const Block& x : blocks) {
      units += x.units;
      longest = std::max(longest, x.cost());
      share += x.units * x.cost() / sms;
    }
    float most = 1e30f;
    const bool few = units <= 4ll * sms;
    const float full = share + (few ? START_US : START_US * static_cast<float>(units) / static_cast<float>(sms));
    // (no end is later than a full machine's by more than the longest block)
    if (units > 0 && (few || longest > 0.05f * full)) {
      // Few blocks are gone through one by one. For many an estimate will do (each step of
      // the search is a pass over the blocks): they are only cut where the longest goes on
      // after the others. One token over 128K keys beside 74 over 1000 (32 / 8 heads, from cold
      // memory) takes 168 us, 1044 uncut; behind 4 chunks of 2048 over 8192 keys 910, 1720 uncut.
      auto end_with = [&](float m) { return few ? makespan(blocks, m, sms) : estimate(blocks, m, sms); };
      float best = end_with(most);
      for (int k = 2; k <= 2 * sms && best > 1.05f * full; k += k < 4 ? 1 : k / 2) {
        const float m = longest / k;
        // shorter pieces cost more than they bring
        if (m < START_US / 2 || m < share / 4) break;
        const float end = end_with(m);
        if (end < 0.97f * best) {
          best = end;
          most = m;
        }
      }
      // and, where an SM takes few pieces, between that length and its neighbours (chunks of 9
      // requests, 1 to 72 tokens, up to 5003 keys: 37.7 us instead of 41.2, from cold memory 49
      // instead of 52; 36 random batches from cold memory 2.30 ms instead of 2.335; with many
      // pieces nothing is gained)
      const float found = most < longest ? most : longest;
      long long pieces = 0;
      if (few)
        for (const Block& x : blocks) pieces += x.units * parts(x, found);
      if (few && pieces <= 2ll * sms)
        for (float f : {1.25f, 1.12f, 0.93f, 0.86f, 0.8f, 0.74f, 0.68f}) {
          const float m = found * f;
          if (best <= 1.02f * full) break;
          if (m >= longest || m < START_US / 2 || m < share / 4) continue;
          const float end = end_with(m);
          if (end < 0.98f * best) {
            best = end;
            most = m;
          }
        }
    }
    long long items = 0, wide = 0, rows = 0, slots = 0;
    for (Block& x : blocks) {
      const int n = most < 1e30f ? parts(x, most) : 1;
      const int tok = x.it.n0 + x.it.n1;
      const int each = (x.tiles + n - 1) / n;
      const int pieces = each > 0 ? std::max(1, (x.tiles + each - 1) / each) : 1;
      x.it.n_parts = pieces;
      if (pieces > 1) {
        if (slots + static_cast<long long>(tok) * pieces > 0x7fffffffLL) return ATF_ERR_UNSUPPORTED;
        x.it.part = static_cast<int>(slots);
        if (rows_host != nullptr)
          for (int i = 0; i < tok; ++i) {
            if (rows + i >= rows_capacity) return ATF_ERR_WORKSPACE;
            int32_t* r = rows_host + 4 * (rows + i);
            r[0] = x.it.q_tok + x.it.row + i;
            r[1] = static_cast<int32_t>(slots + static_cast<long long>(i) * pieces);
            r[2] = pieces;
            r[3] = 0;
          }
        rows += tok;
        slots += static_cast<long long>(tok) * pieces;
      }
      if (items_host != nullptr)
        for (int i = 0; i < pieces; ++i) {
          if (items + i >= items_capacity) return ATF_ERR_WORKSPACE;
          Item it = x.it;
          it.kt0 = i * each;
          it.kt1 = std::min(x.tiles, (i + 1) * each);
          if (pieces > 1) it.part += i;
          std::memcpy(items_host + ATF_PAGED_ITEM_INTS * (items + i), &it, sizeof(Item));
        }
      items += pieces;
      if (!(x.it.flags & PACKED)) wide += pieces;
    }
    if (items > 0x7fffffffLL || items * p->num_qo_heads > 0x7fffffffLL) return ATF_ERR_UNSUPPORTED;
    out->num_items = static_cast<int32_t>(items);
    out->num_wide = static_cast<int32_t>(wide);
    out->num_rows = static_cast<int32_t>(rows);
    out->num_parts = static_cast<int32_t>(slots);
    out->partial_o_floats = slots * p->num_qo_heads * 128;
    out->partial_lse_floats = slots * p->num_qo_heads;
  } catch (...) {  // no host memory for the schedule
    return ATF_ERR_WORKSPACE;
  }
  return ATF_OK;
}

extern "C" int atf_prefill_paged_fwd(const AtfPrefillPagedParams* p, atf_stream_t stream) {
  using namespace atf::paged;
  if (p == nullptr || p->q == nullptr || p->k_cache == nullptr || p->v_cache == nullptr || p->out == nullptr ||
      p->items == nullptr || p->indices == nullptr)
    return ATF_ERR_INVALID_ARG;
  if (p->head_dim != ATF_HEAD_DIM) return ATF_ERR_UNSUPPORTED;
  if (p->total_q < 1 || p->num_pages < 1 || p->num_indices < 0 || p->num_heads_q < 1 || p->num_heads_kv < 1 ||
      p->num_heads_q % p->num_heads_kv != 0 || p->num_items < 0 || p->num_wide < 0 || p->num_wide > p->num_items ||
      p->num_rows < 0 || p->num_parts < 0)
    return ATF_ERR_INVALID_ARG;
  // (a row's place is counted in 32 bits, in steps of 16 bytes)
  if (p->num_parts > 0 && static_cast<long long>(p->num_parts) * p->num_heads_q * 32 >= 0xffffffffLL)
    return ATF_ERR_UNSUPPORTED;
  if (p->num_parts > 0 && (p->partial_o == nullptr || p->partial_lse == nullptr)) return ATF_ERR_INVALID_ARG;
  if (p->num_rows > 0 && p->rows == nullptr) return ATF_ERR_INVALID_ARG;
  if (p->total_q > 0x7fffffffLL - BM * NQ || p->num_pages > 0x7fffffffLL || p->num_heads_q > (1 << 20))
    return ATF_ERR_UNSUPPORTED;
  if (p->page_size != 16 && p->page_size != 32 && p->page_size != 64 && p->page_size != 128 && p->page_size != 256)
    return ATF_ERR_UNSUPPORTED;
  if (p->window != ATF_WINDOW_OFF && p->window != ATF_WINDOW_SNAP16) return ATF_ERR_UNSUPPORTED;
  if (!(p->softmax_scale > 0.f)) return ATF_ERR_INVALID_ARG;
  if (!aligned16(p->q) || !aligned16(p->k_cache) || !aligned16(p->v_cache) || !aligned16(p->out) ||
      !aligned16(p->items) || !aligned16(p->rows) || !aligned16(p->partial_o))
    return ATF_ERR_ALIGNMENT;
  const int64_t strides[10] = {p->q_stride_s,     p->q_stride_h,    p->k_stride_page, p->k_stride_token, p->k_stride_head,
                               p->v_stride_page,  p->v_stride_token, p->v_stride_head, p->o_stride_s,    p->o_stride_h};
  for (int i = 0; i < 10; ++i)
    if (strides[i] < 0 || (strides[i] & 7) != 0) return ATF_ERR_ALIGNMENT;
  if (p->o_stride_s > (1ll << 40) || p->o_stride_h > (1ll << 40) ||
      (((p->total_q - 1) * p->o_stride_s + (p->num_heads_q - 1) * p->o_stride_h) >> 3) >= 0xffffffffLL)
    return ATF_ERR_UNSUPPORTED;
  if (p->window == ATF_WINDOW_SNAP16)
    for (int i = 0; i < ATF_MAX_LEVELS; ++i)
      if (p->zhi[i] < 0 || (i > 0 && p->zhi[i] > p->zhi[i - 1])) return ATF_ERR_INVALID_ARG;
  int dev = 0;
  int rc = check_device(&dev);
  if (rc != ATF_OK) return rc;
  if (p->num_items == 0) return ATF_OK;

  Args a = {};
  a.Hq = static_cast<int>(p->num_heads_q);
  a.Hkv = static_cast<int>(p->num_heads_kv);
  a.G = a.Hq / a.Hkv;
  a.T = BM / a.G;
  if (p->num_wide < p->num_items && a.T < 1) return ATF_ERR_INVALID_ARG;  // packed items of such a group
  for (a.page_shift = 4; (1 << a.page_shift) < p->page_size;) ++a.page_shift;
  a.row_shift = a.page_shift < 7 ? a.page_shift : 7;
  a.merge = p->num_rows > 0 ? 1 : 0;
  auto sane = [](int64_t stride, int64_t size) -> uint64_t {
    return static_cast<uint64_t>(size == 1 ? 16 : stride * 2);
  };
  CUtensorMap tq, tqp, tk, tv;
  {
    const uint64_t dims[4] = {128, static_cast<uint64_t>(p->num_heads_q), static_cast<uint64_t>(p->total_q), 1};
    const uint64_t str[3] = {sane(p->q_stride_h, p->num_heads_q), sane(p->q_stride_s, p->total_q), 16};
    const uint32_t one[4] = {64, 1, BM, 1};
    if ((rc = encode_tiled_bf16(&tq, p->q, 4, dims, str, one, CU_TENSOR_MAP_SWIZZLE_128B)) != ATF_OK) return rc;
    tqp = tq;
    if (p->num_wide < p->num_items) {
      const uint32_t group[4] = {64, static_cast<uint32_t>(a.G), static_cast<uint32_t>(a.T), 1};
      if ((rc = encode_tiled_bf16(&tqp, p->q, 4, dims, str, group, CU_TENSOR_MAP_SWIZZLE_128B)) != ATF_OK) return rc;
    }
  }
  auto pages = [&](CUtensorMap* map, const void* base, int64_t sp, int64_t stok, int64_t sh) -> int {
    const uint64_t dims[4] = {128, static_cast<uint64_t>(p->page_size), static_cast<uint64_t>(p->num_heads_kv),
                              static_cast<uint64_t>(p->num_pages)};
    const uint64_t str[3] = {sane(stok, p->page_size), sane(sh, p->num_heads_kv), sane(sp, p->num_pages)};
    const uint32_t box[4] = {64, 1u << a.row_shift, 1, 1};
    return encode_tiled_bf16(map, base, 4, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  if ((rc = pages(&tk, p->k_cache, p->k_stride_page, p->k_stride_token, p->k_stride_head)) != ATF_OK) return rc;
  if ((rc = pages(&tv, p->v_cache, p->v_stride_page, p->v_stride_token, p->v_stride_head)) != ATF_OK) return rc;
  const bool in_l2 = static_cast<long long>(p->num_indices) * p->page_size * a.Hkv * 512 <= (64ll << 20);
  a.walk = in_l2 ? a.Hq : a.G;
  a.scale_log2 = p->softmax_scale * 1.4426950408889634f;
  a.causal = p->causal ? 1 : 0;
  a.window = p->window == ATF_WINDOW_SNAP16 ? 1 : 0;
  for (int i = 0; i < ATF_MAX_LEVELS; ++i) a.zhi[i] = p->zhi[i];
  a.out = static_cast<__nv_bfloat16*>(p->out);
  a.o_ss = p->o_stride_s;
  a.o_sh = p->o_stride_h;
  a.lse = p->lse;
  a.part_o = p->partial_o;
  a.part_lse = p->partial_lse;
  a.parts = p->num_parts;
  a.err = p->error_flag;
  a.items = p->items;
  a.n_wide = p->num_wide;
  a.n_items = p->num_items;
  a.total_q = p->total_q;
  a.indices = p->indices;
  a.num_indices = p->num_indices;
  a.num_pages = static_cast<int>(p->num_pages);
  const long long units =
      static_cast<long long>(a.n_wide) * a.Hq + static_cast<long long>(a.n_items - a.n_wide) * a.Hkv;
  if (units > 0x7fffffffLL) return ATF_ERR_UNSUPPORTED;
  if (cudaFuncSetAttribute(paged_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SMEM_BYTES)) !=
      cudaSuccess)
    return ATF_ERR_CUDA;
  // setmaxnreg.inc waits until the block's launch registers cover the split: never launch
  // a build whose register count would leave it waiting
  static const int launch_regs = [] {
    cudaFuncAttributes fa{};
    return cudaFuncGetAttributes(&fa, paged_kernel) == cudaSuccess ? fa.numRegs : 0;
  }();
  if (static_cast<long long>(launch_regs) * THREADS < REG_SPLIT_TOTAL) return ATF_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  paged_kernel<<<static_cast<unsigned>(units), THREADS, SMEM_BYTES, st>>>(tq, tqp, tk, tv, a);
  if (cudaGetLastError() != cudaSuccess) return ATF_ERR_CUDA;
  if (p->num_rows == 0) return ATF_OK;
  MergeArgs m = {p->partial_o, p->partial_lse, p->num_parts, p->rows,     p->num_rows, a.Hq,
                 p->total_q,   a.out,          p->o_stride_s, p->o_stride_h, p->lse,    p->error_flag};
  const long long blocks = (static_cast<long long>(p->num_rows) * a.Hq + 7) / 8;
  if (blocks > 0x7fffffffLL) return ATF_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, merge_states_kernel, m) == cudaSuccess ? ATF_OK : ATF_ERR_CUDA;
}
