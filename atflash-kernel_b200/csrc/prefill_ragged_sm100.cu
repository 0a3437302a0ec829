// Causal or full attention over packed sequences of different lengths, for sm_100a:
// the dense prefill's pipeline (prefill_sm100.cu) made persistent.
//
// Mathematics, tiles and arithmetic are the dense kernel's: per query row an online
// softmax in the log2 domain over 128-key tiles, S = Q K^T over the window's 16-dim
// levels and O += P V on the tensor cores with both accumulators in TMEM, P in bf16.
// A sequence's rows are those of a dense run of its own, bit for bit: the window is
// quantised per (query tile, key tile) from the sequence's own first row and key.
//
// A unit is (block of 256 query rows of a sequence, query head): two 128-row tiles.
// The plan lists the blocks of all sequences by falling key count; units go kv head
// by kv head, then block by block, then over the group's heads. The plan deals them
// out in that order to one CTA per SM, each to the one with the least work so far
// (a step of both tiles 1, of one tile 0.9, a unit's start and end 1.8), and the
// kernel walks its list. (Every 148th unit to a CTA: 4 long chunks 780 us instead of
// 730. CTAs that take the next unit from the hardware's queue with
// clusterlaunchcontrol.try_cancel, handed on inside the CTA in shared memory, balanced
// as well but ran each tile 5% slower: 4 x 4096 tokens, 24 heads, 464 against 440 us.)
//
// Why persistent: a block's fixed cost was 8 us against 2.1 us per key tile (start of
// the CTA 0.8, barriers and TMEM 1.5, first loads 1.5, cold first step, a strided
// epilogue 2.3 us; 64 sequences of 256 tokens, 28 heads: 170 us). Here barriers and
// TMEM are set up once, and while a unit's last tiles are still in softmax and
// epilogue the producer loads the next unit's Q, K and V and the MMA warp computes
// its first scores. All barrier phases count on through the units.
//   - Q has one buffer: free when the unit's last S = Q K^T has completed (Q_EMPTY).
//   - O_t is free for the next unit's first O_t = P V once tile t's epilogue has read
//     it from TMEM (OFREE).
//   - S_t and the P in its upper half: the next unit's S is issued after every P V of
//     this unit, by the same thread, so in order; P V waits for P, which follows the
//     read of S.
//   - a tile without keys (rows past the sequence, or before its first key) takes no
//     part in a unit and advances no phase.
// Q comes in rows of 128 bytes (two boxes of 64 dims, 128-byte swizzle; in
// rotate_half order in the dense kernel's 8-dim boxes). Outputs go through shared
// memory, 4 KB per warp, and leave in full 128-byte lines.
//
// A tile's last box may reach into the next sequence: its queries are not stored, its
// keys are masked, and its V rows, whose P is 0, are cleared in shared memory before
// the product (they may hold anything, NaN included).
#include <math.h>

#include <algorithm>
#include <cstring>
#include <functional>
#include <utility>
#include <vector>

#include "atf_internal.h"
#include "atf_ptx.cuh"
#include "prefill_common.cuh"

namespace atf {
namespace ragged {

using namespace prefill;

// The same with Q as two boxes of 64 dims in 128-byte rows (128-byte swizzle, 16
// KB each): level i advances A by 32 bytes inside a row, and to the next box after
// four levels.
__device__ __forceinline__ void qk_group_rows_asm(uint32_t d_tmem, uint64_t qd, uint64_t kd, uint32_t idesc, int L,
                                                  uint32_t bar_addr) {
  asm volatile(
      "{\n\t.reg .pred pe, p1, p2, p3, p4, p5, p6, p7;\n\t.reg .b64 a, b;\n\t"
      "elect.sync _|pe, 0xffffffff;\n\t"
      "setp.gt.and.s32 p1, %4, 1, pe;\n\tsetp.gt.and.s32 p2, %4, 2, pe;\n\tsetp.gt.and.s32 p3, %4, 3, pe;\n\t"
      "setp.gt.and.s32 p4, %4, 4, pe;\n\tsetp.gt.and.s32 p5, %4, 5, pe;\n\tsetp.gt.and.s32 p6, %4, 6, pe;\n\t"
      "setp.gt.and.s32 p7, %4, 7, pe;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, 0;\n\t"
      "add.u64 a, %1, 2;\n\tadd.u64 b, %2, 256;\n\t"
      "@p1 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 2;\n\tadd.u64 b, b, 256;\n\t"
      "@p2 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 2;\n\tadd.u64 b, b, 256;\n\t"
      "@p3 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 1018;\n\tadd.u64 b, b, 256;\n\t"
      "@p4 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 2;\n\tadd.u64 b, b, 256;\n\t"
      "@p5 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 2;\n\tadd.u64 b, b, 256;\n\t"
      "@p6 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 2;\n\tadd.u64 b, b, 256;\n\t"
      "@p7 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "@pe tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t}"
      ::"r"(d_tmem), "l"(qd), "l"(kd), "r"(idesc), "r"(L), "r"(bar_addr)
      : "memory");
}

constexpr uint32_t OFF_Q = 0;
constexpr uint32_t OFF_K = OFF_Q + NQ * QTILE_BYTES;
constexpr uint32_t OFF_V = OFF_K + KST * KSTAGE_BYTES;
constexpr uint32_t OFF_OUT = OFF_V + VST * VSTAGE_BYTES;  // 8 warps x [32 rows][128 B]
constexpr uint32_t OUT_BYTES = 32 * 128;
constexpr uint32_t OFF_BAR = OFF_OUT + 8 * OUT_BYTES;

enum {
  B_QFULL = 0,
  B_QEMPTY,                   // the unit's last S has completed
  B_KFULL,
  B_KEMPTY = B_KFULL + KST,
  B_VFULL = B_KEMPTY + KST,
  B_VEMPTY = B_VFULL + VST,
  B_SFULL = B_VEMPTY + VST,   // [t], one phase per S_t
  B_LOADED = B_SFULL + NQ,    // [t], one phase per S_t: its scores are in registers
  B_PFULL = B_LOADED + NQ,    // [t], one phase per P_t
  B_ODONE = B_PFULL + NQ,     // [t], one phase per O_t += P_t V
  B_OFINAL = B_ODONE + NQ,    // [t], one phase per unit of tile t: its last O += P V done
  B_OFREE = B_OFINAL + NQ,    // [t], one phase per unit of tile t: O has been read
  B_FINAL = B_OFREE + NQ,
  NUM_BARS
};
constexpr uint32_t OFF_ABORT = OFF_BAR + 8 * NUM_BARS;
constexpr uint32_t OFF_TMEM = OFF_ABORT + 16;
constexpr uint32_t SMEM_BYTES = OFF_TMEM + 16 + 1024;  // slack for 1024-B alignment
static_assert(SMEM_BYTES <= 227 * 1024, "one CTA per SM");

// One work item of the plan: 256 query rows from `row` on of one sequence. Rows and
// keys are the sequence's own; the packed tensors hold them from q_beg and k_beg on.
struct Item {
  int q_beg, q_len, k_beg, k_len, row, pad[3];
};
static_assert(sizeof(Item) == 32, "eight ints per item");

struct Args {
  int Hq, G;
  float scale_log2;
  int causal, layout, window;
  int zhi[ATF_MAX_LEVELS];
  __nv_bfloat16* out;
  long long o_ss, o_sh;
  float* lse;
  int* err;
  const int* items;
  const int* cta_units;  // [grid + 1]: where a CTA's units begin in `units`
  const int* units;      // (kv head, item, head of the group) as one index
  int n_items, n_units;
  long long total_q, total_k;
};

struct Unit {
  int q_tok, k_tok, sk, row_end, row0, hk, h;
  int q_offset;  // position of the sequence's query row 0 among its keys (may be negative)
  int nk[NQ];    // key tiles of each query tile

  __device__ __forceinline__ int nk_max() const { return max(nk[0], nk[1]); }
};

// a CTA's units, one after another; -1 past the last
struct Walk {
  const int* at;
  int left;
  __device__ __forceinline__ explicit Walk(const Args& a) {
    const int b = __ldg(a.cta_units + blockIdx.x), e = __ldg(a.cta_units + blockIdx.x + 1);
    at = a.units + b;
    left = b >= 0 && e <= a.n_units ? e - b : 0;
  }
  __device__ __forceinline__ int next(const Args& a) {
    if (left <= 0) return -1;
    --left;
    const int u = __ldg(at++);
    return u >= 0 && u < a.n_units ? u : -1;
  }
};
__device__ __forceinline__ Item load_item(const Args& a, int u) {
  const int rem = u % (a.n_items * a.G);
  const int4* p = reinterpret_cast<const int4*>(a.items) + 2 * (rem / a.G);
  const int4 x = __ldg(p), y = __ldg(p + 1);
  return Item{x.x, x.y, x.z, x.w, y.x, {0, 0, 0}};
}
// An item outside the packed rows (a plan made for others) has no tiles and no rows.
__device__ __forceinline__ Unit make_unit(const Args& a, int u, const Item& it) {
  const int per_head = a.n_items * a.G, rem = u % per_head;
  Unit x;
  x.hk = u / per_head;
  x.h = x.hk * a.G + rem % a.G;
  const bool bad = it.q_beg < 0 || it.q_len < 0 || it.k_beg < 0 || it.k_len < 0 || it.row < 0 ||
                   static_cast<long long>(it.q_beg) + it.q_len > a.total_q ||
                   static_cast<long long>(it.k_beg) + it.k_len > a.total_k;
  if (bad && a.err != nullptr) atomicCAS(a.err, 0, kDevErrIndex);
  x.q_tok = it.q_beg;
  x.k_tok = it.k_beg;
  x.sk = it.k_len;
  x.row0 = it.row;
  x.row_end = bad ? 0 : it.q_len;
  x.q_offset = it.k_len - it.q_len;
#pragma unroll
  for (int t = 0; t < NQ; ++t) {
    const int r = it.row + t * BM;
    int kend = a.causal ? min(x.q_offset + r + BM, x.sk) : x.sk;
    x.nk[t] = (r < x.row_end && kend > 0) ? (kend + BN - 1) / BN : 0;
  }
  return x;
}
// key tile j reads level i when j >= lim[i] (the dense kernel's rule)
__device__ __forceinline__ void window_limits(const Args& a, int q_offset, int row0, int (&lim)[ATF_MAX_LEVELS]) {
  const long long base = static_cast<long long>(q_offset) + row0 - (BN - 1);
#pragma unroll
  for (int i = 0; i < ATF_MAX_LEVELS; ++i) {
    const long long x = base - a.zhi[i];
    lim[i] = (!a.window || i == 0 || x <= 0) ? 0 : static_cast<int>((x + BN - 1) / BN);
  }
}

__global__ void __launch_bounds__(THREADS, 1)
    ragged_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ KLevelMaps tmKL, const __grid_constant__ CUtensorMap tmV, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  const uint32_t sb = (raw_u32 + 1023u) & ~1023u;
  uint8_t* sp = smem_raw + (sb - raw_u32);
  volatile int* s_abort = reinterpret_cast<volatile int*>(sp + OFF_ABORT);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(sp + OFF_TMEM);
  auto bar = [&](int i) -> uint32_t { return sb + OFF_BAR + 8u * static_cast<uint32_t>(i); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool sorted = a.layout == ATF_LAYOUT_SORTED_PAIR;

  if (threadIdx.x == 0) {
    *s_abort = (a.err != nullptr && *reinterpret_cast<volatile int*>(a.err) != 0) ? 1 : 0;
    for (int i = 0; i < NUM_BARS; ++i) {
      const bool wide = (i >= B_LOADED && i < B_ODONE) || (i >= B_OFREE && i < B_FINAL);
      mbar_init(bar(i), wide ? 128 : 1);  // LOADED, PFULL, OFREE: a whole softmax group
    }
    fence_mbar_init();
  }
  if (warp == WARP_LOAD && lane == 0) {
    tma_prefetch_desc(&tmQ);
    if (!sorted)
      tma_prefetch_desc(&tmK);
    else
      for (int L = a.window ? 0 : ATF_MAX_LEVELS - 1; L < ATF_MAX_LEVELS; ++L) tma_prefetch_desc(&tmKL.lv[L]);
    tma_prefetch_desc(&tmV);
  }
  if (warp == WARP_MMA) {
    tmem_alloc(smem_u32(s_tmem), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const AbortCtl ab{s_abort, a.err};
  const bool start_ok = (*s_abort == 0);
  if (warp >= 8) {
    reg_dealloc<REG_SMALL>();
    if (start_ok && warp == WARP_LOAD) {
      // ---------------------------------------------------------------- producer
      int kc = 0, vc = 0, qc = 0;  // K and V stages and Q loads issued
      bool ok = true;
      Walk walk(a);
      int u = walk.next(a);
      Item it = u >= 0 ? load_item(a, u) : Item{};
      while (ok && u >= 0) {
        const Unit x = make_unit(a, u, it);
        u = walk.next(a);
        if (u >= 0) it = load_item(a, u);  // of the next unit
        const int nk_max = x.nk_max();
        if (nk_max == 0) continue;
        int lim[NQ][ATF_MAX_LEVELS];
#pragma unroll
        for (int t = 0; t < NQ; ++t) window_limits(a, x.q_offset, x.row0 + t * BM, lim[t]);
        ok = __all_sync(FULL, mbar_wait_inl(bar(B_QEMPTY), (qc & 1) ^ 1, ab, kDevErrTimeout));
        if (!ok) break;
        mbar_arrive_expect_tx_elect(bar(B_QFULL), ((x.nk[0] > 0) + (x.nk[1] > 0)) * QTILE_BYTES);
#pragma unroll
        for (int t = 0; t < NQ; ++t) {
          if (x.nk[t] == 0) continue;
          const uint32_t dst = sb + OFF_Q + t * QTILE_BYTES;
          const int row = x.q_tok + x.row0 + t * BM;
          if (sorted) {
            tma_load_4d_elect(dst, &tmQ, bar(B_QFULL), 0, row, x.h, 0);
            tma_load_4d_elect(dst + QTILE_BYTES / 2, &tmQ, bar(B_QFULL), 64, row, x.h, 0);
          } else {
            for (int i = 0; i < 16; ++i)
              tma_load_4d_elect(dst + (i >> 1) * QSLAB_BYTES + (i & 1) * QHALF_BYTES, &tmQ, bar(B_QFULL),
                                level_col(a.layout, i >> 1, i & 1), row, x.h, 0);
          }
        }
        ++qc;
        for (int j = 0; j < nk_max; ++j) {
          const int ks = kc % KST, vs = vc % VST;
          ok = __all_sync(FULL, mbar_wait_inl(bar(B_KEMPTY + ks), ((kc / KST) & 1) ^ 1, ab, kDevErrTimeout));
          if (!ok) break;
          int L = 0;
#pragma unroll
          for (int t = 0; t < NQ; ++t)
            if (j < x.nk[t]) L = max(L, levels_for(lim[t], j));
          const uint32_t kdst = sb + OFF_K + ks * KSTAGE_BYTES;
          const int key = x.k_tok + j * BN;
          mbar_arrive_expect_tx_elect(bar(B_KFULL + ks), static_cast<uint32_t>(L) * KSLAB_BYTES);
          if (sorted) {
            if (elect_one_lane()) tma_load_5d(kdst, &tmKL.lv[L - 1], bar(B_KFULL + ks), 0, key, 0, x.hk, 0);
            __syncwarp();
          } else {
            for (int i = 0; i < L; ++i) {
              tma_load_4d_elect(kdst + i * KSLAB_BYTES, &tmK, bar(B_KFULL + ks), level_col(a.layout, i, 0), key, x.hk,
                                0);
              tma_load_4d_elect(kdst + i * KSLAB_BYTES + KHALF_BYTES, &tmK, bar(B_KFULL + ks),
                                level_col(a.layout, i, 1), key, x.hk, 0);
            }
          }
          ++kc;
          ok = __all_sync(FULL, mbar_wait_inl(bar(B_VEMPTY + vs), ((vc / VST) & 1) ^ 1, ab, kDevErrTimeout));
          if (!ok) break;
          const uint32_t vdst = sb + OFF_V + vs * VSTAGE_BYTES;
          mbar_arrive_expect_tx_elect(bar(B_VFULL + vs), VSTAGE_BYTES);
          tma_load_4d_elect(vdst, &tmV, bar(B_VFULL + vs), 0, key, x.hk, 0);
          tma_load_4d_elect(vdst + VBOX_BYTES, &tmV, bar(B_VFULL + vs), 64, key, x.hk, 0);
          ++vc;
        }
      }
      // every copy issued lands before shared memory is released
      if (qc > 0) drain_wait(bar(B_QFULL), (qc - 1) & 1);
      for (int j = max(0, kc - KST); j < kc; ++j) drain_wait(bar(B_KFULL + j % KST), (j / KST) & 1);
      for (int j = max(0, vc - VST); j < vc; ++j) drain_wait(bar(B_VFULL + j % VST), (j / VST) & 1);
      __syncwarp();
    } else if (start_ok && warp == WARP_MMA) {
      // ---------------------------------------------------------------- MMA issuer
      const uint32_t tm = __shfl_sync(FULL, tmem, 0);
      const uint64_t qrows0 = make_sdesc(sb + OFF_Q, 16, 1024, kLayoutSw128);
      const uint64_t qslab0 = make_sdesc(sb + OFF_Q, QHALF_BYTES, 128, kLayoutNone);
      const uint64_t kslab0 = make_sdesc(sb + OFF_K, KHALF_BYTES, 128, kLayoutNone);
      const uint64_t kswz0 = make_sdesc(sb + OFF_K, 16, 256, kLayoutSw32);
      const uint64_t vdesc0 = make_sdesc(sb + OFF_V, VBOX_BYTES, 1024, kLayoutSw128);
      int kb = 0, vb = 0, qc = 0;               // stages and Q loads of the units before
      int sc0 = 0, sc1 = 0, oc0 = 0, oc1 = 0;   // S of each tile, and its units, before
      bool ok = true;
      Walk walk(a);
      int u = walk.next(a);
      Item it = u >= 0 ? load_item(a, u) : Item{};
      while (ok && u >= 0) {
        const Unit x = make_unit(a, u, it);
        u = walk.next(a);
        if (u >= 0) it = load_item(a, u);
        const int nk0 = x.nk[0], nk1 = x.nk[1], nk_max = x.nk_max();
        if (nk_max == 0) continue;
        int lim[NQ][ATF_MAX_LEVELS];
#pragma unroll
        for (int t = 0; t < NQ; ++t) window_limits(a, x.q_offset, x.row0 + t * BM, lim[t]);
        int s_left = nk0 + nk1;
        // S_t(j) into tile t's S columns; after the unit's last one Q is free
        auto issue_S = [&](int t, int j) {
          const int L = levels_for(lim[t], j);
          const uint32_t d_tmem = tm + static_cast<uint32_t>(t * 128);
          const uint64_t kd = (sorted ? kswz0 : kslab0) + ((((kb + j) % KST) * KSTAGE_BYTES) >> 4);
          if (sorted)
            qk_group_rows_asm(d_tmem, qrows0 + ((t * QTILE_BYTES) >> 4), kd, IDESC_QK, L, bar(B_SFULL + t));
          else
            qk_group_asm(d_tmem, qslab0 + ((t * QTILE_BYTES) >> 4), kd, IDESC_QK, L, bar(B_SFULL + t));
          if (--s_left == 0) tc_commit_elect(bar(B_QEMPTY));
        };
        // O_t += P_t(j) V_j; P_t sits in columns 64..127 of the other tile's S
        auto issue_PV = [&](int t, int j) {
          const uint32_t o_tmem = tm + 256u + static_cast<uint32_t>(t * 128);
          const uint32_t p_tmem = tm + static_cast<uint32_t>((1 - t) * 128 + 64);
          const uint64_t vd = vdesc0 + ((((vb + j) % VST) * VSTAGE_BYTES) >> 4);
          pv_group_asm(o_tmem, p_tmem, vd, IDESC_PV, j > 0 ? 1u : 0u, bar(B_ODONE + t));
        };
        auto wait = [&](int b, int phase) -> bool {
          const bool w = __all_sync(FULL, mbar_wait_inl(bar(b), static_cast<uint32_t>(phase) & 1u, ab, kDevErrTimeout));
          tc_fence_after();
          return w;
        };
        int k_waited = -1;  // K tiles are waited for in order, once each
        auto kwait = [&](int j) -> bool {
          while (k_waited < j) {
            ++k_waited;
            if (!wait(B_KFULL + (kb + k_waited) % KST, (kb + k_waited) / KST)) return false;
          }
          return true;
        };
        // A K stage is released after the last S that reads it: S_1(j) when tile 1
        // has key tile j, else S_0(j).
        ok = wait(B_QFULL, qc) && kwait(0);
        if (ok) {
          if (nk0 > 0) issue_S(0, 0);
          if (nk1 > 0) issue_S(1, 0);
          tc_commit_elect(bar(B_KEMPTY + kb % KST));
        }
        // S_0(1) once tile 0 has read S_0(0)
        if (ok && nk0 > 1 && (ok = kwait(1) && wait(B_LOADED + 0, sc0))) {
          issue_S(0, 1);
          if (1 >= nk1) tc_commit_elect(bar(B_KEMPTY + (kb + 1) % KST));
        }
        for (int j = 0; ok && j < nk_max; ++j) {
          const int vs = (vb + j) % VST;
          if (!(ok = wait(B_VFULL + vs, (vb + j) / VST))) break;
          // V rows past the sequence's last key: another sequence's
          const int live = x.sk - j * BN;
          if (live < BN) {
            uint8_t* v0 = sp + OFF_V + vs * VSTAGE_BYTES;
            for (int e = live * 8 + lane; e < BN * 8; e += 32) {
              *reinterpret_cast<uint4*>(v0 + 16 * e) = make_uint4(0, 0, 0, 0);
              *reinterpret_cast<uint4*>(v0 + VBOX_BYTES + 16 * e) = make_uint4(0, 0, 0, 0);
            }
            // the MMAs read V through the async proxy
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
          if (j < nk0) {
            // (the first one overwrites O_0: the unit before it has been read)
            if (!(ok = (j > 0 || wait(B_OFREE + 0, oc0 + 1)) && wait(B_PFULL + 0, sc0 + j))) break;
            issue_PV(0, j);
            if (j + 1 == nk0) tc_commit_elect(bar(B_OFINAL + 0));
          }
          // S_1(j+1) overwrites the columns P_0(j) occupies (O_0 += P_0(j) V_j was
          // issued first; tcgen05.mma ops of one thread run in order) and needs
          // tile 1 to have read S_1(j)
          if (j + 1 < nk1) {
            if (!(ok = kwait(j + 1) && wait(B_LOADED + 1, sc1 + j))) break;
            issue_S(1, j + 1);
            tc_commit_elect(bar(B_KEMPTY + (kb + j + 1) % KST));
          }
          if (j < nk1) {
            if (!(ok = (j > 0 || wait(B_OFREE + 1, oc1 + 1)) && wait(B_PFULL + 1, sc1 + j))) break;
            issue_PV(1, j);
            if (j + 1 == nk1) tc_commit_elect(bar(B_OFINAL + 1));
          }
          // S_0(j+2): after O_1 += P_1(j) V_j (P_1(j) sits in S_0's columns) and
          // tile 0's read of S_0(j+1)
          if (j + 2 < nk0) {
            if (!(ok = kwait(j + 2) && wait(B_LOADED + 0, sc0 + j + 1))) break;
            issue_S(0, j + 2);
            if (j + 2 >= nk1) tc_commit_elect(bar(B_KEMPTY + (kb + j + 2) % KST));
          }
          tc_commit_elect(bar(B_VEMPTY + vs));
        }
        kb += nk_max;
        vb += nk_max;
        ++qc;
        sc0 += nk0;
        sc1 += nk1;
        oc0 += nk0 > 0 ? 1 : 0;
        oc1 += nk1 > 0 ? 1 : 0;
      }
      // Every MMA issued by this CTA completes before TMEM is released.
      tc_commit_elect(bar(B_FINAL));
      __syncwarp();
      drain_wait(bar(B_FINAL), 0);
      __syncwarp();
    }
  } else {
    reg_alloc<REG_SOFTMAX>();
    if (start_ok) {
      // ---------------------------------------------------------------- softmax
      const int t = warp >> 2;
      const int wq = warp & 3;
      const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
      const uint32_t tS = tmem + static_cast<uint32_t>(t * 128) + lane_off;
      const uint32_t tP = tmem + static_cast<uint32_t>((1 - t) * 128 + 64) + lane_off;
      const uint32_t tO = tmem + 256u + static_cast<uint32_t>(t * 128) + lane_off;
      uint8_t* s_out = sp + OFF_OUT + warp * OUT_BYTES;
      const float sl2 = a.scale_log2;
      int mine = 0, other = 0, units = 0;  // S of this and of the other tile, and this tile's units, before
      bool ok = true;
      Walk walk(a);
      int u = walk.next(a);
      Item it = u >= 0 ? load_item(a, u) : Item{};
      while (ok && u >= 0) {
        const Unit x = make_unit(a, u, it);
        u = walk.next(a);
        if (u >= 0) it = load_item(a, u);
        const int my_nk = t ? x.nk[1] : x.nk[0], other_nk = t ? x.nk[0] : x.nk[1];
        const int row_w = x.row0 + t * BM + wq * 32;  // the warp's first row
        const int qrow = row_w + lane;
        if (my_nk == 0) {  // rows without keys (none, where the tile lies past the sequence)
          if (qrow < x.row_end) {
            uint4* dst = reinterpret_cast<uint4*>(a.out + static_cast<long long>(x.q_tok + qrow) * a.o_ss +
                                                  static_cast<long long>(x.h) * a.o_sh);
#pragma unroll
            for (int e = 0; e < HD / 8; ++e) dst[e] = make_uint4(0, 0, 0, 0);
            if (a.lse != nullptr) a.lse[static_cast<long long>(x.q_tok + qrow) * a.Hq + x.h] = -INFINITY;
          }
          other += other_nk;
          continue;
        }
        // this row sees the keys before `seen`
        const int seen = a.causal ? min(x.sk, x.q_offset + qrow + 1) : x.sk;
        // first key tile with a key that a row of the tile does not see
        const int j_mask = max(0, min(x.sk, a.causal ? x.q_offset + x.row0 + t * BM + 1 : x.sk)) / BN;
        float m2 = -INFINITY, l = 0.f;
        for (int j = 0; j < my_nk; ++j) {
          ok = __all_sync(FULL, mbar_wait_inl(bar(B_SFULL + t), (mine + j) & 1, ab, kDevErrTimeout));
          if (!ok) break;
          tc_fence_after();
          float s[BN];
          {
            uint32_t rr[BN];
            tmem_ld128(tS, rr);
#pragma unroll
            for (int e = 0; e < BN; ++e) s[e] = __uint_as_float(rr[e]);
          }
          // S_t's columns are free now: the MMA warp may compute S_t(j+1) into
          // them, and the other tile may store its P there
          tc_fence_before();
          mbar_arrive(bar(B_LOADED + t));
          if (j >= j_mask) {
            const int left = seen - j * BN;
#pragma unroll
            for (int c = 0; c < BN; ++c) s[c] = c < left ? s[c] : -INFINITY;
          }
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
          // Lazy rescale, as in the dense kernel: the running max only moves when it
          // grows by more than 8 (log2 units).
          float alpha = 1.0f;
          bool need = false;
          if (j == 0) {
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
          uint32_t pk[BN / 2];
          float2 ls0 = make_float2(0.f, 0.f), ls1 = make_float2(0.f, 0.f);
          const float2 sl2x2 = make_float2(sl2, sl2), negm = make_float2(-msub, -msub);
#pragma unroll
          for (int c = 0; c < BN / 2; ++c) {
            const float2 y = __ffma2_rn(make_float2(s[2 * c], s[2 * c + 1]), sl2x2, negm);
            const float2 p = make_float2(ex2_approx(y.x), ex2_approx(y.y));
            if (c & 1) ls1 = __fadd2_rn(ls1, p); else ls0 = __fadd2_rn(ls0, p);
            pk[c] = pack_bf16x2(p.x, p.y);
          }
          {
            const float2 ls = __fadd2_rn(ls0, ls1);
            l += ls.x + ls.y;
          }
          // P_t(j) goes into columns 64..127 of the other tile's S once the scores
          // there have been read: S_1(j) for tile 0, S_0(j+1) for tile 1 (whose
          // computation followed O_1 += P_1(j-1) V, the last reader of those
          // columns). Past the other tile's last key tile, wait for its last read
          // and for this tile's previous O += P V instead.
          {
            const int want = j + t;
            bool w = true;
            if (want < other_nk) {
              w = mbar_wait_inl(bar(B_LOADED + (t ^ 1)), (other + want) & 1, ab, kDevErrTimeout);
            } else {
              if (other_nk > 0)
                w = mbar_wait_inl(bar(B_LOADED + (t ^ 1)), (other + other_nk - 1) & 1, ab, kDevErrTimeout);
              if (w && j > 0) w = mbar_wait_inl(bar(B_ODONE + t), (mine + j - 1) & 1, ab, kDevErrTimeout);
            }
            ok = __all_sync(FULL, w);
            if (!ok) break;
            tc_fence_after();
          }
          tmem_st64(tP, pk);
          if (__any_sync(FULL, need)) {
            // O holds the sum up to tile j-1 once O += P(j-1) V has completed; the next
            // one is not issued before this warpgroup arrives on PFULL below
            ok = __all_sync(FULL, mbar_wait_inl(bar(B_ODONE + t), (mine + j - 1) & 1, ab, kDevErrTimeout));
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
          mbar_arrive(bar(B_PFULL + t));
        }
        if (!ok) break;
        ok = __all_sync(FULL, mbar_wait_inl(bar(B_OFINAL + t), units & 1, ab, kDevErrTimeout));
        if (!ok) break;
        tc_fence_after();
        const float inv = l > 0.f ? 1.0f / l : 0.f;
        const bool keyless = seen <= 0;  // 0, whatever V holds
        const int nrows = min(32, x.row_end - row_w);  // rows of this warp to store
        __nv_bfloat16* orow = a.out + static_cast<long long>(x.q_tok + row_w) * a.o_ss +
                              static_cast<long long>(x.h) * a.o_sh;
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // 64 dims
#pragma unroll
          for (int c4 = 0; c4 < 2; ++c4) {
            uint32_t rr[32];
            tmem_ld32(tO + static_cast<uint32_t>(64 * half + 32 * c4), rr);
            if (half == 1 && c4 == 1) {  // O_t has been read
              tc_fence_before();
              mbar_arrive(bar(B_OFREE + t));
            }
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
              pk[e] = keyless ? 0u
                              : pack_bf16x2(__uint_as_float(rr[2 * e]) * inv, __uint_as_float(rr[2 * e + 1]) * inv);
            // rows of 128 bytes, 16-byte chunks XORed with the row
#pragma unroll
            for (int v4 = 0; v4 < 4; ++v4)
              *reinterpret_cast<uint4*>(s_out + lane * 128 + 16 * ((4 * c4 + v4) ^ (lane & 7))) =
                  make_uint4(pk[4 * v4], pk[4 * v4 + 1], pk[4 * v4 + 2], pk[4 * v4 + 3]);
          }
          __syncwarp();
          // eight lanes per row: 128 bytes in one line
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int r = 4 * k + (lane >> 3), c = lane & 7;
            const uint4 v = *reinterpret_cast<const uint4*>(s_out + r * 128 + 16 * (c ^ (r & 7)));
            if (r < nrows)
              *reinterpret_cast<uint4*>(orow + static_cast<long long>(r) * a.o_ss + 64 * half + 8 * c) = v;
          }
          __syncwarp();
        }
        if (a.lse != nullptr && qrow < x.row_end)
          a.lse[static_cast<long long>(x.q_tok + qrow) * a.Hq + x.h] = (m2 + log2f(l)) * 0.69314718055994531f;
        mine += my_nk;
        other += other_nk;
        ++units;
      }
    }
  }

  __syncthreads();
  if (warp == WARP_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace ragged
}  // namespace atf

using namespace atf;

extern "C" int atf_prefill_ragged_plan(const AtfPrefillRaggedPlanParams* p, int32_t* plan_host, int64_t capacity,
                                       AtfPrefillRaggedPlan* out) {
  using namespace atf::ragged;
  if (p == nullptr || out == nullptr || p->qo_indptr_host == nullptr || p->kv_indptr_host == nullptr ||
      p->batch_size < 1 || (plan_host == nullptr && capacity > 0) || p->num_heads_q < 1 || p->num_heads_kv < 1 ||
      p->num_heads_q % p->num_heads_kv != 0 || p->num_sms < 0)
    return ATF_ERR_INVALID_ARG;
  long long n = 0;
  for (int b = 0; b < p->batch_size; ++b) {
    const long long nq = static_cast<long long>(p->qo_indptr_host[b + 1]) - p->qo_indptr_host[b];
    const long long nk = static_cast<long long>(p->kv_indptr_host[b + 1]) - p->kv_indptr_host[b];
    if (p->qo_indptr_host[b] < 0 || p->kv_indptr_host[b] < 0 || nq < 0 || nk < 0) return ATF_ERR_INVALID_ARG;
    if (nq > (1ll << 30) || nk > (1ll << 30)) return ATF_ERR_UNSUPPORTED;
    n += (nq + BM * NQ - 1) / (BM * NQ);
  }
  const long long units = n * p->num_heads_q;
  if (units > 0x3fffffffLL) return ATF_ERR_UNSUPPORTED;
  int sms = p->num_sms;
  if (sms == 0) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return ATF_ERR_CUDA;
  }
  const int ctas = static_cast<int>(units < sms ? units : sms);
  out->num_items = static_cast<int32_t>(n);
  out->num_ctas = ctas;
  out->plan_ints = 8 * n + ctas + 1 + units;
  if (plan_host == nullptr) return ATF_OK;
  if (capacity < out->plan_ints) return ATF_ERR_WORKSPACE;
  struct Planned {
    Item it;
    int steps[NQ];  // key tiles of each query tile
  };
  std::vector<Planned> all;
  all.reserve(static_cast<size_t>(n));
  for (int b = 0; b < p->batch_size; ++b) {
    Planned x = {};
    x.it.q_beg = p->qo_indptr_host[b];
    x.it.q_len = p->qo_indptr_host[b + 1] - p->qo_indptr_host[b];
    x.it.k_beg = p->kv_indptr_host[b];
    x.it.k_len = p->kv_indptr_host[b + 1] - p->kv_indptr_host[b];
    for (int row = 0; row < x.it.q_len; row += BM * NQ) {
      x.it.row = row;
      for (int t = 0; t < NQ; ++t) {
        long long kend = p->causal ? static_cast<long long>(x.it.k_len) - x.it.q_len + row + (t + 1) * BM : x.it.k_len;
        if (kend > x.it.k_len) kend = x.it.k_len;
        x.steps[t] = row + t * BM < x.it.q_len && kend > 0 ? static_cast<int>((kend + BN - 1) / BN) : 0;
      }
      all.push_back(x);
    }
  }
  auto longest = [](const Planned& x) { return x.steps[0] > x.steps[1] ? x.steps[0] : x.steps[1]; };
  std::stable_sort(all.begin(), all.end(),
                   [&](const Planned& x, const Planned& y) { return longest(x) > longest(y); });
  for (size_t i = 0; i < all.size(); ++i) std::memcpy(plan_host + 8 * i, &all[i].it, sizeof(Item));
  int32_t* offsets = plan_host + 8 * n;
  int32_t* list = offsets + ctas + 1;
  if (ctas == 0) {
    offsets[0] = 0;
    return ATF_OK;
  }
  // Each unit, in order, to the CTA with the least work so far (ties: the lowest),
  // in hundredths of a step of both tiles.
  const int G = p->num_heads_q / p->num_heads_kv;
  std::vector<int32_t> owner(static_cast<size_t>(units));
  std::vector<long long> count(static_cast<size_t>(ctas), 0);
  using Load = std::pair<long long, int>;
  std::vector<Load> heap;
  for (int c = 0; c < ctas; ++c) heap.emplace_back(0, c);
  const auto more = std::greater<Load>();
  std::make_heap(heap.begin(), heap.end(), more);
  size_t u = 0;
  for (int hk = 0; hk < p->num_heads_kv; ++hk)
    for (const Planned& x : all) {
      const int both = x.steps[0] < x.steps[1] ? x.steps[0] : x.steps[1];
      const long long cost = 100ll * both + 90ll * (longest(x) - both) + 180;
      for (int g = 0; g < G; ++g, ++u) {
        std::pop_heap(heap.begin(), heap.end(), more);
        heap.back().first += cost;
        owner[u] = heap.back().second;
        ++count[static_cast<size_t>(owner[u])];
        std::push_heap(heap.begin(), heap.end(), more);
      }
    }
  offsets[0] = 0;
  for (int c = 0; c < ctas; ++c) offsets[c + 1] = offsets[c] + static_cast<int32_t>(count[static_cast<size_t>(c)]);
  std::vector<int32_t> next(offsets, offsets + ctas);
  for (size_t i = 0; i < owner.size(); ++i) list[next[static_cast<size_t>(owner[i])]++] = static_cast<int32_t>(i);
  return ATF_OK;
}

extern "C" int atf_prefill_ragged_fwd(const AtfPrefillRaggedParams* p, atf_stream_t stream) {
  using namespace atf::ragged;
  if (p == nullptr || p->q == nullptr || p->k == nullptr || p->v == nullptr || p->out == nullptr ||
      p->plan == nullptr)
    return ATF_ERR_INVALID_ARG;
  if (p->head_dim != ATF_HEAD_DIM) return ATF_ERR_UNSUPPORTED;
  if (p->total_q < 1 || p->total_k < 1 || p->num_heads_q < 1 || p->num_heads_kv < 1 ||
      p->num_heads_q % p->num_heads_kv != 0 || p->num_items < 0 || p->num_ctas < 0)
    return ATF_ERR_INVALID_ARG;
  if (p->total_q > 0x7fffffffLL - BM * NQ || p->total_k > 0x7fffffffLL - BN || p->num_heads_q > (1 << 20))
    return ATF_ERR_UNSUPPORTED;
  if (p->qk_layout != ATF_LAYOUT_SORTED_PAIR && p->qk_layout != ATF_LAYOUT_ROTATE_HALF) return ATF_ERR_INVALID_ARG;
  if (p->window != ATF_WINDOW_OFF && p->window != ATF_WINDOW_SNAP16) return ATF_ERR_UNSUPPORTED;
  if (!(p->softmax_scale > 0.f)) return ATF_ERR_INVALID_ARG;
  if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->v) || !aligned16(p->out) || !aligned16(p->plan))
    return ATF_ERR_ALIGNMENT;
  const int64_t strides[8] = {p->q_stride_s, p->q_stride_h, p->k_stride_s, p->k_stride_h,
                              p->v_stride_s, p->v_stride_h, p->o_stride_s, p->o_stride_h};
  for (int i = 0; i < 8; ++i)
    if (strides[i] < 0 || (strides[i] & 7) != 0) return ATF_ERR_ALIGNMENT;
  if (p->window == ATF_WINDOW_SNAP16)
    for (int i = 0; i < ATF_MAX_LEVELS; ++i)
      if (p->zhi[i] < 0 || (i > 0 && p->zhi[i] > p->zhi[i - 1])) return ATF_ERR_INVALID_ARG;
  int dev = 0;
  int rc = check_device(&dev);
  if (rc != ATF_OK) return rc;
  if (p->num_items == 0 || p->num_ctas == 0) return ATF_OK;

  // one batch of all packed rows; only the K maps that the call reads are encoded
  CUtensorMap tq, tk, tv;
  KLevelMaps tkl;
  auto sane = [](int64_t stride, int64_t size) -> uint64_t {
    return static_cast<uint64_t>(size == 1 ? 16 : stride * 2);
  };
  const bool sorted = p->qk_layout == ATF_LAYOUT_SORTED_PAIR;
  const uint64_t nq = static_cast<uint64_t>(p->total_q), nk = static_cast<uint64_t>(p->total_k);
  const uint64_t hq = static_cast<uint64_t>(p->num_heads_q), hkv = static_cast<uint64_t>(p->num_heads_kv);
  {
    const uint64_t dims[4] = {128, nq, hq, 1};
    const uint64_t str[3] = {sane(p->q_stride_s, p->total_q), sane(p->q_stride_h, p->num_heads_q), 16};
    const uint32_t box[4] = {sorted ? 64u : 8u, static_cast<uint32_t>(BM), 1, 1};
    if ((rc = encode_tiled_bf16(&tq, p->q, 4, dims, str, box,
                                sorted ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE)) != ATF_OK)
      return rc;
  }
  const uint64_t ks = sane(p->k_stride_s, p->total_k), kh = sane(p->k_stride_h, p->num_heads_kv);
  if (!sorted) {
    const uint64_t dims[4] = {128, nk, hkv, 1};
    const uint64_t str[3] = {ks, kh, 16};
    const uint32_t box[4] = {8, static_cast<uint32_t>(BN), 1, 1};
    if ((rc = encode_tiled_bf16(&tk, p->k, 4, dims, str, box, CU_TENSOR_MAP_SWIZZLE_NONE)) != ATF_OK) return rc;
  } else {
    const uint64_t dims[5] = {16, nk, ATF_MAX_LEVELS, hkv, 1};
    const uint64_t str[4] = {ks, 32, kh, 16};
    for (int L = p->window ? 1 : ATF_MAX_LEVELS; L <= ATF_MAX_LEVELS; ++L) {
      const uint32_t box[5] = {16, static_cast<uint32_t>(BN), static_cast<uint32_t>(L), 1, 1};
      if ((rc = encode_tiled_bf16(&tkl.lv[L - 1], p->k, 5, dims, str, box, CU_TENSOR_MAP_SWIZZLE_32B)) != ATF_OK)
        return rc;
    }
  }
  {
    const uint64_t dims[4] = {128, nk, hkv, 1};
    const uint64_t str[3] = {sane(p->v_stride_s, p->total_k), sane(p->v_stride_h, p->num_heads_kv), 16};
    const uint32_t box[4] = {64, static_cast<uint32_t>(BN), 1, 1};
    if ((rc = encode_tiled_bf16(&tv, p->v, 4, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B)) != ATF_OK) return rc;
  }
  Args a = {};
  a.Hq = static_cast<int>(p->num_heads_q);
  a.G = static_cast<int>(p->num_heads_q / p->num_heads_kv);
  a.scale_log2 = p->softmax_scale * 1.4426950408889634f;
  a.causal = p->causal ? 1 : 0;
  a.layout = p->qk_layout;
  a.window = p->window == ATF_WINDOW_SNAP16 ? 1 : 0;
  for (int i = 0; i < ATF_MAX_LEVELS; ++i) a.zhi[i] = p->zhi[i];
  a.out = static_cast<__nv_bfloat16*>(p->out);
  a.o_ss = p->o_stride_s;
  a.o_sh = p->o_stride_h;
  a.lse = p->lse;
  a.err = p->error_flag;
  const long long units = static_cast<long long>(p->num_items) * a.Hq;
  if (units > 0x3fffffffLL) return ATF_ERR_UNSUPPORTED;
  a.items = p->plan;
  a.cta_units = p->plan + 8ll * p->num_items;
  a.units = a.cta_units + p->num_ctas + 1;
  a.n_items = p->num_items;
  a.n_units = static_cast<int>(units);
  a.total_q = p->total_q;
  a.total_k = p->total_k;
  if (cudaFuncSetAttribute(ragged_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(SMEM_BYTES)) != cudaSuccess)
    return ATF_ERR_CUDA;
  // setmaxnreg.inc waits until the block's launch registers cover the split:
  // never launch a build whose register count would leave it waiting
  static const int launch_regs = [] {
    cudaFuncAttributes fa{};
    return cudaFuncGetAttributes(&fa, ragged_kernel) == cudaSuccess ? fa.numRegs : 0;
  }();
  if (static_cast<long long>(launch_regs) * THREADS < REG_SPLIT_TOTAL) return ATF_ERR_UNSUPPORTED;
  ragged_kernel<<<static_cast<unsigned>(p->num_ctas), THREADS, SMEM_BYTES, reinterpret_cast<cudaStream_t>(stream)>>>(
      tq, tk, tkl, tv, a);
  return cudaGetLastError() == cudaSuccess ? ATF_OK : ATF_ERR_CUDA;
}
