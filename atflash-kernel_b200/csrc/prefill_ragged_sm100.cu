// Causal or full attention over packed sequences of different lengths, for sm_100a.
//
// Mathematics, tiles and pipeline are the dense prefill's (prefill_sm100.cu): per
// query row an online softmax in the log2 domain over 128-key tiles, S = Q K^T over
// the window's 16-dim levels and O += P V on the tensor cores with both accumulators
// in TMEM, P in bf16; a producer warp, an MMA warp and two softmax groups. A
// sequence's rows are those of a dense run of its own, bit for bit: the window is
// quantised per (query tile, key tile) from the sequence's own first row and key.
//
// CTA = (block of 256 query rows of a sequence, query head). The plan lists the blocks
// of all sequences by falling key count. Where K and V of all heads fit L2 beside the
// rest, the grid walks blocks, then heads: the longest start first and the last ones
// are the shortest (one prompt of 2500, 24 / 8 heads, 65 -> 45 us; of 8000 383 -> 338-350).
// Else it walks kv heads, then blocks, then the heads of the group, so that CTAs
// resident together share K and V in L2 (both ways within 3% at 100 MB and more).
//
// P is rounded to bf16 (8 bits) for the product with V: both operands of the tensor
// core's f16 kind have one type, and V is bf16. The row sum adds P as it was in fp32.
//
// What bounds it: a step of two query tiles against a key tile takes 1.65 us (1.5 where
// the window leaves half of K; exponentials and tensor work, as in the dense kernel),
// and a CTA's start and end cost extra, which short sequences feel. So Q comes in
// rows of 128 bytes (two boxes of 64 dims, 128-byte swizzle; 8-dim boxes as in the
// dense kernel took 1-2 us longer; rotate_half keeps them), the item, the error flag,
// the barriers and TMEM are set up side by side, and the outputs leave through shared
// memory in whole lines. A persistent form of this kernel, whose next unit's loads
// and scores ran under the epilogue, cost 2.5 us less per block but 0.3 us more per
// step: its barrier phases and stages, counted on through the units, are no longer
// known to be uniform, and the MMA warp's issue is what a step waits for. It lost
// wherever a block has more than about 8 key tiles.
//
// A tile's last box may reach into the next sequence: its queries are not stored, its
// keys are masked, and its V rows, whose P is 0, are cleared in shared memory before
// the product (they may hold anything, NaN included).
#include <math.h>

#include <algorithm>
#include <cstring>
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
constexpr uint32_t OFF_BAR = OFF_V + VST * VSTAGE_BYTES;

enum {
  B_Q = 0,
  B_KFULL = 1,
  B_KEMPTY = B_KFULL + KST,
  B_VFULL = B_KEMPTY + KST,
  B_VEMPTY = B_VFULL + VST,
  B_SFULL = B_VEMPTY + VST,   // [t]
  B_PFULL = B_SFULL + NQ,     // [t]
  B_ODONE = B_PFULL + NQ,     // [t], one phase per O += P V
  B_OFINAL = B_ODONE + NQ,    // [t], single phase: the tile's last O += P V done
  B_LOADED = B_OFINAL + NQ,   // [t], phase j: tile t's softmax has read S_t(j) into registers
  B_FINAL = B_LOADED + NQ,
  NUM_BARS
};
constexpr uint32_t OFF_ABORT = OFF_BAR + 8 * NUM_BARS;
constexpr uint32_t OFF_TMEM = OFF_ABORT + 16;
constexpr uint32_t SMEM_BYTES = OFF_TMEM + 16 + 1024;  // slack for 1024-B alignment

// One work item of the plan: 256 query rows from `row` on of one sequence. Rows and
// keys are the sequence's own; the packed tensors hold them from q_beg and k_beg on.
struct Item {
  int q_beg, q_len, k_beg, k_len, row, pad[3];
};
static_assert(sizeof(Item) == 32, "eight ints per item");

struct Args {
  int Hq, G, walk;
  float scale_log2;
  int causal, layout, window;
  int zhi[ATF_MAX_LEVELS];
  __nv_bfloat16* out;
  long long o_ss, o_sh;
  float* lse;
  int* err;
  const int* items;
  int n_items;
  long long total_q, total_k;
};

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
                   const __grid_constant__ KLevelMaps tmKL,
                   const __grid_constant__ CUtensorMap tmV, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  const uint32_t sb = (raw_u32 + 1023u) & ~1023u;
  uint8_t* sp = smem_raw + (sb - raw_u32);
  volatile int* s_abort = reinterpret_cast<volatile int*>(sp + OFF_ABORT);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(sp + OFF_TMEM);
  auto bar = [&](int i) -> uint32_t { return sb + OFF_BAR + 8u * static_cast<uint32_t>(i); };

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  // This CTA's unit. Its loads are issued side by side: thread 0's of the error flag
  // does not hold up the barriers, and the barriers do not wait for the item.
  const int per_walk = a.n_items * a.walk;  // a walk over the items, with `walk` heads
  const int rem = static_cast<int>(blockIdx.x) % per_walk;
  const int h = static_cast<int>(blockIdx.x) / per_walk * a.walk + rem % a.walk;
  const int hk = h / a.G;
  const int4* src = reinterpret_cast<const int4*>(a.items) + 2 * (rem / a.walk);
  const int4 it0 = __ldg(src), it1 = __ldg(src + 1);
  const bool stop0 = threadIdx.x == 0 && stops(a.err);
  if (threadIdx.x == 0) {
    mbar_init(bar(B_Q), 1);
    for (int s = 0; s < KST; ++s) {
      mbar_init(bar(B_KFULL + s), 1);
      mbar_init(bar(B_KEMPTY + s), 1);
    }
    for (int s = 0; s < VST; ++s) {
      mbar_init(bar(B_VFULL + s), 1);
      mbar_init(bar(B_VEMPTY + s), 1);
    }
    for (int t = 0; t < NQ; ++t) {
      mbar_init(bar(B_SFULL + t), 1);
      mbar_init(bar(B_PFULL + t), 128);
      mbar_init(bar(B_ODONE + t), 1);
      mbar_init(bar(B_OFINAL + t), 1);
      mbar_init(bar(B_LOADED + t), 128);
    }
    mbar_init(bar(B_FINAL), 1);
    fence_mbar_init();
  }
  if (warp == WARP_LOAD && lane == 0) {
    tma_prefetch_desc(&tmQ);
    // only the maps that this call uses are there
    if (a.layout != ATF_LAYOUT_SORTED_PAIR)
      tma_prefetch_desc(&tmK);
    else
      for (int L = a.window ? 0 : ATF_MAX_LEVELS - 1; L < ATF_MAX_LEVELS; ++L) tma_prefetch_desc(&tmKL.lv[L]);
    tma_prefetch_desc(&tmV);
  }
  if (warp == WARP_MMA) {
    tmem_alloc(smem_u32(s_tmem), 512);
    tmem_relinquish();
  }
  // first packed row of the sequence's queries and keys, its keys, its rows and the
  // position of its query row 0 among its keys (negative: rows without keys)
  const int q_tok = it0.x, k_tok = it0.z, sk = it0.w, row_base = it1.x;
  const int q_offset = it0.w - it0.y;
  // an item outside the packed rows (a plan made for others) has no rows
  const bool bad = it0.x < 0 || it0.y < 0 || it0.z < 0 || it0.w < 0 || it1.x < 0 ||
                   static_cast<long long>(it0.x) + it0.y > a.total_q ||
                   static_cast<long long>(it0.z) + it0.w > a.total_k;
  const int row_end = bad ? 0 : it0.y;
  if (threadIdx.x == 0) {
    *s_abort = stop0 ? 1 : 0;
    if (bad && a.err != nullptr) atomicCAS(a.err, 0, kDevErrIndex);
  }
  int row0[NQ], nk[NQ];
#pragma unroll
  for (int t = 0; t < NQ; ++t) {
    row0[t] = row_base + t * BM;
    if (row0[t] >= row_end) {
      nk[t] = 0;
    } else {
      const int kend = a.causal ? min(q_offset + row0[t] + BM, sk) : sk;
      nk[t] = kend > 0 ? (kend + BN - 1) / BN : 0;
    }
  }
  const int nk_max = nk[0] > nk[1] ? nk[0] : nk[1];
  int lim[NQ][ATF_MAX_LEVELS];
#pragma unroll
  for (int t = 0; t < NQ; ++t) window_limits(a, q_offset, row0[t], lim[t]);

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
      // All 32 lanes run this loop with warp-uniform values; one elected lane
      // issues each TMA / expect_tx.
      int issued_k = 0, issued_v = 0;
      bool ok = true;
      {
        uint32_t qbytes = 0;
#pragma unroll
        for (int t = 0; t < NQ; ++t) qbytes += nk[t] > 0 ? QTILE_BYTES : 0u;
        mbar_arrive_expect_tx_elect(bar(B_Q), qbytes);
#pragma unroll
        for (int t = 0; t < NQ; ++t) {
          if (nk[t] == 0) continue;
          if (a.layout == ATF_LAYOUT_SORTED_PAIR) {
            // two boxes of 128-byte rows: an eighth of the 8-dim boxes' row pieces
            tma_load_4d_elect(sb + OFF_Q + t * QTILE_BYTES, &tmQ, bar(B_Q), 0, q_tok + row0[t], h, 0);
            tma_load_4d_elect(sb + OFF_Q + t * QTILE_BYTES + QTILE_BYTES / 2, &tmQ, bar(B_Q), 64, q_tok + row0[t], h,
                              0);
            continue;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
              tma_load_4d_elect(sb + OFF_Q + t * QTILE_BYTES + i * QSLAB_BYTES + hh * QHALF_BYTES, &tmQ,
                                bar(B_Q), level_col(a.layout, i, hh), q_tok + row0[t], h, 0);
        }
      }
      for (int j = 0; j < nk_max; ++j) {
        const int ks = j % KST, vs = j % VST;
        ok = __all_sync(FULL, mbar_wait_inl(bar(B_KEMPTY + ks), ((j / KST) & 1) ^ 1, ab, kDevErrTimeout));
        if (!ok) break;
        int L = 0;
#pragma unroll
        for (int t = 0; t < NQ; ++t)
          if (j < nk[t]) {
            const int lt = levels_for(lim[t], j);
            L = lt > L ? lt : L;
          }
        const uint32_t kdst = sb + OFF_K + ks * KSTAGE_BYTES;
        if (a.layout == ATF_LAYOUT_SORTED_PAIR) {
          // one 5-d box: the L in-window levels (dims 0..16L-1), one 4 KB slab each
          mbar_arrive_expect_tx_elect(bar(B_KFULL + ks), static_cast<uint32_t>(L) * KSLAB_BYTES);
          if (elect_one_lane()) tma_load_5d(kdst, &tmKL.lv[L - 1], bar(B_KFULL + ks), 0, k_tok + j * BN, 0, hk, 0);
          __syncwarp();
        } else {
          // rotate_half: a level is two 8-dim chunks 64 dims apart, one box each
          mbar_arrive_expect_tx_elect(bar(B_KFULL + ks), static_cast<uint32_t>(L) * KSLAB_BYTES);
          for (int i = 0; i < L; ++i) {
            tma_load_4d_elect(kdst + i * KSLAB_BYTES, &tmK, bar(B_KFULL + ks), level_col(a.layout, i, 0),
                              k_tok + j * BN, hk, 0);
            tma_load_4d_elect(kdst + i * KSLAB_BYTES + KHALF_BYTES, &tmK, bar(B_KFULL + ks),
                              level_col(a.layout, i, 1), k_tok + j * BN, hk, 0);
          }
        }
        issued_k = j + 1;
        ok = __all_sync(FULL, mbar_wait_inl(bar(B_VEMPTY + vs), ((j / VST) & 1) ^ 1, ab, kDevErrTimeout));
        if (!ok) break;
        mbar_arrive_expect_tx_elect(bar(B_VFULL + vs), VSTAGE_BYTES);
        tma_load_4d_elect(sb + OFF_V + vs * VSTAGE_BYTES, &tmV, bar(B_VFULL + vs), 0, k_tok + j * BN, hk, 0);
        tma_load_4d_elect(sb + OFF_V + vs * VSTAGE_BYTES + VBOX_BYTES, &tmV, bar(B_VFULL + vs), 64,
                          k_tok + j * BN, hk, 0);
        issued_v = j + 1;
      }
      // Drain: every copy this warp issued must land before shared memory is
      // released (no-op on the normal path, where the MMA warp consumed them).
      drain_wait(bar(B_Q), 0);
      for (int j = issued_k - KST; j < issued_k; ++j)
        if (j >= 0) drain_wait(bar(B_KFULL + j % KST), (j / KST) & 1);
      for (int j = issued_v - VST; j < issued_v; ++j)
        if (j >= 0) drain_wait(bar(B_VFULL + j % VST), (j / VST) & 1);
      __syncwarp();
    } else if (start_ok && warp == WARP_MMA) {
      // ---------------------------------------------------------------- MMA issuer
      // Descriptors are built once and advanced by adding (byte offset >> 4) to
      // the start-address field (all offsets stay inside the 14-bit field).
      const uint32_t tm = __shfl_sync(FULL, tmem, 0);
      const uint64_t qdesc0 = make_sdesc(sb + OFF_Q, QHALF_BYTES, 128, kLayoutNone);
      const uint64_t qrows0 = make_sdesc(sb + OFF_Q, 16, 1024, kLayoutSw128);
      const uint64_t kdesc0 = make_sdesc(sb + OFF_K, KHALF_BYTES, 128, kLayoutNone);
      // sorted-pair K level slabs: 128 keys x 32 B, 32-byte swizzle (SBO = 8 rows)
      const uint64_t kdesc32 = make_sdesc(sb + OFF_K, 16, 256, kLayoutSw32);
      const bool sorted = a.layout == ATF_LAYOUT_SORTED_PAIR;
      const uint64_t vdesc0 = make_sdesc(sb + OFF_V, VBOX_BYTES, 1024, kLayoutSw128);
      const int nk0 = nk[0], nk1 = nk[1];
      // S_t(j) into tile t's S columns
      auto issue_S = [&](int t, int j) {
        const int L = levels_for(lim[t], j);
        const uint32_t d_tmem = tm + static_cast<uint32_t>(t * 128);
        const uint64_t qd = qdesc0 + ((t * QTILE_BYTES) >> 4);
        const uint64_t kd = (sorted ? kdesc32 : kdesc0) + (((j % KST) * KSTAGE_BYTES) >> 4);
        if (sorted)
          qk_group_rows_asm(d_tmem, qrows0 + ((t * QTILE_BYTES) >> 4), kd, IDESC_QK, L, bar(B_SFULL + t));
        else
          qk_group_asm(d_tmem, qd, kd, IDESC_QK, L, bar(B_SFULL + t));
      };
      // O_t += P_t(j) V_j; P_t sits in columns 64..127 of the other tile's S
      auto issue_PV = [&](int t, int j) {
        const uint32_t o_tmem = tm + 256u + static_cast<uint32_t>(t * 128);
        const uint32_t p_tmem = tm + static_cast<uint32_t>((1 - t) * 128 + 64);
        const uint64_t vd = vdesc0 + (((j % VST) * VSTAGE_BYTES) >> 4);
        pv_group_asm(o_tmem, p_tmem, vd, IDESC_PV, j > 0 ? 1u : 0u, bar(B_ODONE + t));
      };
      // K tiles are waited for in order, once each
      int k_waited = -1;
      auto kwait = [&](int j) -> bool {
        while (k_waited < j) {
          ++k_waited;
          if (!__all_sync(FULL, mbar_wait_inl(bar(B_KFULL + k_waited % KST), (k_waited / KST) & 1, ab,
                                          kDevErrTimeout)))
            return false;
          tc_fence_after();
        }
        return true;
      };
      auto wait_loaded = [&](int t, int j) -> bool {
        const bool w = __all_sync(FULL, mbar_wait_inl(bar(B_LOADED + t), j & 1, ab, kDevErrTimeout));
        tc_fence_after();
        return w;
      };
      // A K stage is released after the last S that reads it: S_1(j) when tile 1
      // has key tile j, else S_0(j).
      bool ok = __all_sync(FULL, mbar_wait_inl(bar(B_Q), 0, ab, kDevErrTimeout));
      tc_fence_after();
      if (ok && nk_max > 0 && (ok = kwait(0))) {
        if (nk0 > 0) issue_S(0, 0);
        if (nk1 > 0) issue_S(1, 0);
        tc_commit_elect(bar(B_KEMPTY + 0));
      }
      // S_0(1) once tile 0 has read S_0(0)
      if (ok && nk0 > 1 && (ok = kwait(1) && wait_loaded(0, 0))) {
        issue_S(0, 1);
        if (1 >= nk1) tc_commit_elect(bar(B_KEMPTY + 1 % KST));
      }
      for (int j = 0; ok && j < nk_max; ++j) {
        const int vs = j % VST;
        ok = __all_sync(FULL, mbar_wait_inl(bar(B_VFULL + vs), (j / VST) & 1, ab, kDevErrTimeout));
        if (!ok) break;
        {
          // V rows past the sequence's last key: another sequence's
          const int live = sk - j * BN;
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
        }
        tc_fence_after();
        if (j < nk0) {
          ok = __all_sync(FULL, mbar_wait_inl(bar(B_PFULL + 0), j & 1, ab, kDevErrTimeout));
          if (!ok) break;
          tc_fence_after();
          issue_PV(0, j);
          if (j + 1 == nk0) tc_commit_elect(bar(B_OFINAL + 0));
        }
        // S_1(j+1) overwrites the columns P_0(j) occupies (O_0 += P_0(j) V_j was
        // issued first; tcgen05.mma ops of one thread run in order) and needs
        // tile 1 to have read S_1(j)
        if (j + 1 < nk1) {
          if (!(ok = kwait(j + 1) && wait_loaded(1, j))) break;
          issue_S(1, j + 1);
          tc_commit_elect(bar(B_KEMPTY + (j + 1) % KST));
        }
        if (j < nk1) {
          ok = __all_sync(FULL, mbar_wait_inl(bar(B_PFULL + 1), j & 1, ab, kDevErrTimeout));
          if (!ok) break;
          tc_fence_after();
          issue_PV(1, j);
          if (j + 1 == nk1) tc_commit_elect(bar(B_OFINAL + 1));
        }
        // S_0(j+2): after O_1 += P_1(j) V_j (P_1(j) sits in S_0's columns) and
        // tile 0's read of S_0(j+1)
        if (j + 2 < nk0) {
          if (!(ok = kwait(j + 2) && wait_loaded(0, j + 1))) break;
          issue_S(0, j + 2);
          if (j + 2 >= nk1) tc_commit_elect(bar(B_KEMPTY + (j + 2) % KST));
        }
        tc_commit_elect(bar(B_VEMPTY + vs));
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
        const int my_row0 = t ? row0[1] : row0[0];
        const int my_nk = t ? nk[1] : nk[0];
        const int row_w = my_row0 + wq * 32;  // the warp's first row
        const int qrow = row_w + lane;
        // this row sees the keys before `seen`; from key tile j_mask on, a row of the
        // tile does not see every key
        const int seen = a.causal ? min(sk, q_offset + qrow + 1) : sk;
        const int j_mask = max(0, a.causal ? min(sk, q_offset + my_row0 + 1) : sk) / BN;
        const float sl2 = a.scale_log2;
        float m2 = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; j < my_nk; ++j) {
          ok = __all_sync(FULL, mbar_wait_inl(bar(B_SFULL + t), j & 1, ab, kDevErrTimeout));
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
          // Lazy rescale: the running max only moves when it grows by more than
          // 8 (log2 units), so P <= 2^8 stays exact enough in bf16 and O is
          // rescaled rarely. The O update itself happens after P is stored.
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
          // exponentials, the row sum and the bf16 packing of P, two columns at a
          // time with packed f32x2 arithmetic (half the FMA / add instructions)
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
          // P_t(j) goes into columns 64..127 of the other tile's S once the scores
          // there have been read: S_1(j) for tile 0, S_0(j+1) for tile 1 (whose
          // computation followed O_1 += P_1(j-1) V, the last reader of those
          // columns). Past the other tile's last key tile, wait for its last read
          // and for this tile's previous O += P V instead.
          {
            const int other_nk = t ? nk[0] : nk[1];
            const int want = j + t;  // tile 0: S_1(j); tile 1: S_0(j + 1)
            bool w = true;
            if (want < other_nk) {
              w = mbar_wait_inl(bar(B_LOADED + (t ^ 1)), want & 1, ab, kDevErrTimeout);
            } else {
              if (other_nk > 0) w = mbar_wait_inl(bar(B_LOADED + (t ^ 1)), (other_nk - 1) & 1, ab, kDevErrTimeout);
              if (w && j > 0) w = mbar_wait_inl(bar(B_ODONE + t), (j - 1) & 1, ab, kDevErrTimeout);
            }
            ok = __all_sync(FULL, w);
            if (!ok) break;
            tc_fence_after();
          }
          tmem_st64(tP, pk);
          if (__any_sync(FULL, need)) {
            // O holds the sum up to tile j-1 once PV(t, j-1) has completed (S_t(j) was
            // issued after it, so at most that one is in flight); PV(t, j) is not
            // issued before this warpgroup arrives on PFULL below.
            ok = __all_sync(FULL, mbar_wait_inl(bar(B_ODONE + t), (j - 1) & 1, ab, kDevErrTimeout));
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
        if (ok && my_nk > 0) {
          ok = __all_sync(FULL, mbar_wait_inl(bar(B_OFINAL + t), 0, ab, kDevErrTimeout));
          if (ok) {
            tc_fence_after();
            const float inv = l > 0.f ? 1.0f / l : 0.f;
            const bool keyless = seen <= 0;             // 0, whatever V holds
            const int nrows = min(32, row_end - row_w);  // rows of this warp to store
            // Through the tile's own Q in shared memory (its last product has read it):
            // rows of 128 bytes, 16-byte chunks XORed with the row, then eight lanes per
            // row, so that whole 128-byte lines leave.
            uint8_t* s_out = sp + OFF_Q + t * QTILE_BYTES + wq * (32 * 128);
            __nv_bfloat16* orow = a.out + static_cast<long long>(q_tok + row_w) * a.o_ss +
                                  static_cast<long long>(h) * a.o_sh;
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // 64 dims
#pragma unroll
              for (int c4 = 0; c4 < 2; ++c4) {
                uint32_t rr[32];
                tmem_ld32(tO + static_cast<uint32_t>(64 * half + 32 * c4), rr);
                uint32_t pk[16];
#pragma unroll
                for (int e = 0; e < 16; ++e)
                  pk[e] = keyless ? 0u
                                  : pack_bf16x2(__uint_as_float(rr[2 * e]) * inv, __uint_as_float(rr[2 * e + 1]) * inv);
#pragma unroll
                for (int v4 = 0; v4 < 4; ++v4)
                  *reinterpret_cast<uint4*>(s_out + lane * 128 + 16 * ((4 * c4 + v4) ^ (lane & 7))) =
                      make_uint4(pk[4 * v4], pk[4 * v4 + 1], pk[4 * v4 + 2], pk[4 * v4 + 3]);
              }
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int r = 4 * i + (lane >> 3), c = lane & 7;
                const uint4 v = *reinterpret_cast<const uint4*>(s_out + r * 128 + 16 * (c ^ (r & 7)));
                if (r < nrows)
                  *reinterpret_cast<uint4*>(orow + static_cast<long long>(r) * a.o_ss + 64 * half + 8 * c) = v;
              }
              __syncwarp();
            }
            if (a.lse != nullptr && qrow < row_end)
              a.lse[static_cast<long long>(q_tok + qrow) * a.Hq + h] = (m2 + log2f(l)) * 0.69314718055994531f;
          }
        }
        if (my_nk == 0 && qrow < row_end) {  // a tile whose rows have no keys
          uint4* dst = reinterpret_cast<uint4*>(a.out + static_cast<long long>(q_tok + qrow) * a.o_ss +
                                                static_cast<long long>(h) * a.o_sh);
#pragma unroll
          for (int e = 0; e < HD / 8; ++e) dst[e] = make_uint4(0, 0, 0, 0);
          if (a.lse != nullptr) a.lse[static_cast<long long>(q_tok + qrow) * a.Hq + h] = -INFINITY;
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

extern "C" int atf_prefill_ragged_plan(const AtfPrefillRaggedPlanParams* p, int32_t* items_host,
                                       int32_t items_capacity, int32_t* num_items) {
  using namespace atf::ragged;
  if (p == nullptr || num_items == nullptr || p->qo_indptr_host == nullptr || p->kv_indptr_host == nullptr ||
      p->batch_size < 1 || (items_host == nullptr && items_capacity > 0))
    return ATF_ERR_INVALID_ARG;
  long long n = 0;
  for (int b = 0; b < p->batch_size; ++b) {
    const long long nq = static_cast<long long>(p->qo_indptr_host[b + 1]) - p->qo_indptr_host[b];
    const long long nk = static_cast<long long>(p->kv_indptr_host[b + 1]) - p->kv_indptr_host[b];
    if (p->qo_indptr_host[b] < 0 || p->kv_indptr_host[b] < 0 || nq < 0 || nk < 0) return ATF_ERR_INVALID_ARG;
    if (nq > (1ll << 30) || nk > (1ll << 30)) return ATF_ERR_UNSUPPORTED;
    n += (nq + BM * NQ - 1) / (BM * NQ);
  }
  if (n > 0x7fffffffLL) return ATF_ERR_UNSUPPORTED;
  *num_items = static_cast<int32_t>(n);
  if (items_host == nullptr) return ATF_OK;
  if (n > items_capacity) return ATF_ERR_WORKSPACE;
  struct Planned {
    long long tiles;
    Item it;
  };
  std::vector<Planned> all;
  try {
    all.reserve(static_cast<size_t>(n));
  } catch (...) {  // no host memory for the schedule
    return ATF_ERR_WORKSPACE;
  }
  for (int b = 0; b < p->batch_size; ++b) {
    Planned x = {};
    x.it.q_beg = p->qo_indptr_host[b];
    x.it.q_len = p->qo_indptr_host[b + 1] - p->qo_indptr_host[b];
    x.it.k_beg = p->kv_indptr_host[b];
    x.it.k_len = p->kv_indptr_host[b + 1] - p->kv_indptr_host[b];
    for (int row = 0; row < x.it.q_len; row += BM * NQ) {
      x.it.row = row;
      long long kend = p->causal ? static_cast<long long>(x.it.k_len) - x.it.q_len + row + BM * NQ : x.it.k_len;
      kend = kend > x.it.k_len ? x.it.k_len : (kend < 0 ? 0 : kend);
      x.tiles = (kend + BN - 1) / BN;
      all.push_back(x);
    }
  }
  std::stable_sort(all.begin(), all.end(), [](const Planned& x, const Planned& y) { return x.tiles > y.tiles; });
  for (size_t i = 0; i < all.size(); ++i) std::memcpy(items_host + 8 * i, &all[i].it, sizeof(Item));
  return ATF_OK;
}

extern "C" int atf_prefill_ragged_fwd(const AtfPrefillRaggedParams* p, atf_stream_t stream) {
  using namespace atf::ragged;
  if (p == nullptr || p->q == nullptr || p->k == nullptr || p->v == nullptr || p->out == nullptr ||
      p->items == nullptr)
    return ATF_ERR_INVALID_ARG;
  if (p->head_dim != ATF_HEAD_DIM) return ATF_ERR_UNSUPPORTED;
  if (p->total_q < 1 || p->total_k < 1 || p->num_heads_q < 1 || p->num_heads_kv < 1 ||
      p->num_heads_q % p->num_heads_kv != 0 || p->num_items < 0)
    return ATF_ERR_INVALID_ARG;
  if (p->total_q > 0x7fffffffLL - BM * NQ || p->total_k > 0x7fffffffLL - BN || p->num_heads_q > (1 << 20))
    return ATF_ERR_UNSUPPORTED;
  if (p->qk_layout != ATF_LAYOUT_SORTED_PAIR && p->qk_layout != ATF_LAYOUT_ROTATE_HALF) return ATF_ERR_INVALID_ARG;
  if (p->window != ATF_WINDOW_OFF && p->window != ATF_WINDOW_SNAP16) return ATF_ERR_UNSUPPORTED;
  if (!(p->softmax_scale > 0.f)) return ATF_ERR_INVALID_ARG;
  if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->v) || !aligned16(p->out) || !aligned16(p->items))
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
  if (p->num_items == 0) return ATF_OK;

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
  const bool in_l2 = p->total_k * p->num_heads_kv * 512 <= (64ll << 20);
  a.walk = in_l2 ? a.Hq : static_cast<int>(p->num_heads_q / p->num_heads_kv);
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
  a.items = p->items;
  a.n_items = p->num_items;
  a.total_q = p->total_q;
  a.total_k = p->total_k;
  const long long units = static_cast<long long>(p->num_items) * a.Hq;
  if (units > 0x7fffffffLL) return ATF_ERR_UNSUPPORTED;
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
  ragged_kernel<<<static_cast<unsigned>(units), THREADS, SMEM_BYTES, reinterpret_cast<cudaStream_t>(stream)>>>(
      tq, tk, tkl, tv, a);
  return cudaGetLastError() == cudaSuccess ? ATF_OK : ATF_ERR_CUDA;
}
