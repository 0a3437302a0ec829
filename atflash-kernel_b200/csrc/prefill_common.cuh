// Pieces shared by the dense and the packed prefill kernels: MMA groups, tile sizes,
// shared memory slabs, the register split and the window's level counts.
#pragma once
#include "atf_internal.h"
#include "atf_ptx.cuh"

namespace atf {
namespace prefill {

// MMA groups are issued from one asm block each, under a single elect: the MMA
// warp shares its sub-partition with two softmax warps, so fewer instructions
// per tcgen05.mma keep the tensor pipe fed.
//
// one elected lane issues the 8 PV MMAs (K = 128 keys) of a tile and the commit
__device__ __forceinline__ void pv_group_asm(uint32_t o_tmem, uint32_t p_tmem, uint64_t vd, uint32_t idesc,
                                             uint32_t acc0, uint32_t bar_addr) {
  asm volatile(
      "{\n\t.reg .pred pe, pa;\n\t.reg .b64 b;\n\t.reg .b32 a;\n\t"
      "elect.sync _|pe, 0xffffffff;\n\t"
      "setp.ne.b32 pa, %4, 0;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, pa;\n\t"
      "add.u32 a, %1, 8;\n\tadd.u64 b, %2, 128;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, 1;\n\t"
      "add.u32 a, a, 8;\n\tadd.u64 b, b, 128;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, 1;\n\t"
      "add.u32 a, a, 8;\n\tadd.u64 b, b, 128;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, 1;\n\t"
      "add.u32 a, a, 8;\n\tadd.u64 b, b, 128;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, 1;\n\t"
      "add.u32 a, a, 8;\n\tadd.u64 b, b, 128;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, 1;\n\t"
      "add.u32 a, a, 8;\n\tadd.u64 b, b, 128;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, 1;\n\t"
      "add.u32 a, a, 8;\n\tadd.u64 b, b, 128;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, 1;\n\t"
      "@pe tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t}"
      ::"r"(o_tmem), "r"(p_tmem), "l"(vd), "r"(idesc), "r"(acc0), "r"(bar_addr)
      : "memory");
}
// one elected lane issues the L (1..8) QK MMAs of a tile and the commit; level
// i advances A and B by one 4 KB slab (descriptor start field += 256)
__device__ __forceinline__ void qk_group_asm(uint32_t d_tmem, uint64_t qd, uint64_t kd, uint32_t idesc, int L,
                                             uint32_t bar_addr) {
  asm volatile(
      "{\n\t.reg .pred pe, p1, p2, p3, p4, p5, p6, p7;\n\t.reg .b64 a, b;\n\t"
      "elect.sync _|pe, 0xffffffff;\n\t"
      "setp.gt.and.s32 p1, %4, 1, pe;\n\tsetp.gt.and.s32 p2, %4, 2, pe;\n\tsetp.gt.and.s32 p3, %4, 3, pe;\n\t"
      "setp.gt.and.s32 p4, %4, 4, pe;\n\tsetp.gt.and.s32 p5, %4, 5, pe;\n\tsetp.gt.and.s32 p6, %4, 6, pe;\n\t"
      "setp.gt.and.s32 p7, %4, 7, pe;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, 0;\n\t"
      "add.u64 a, %1, 256;\n\tadd.u64 b, %2, 256;\n\t"
      "@p1 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 256;\n\tadd.u64 b, b, 256;\n\t"
      "@p2 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 256;\n\tadd.u64 b, b, 256;\n\t"
      "@p3 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 256;\n\tadd.u64 b, b, 256;\n\t"
      "@p4 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 256;\n\tadd.u64 b, b, 256;\n\t"
      "@p5 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 256;\n\tadd.u64 b, b, 256;\n\t"
      "@p6 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "add.u64 a, a, 256;\n\tadd.u64 b, b, 256;\n\t"
      "@p7 tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n\t"
      "@pe tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t}"
      ::"r"(d_tmem), "l"(qd), "l"(kd), "r"(idesc), "r"(L), "r"(bar_addr)
      : "memory");
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

constexpr int BM = 128, BN = 128, HD = 128, NQ = 2, KST = 2, VST = 2;
// Warps 10 and 11 have no role: they complete the third warpgroup so that the
// register split below (setmaxnreg acts on whole warpgroups) can take
// registers from the producer / MMA group and give them to the softmax groups.
constexpr int WARP_LOAD = 8, WARP_MMA = 9, NUM_WARPS = 12, THREADS = NUM_WARPS * 32;
// Registers per thread after the split. The block launches with THREADS x the
// compiled count (168 under __launch_bounds__(THREADS, 1)); the host refuses to
// launch unless 128 x REG_SMALL + 256 x REG_SOFTMAX fits in that.
constexpr int REG_SMALL = 80, REG_SOFTMAX = 208;
constexpr long long REG_SPLIT_TOTAL = 128LL * REG_SMALL + 256LL * REG_SOFTMAX;
template <int N>
__device__ __forceinline__ void reg_dealloc() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_alloc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
constexpr uint32_t QHALF_BYTES = BM * 16;             // 2 KB
constexpr uint32_t QSLAB_BYTES = 2 * QHALF_BYTES;     // 4 KB
constexpr uint32_t QTILE_BYTES = 8 * QSLAB_BYTES;     // 32 KB
constexpr uint32_t KHALF_BYTES = BN * 16;             // 2 KB
constexpr uint32_t KSLAB_BYTES = 2 * KHALF_BYTES;     // 4 KB
constexpr uint32_t KSTAGE_BYTES = 8 * KSLAB_BYTES;    // 32 KB
// sorted-pair K tensor maps over (16 dims of a level, key, level, kv head,
// batch); map L-1 moves the box {16, 128, L}: exactly the L in-window levels,
// as [L][128 keys][32 B] with 32-byte swizzle
struct KLevelMaps {
  CUtensorMap lv[ATF_MAX_LEVELS];
};
constexpr uint32_t VBOX_BYTES = BN * 128;             // 16 KB
constexpr uint32_t VSTAGE_BYTES = 2 * VBOX_BYTES;     // 32 KB

constexpr uint32_t IDESC_QK = make_idesc_bf16(128, BN, 0, 0);
constexpr uint32_t IDESC_PV = make_idesc_bf16(128, HD, 0, 1);
constexpr uint32_t FULL = 0xffffffffu;

// levels of key tile j: the L (1..8) in-window 16-dim levels of the pair
__device__ __forceinline__ int levels_for(const int (&lim)[ATF_MAX_LEVELS], int j) {
  int L = 0;
#pragma unroll
  for (int i = 0; i < ATF_MAX_LEVELS; ++i) L += j >= lim[i] ? 1 : 0;
  return L;
}
// Column of the first element of half `hh` of level `i` along head_dim.
// sorted-pair order: level i = dims [16i, 16i+16).
// rotate_half order (HF): sorted pairs 8i..8i+7 are HF dims [56-8i, 64-8i) and
// [120-8i, 128-8i).
__device__ __forceinline__ int level_col(int layout, int i, int hh) {
  return layout == ATF_LAYOUT_SORTED_PAIR ? 16 * i + 8 * hh : 64 * hh + 8 * (7 - i);
}

// Waits with no abort short-cut: used to drain this CTA's own asynchronous
// copies / MMAs before the CTA's shared memory or TMEM is released.
__device__ __forceinline__ void drain_wait(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer_ns() - t0 > kWaitLimitNs) break;
  }
}

}  // namespace prefill
}  // namespace atf
