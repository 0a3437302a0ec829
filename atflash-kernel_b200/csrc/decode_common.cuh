// Pieces shared by the bf16 and the e4m3 decode kernels: window limits on local
// keys, fragment loads and the launch.
#pragma once
#include <limits.h>

#include "atf_internal.h"

namespace atf {
namespace decode {

// The window as limits on local key indices, computed once per CTA and kept in
// registers: a key of local index n is at distance z = zb - n (zb = q_pos -
// kv_pos0) and reads a level or chunk whose zhi is >= z, i.e. when n >= zb - zhi.
// Per-key level counts are then 32-bit compares against registers; evaluating
// 64-bit distances against the table in the kernel parameters for every key
// group took most of a consumer warp's time per stage.
__device__ __forceinline__ int key_limit(long long zb, long long zhi) {
  const long long v = zb - zhi;
  return static_cast<int>(v < INT_MIN ? INT_MIN : (v > INT_MAX ? INT_MAX : v));
}
// levels read by local key n
__device__ __forceinline__ int levels_of(const int (&lim)[ATF_MAX_LEVELS], int n) {
  int L = 0;
#pragma unroll
  for (int i = 0; i < ATF_MAX_LEVELS; ++i) L += n >= lim[i] ? 1 : 0;
  return L;
}

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2,
                                        uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2,
                                          uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
// Transpose of an 8x8 b16 matrix held one row pair per thread (the mma
// fragment layout): lane (g, t4) gets elements (2 t4, g) and (2 t4 + 1, g).
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace decode

// A kernel launch, with programmatic stream serialization when `pdl`: the grid
// may then start while the previous kernel on the stream is still running; the
// decode kernels read only the plan and the page table before their
// griddepcontrol.wait.
template <typename... KArgs, typename... Args>
static cudaError_t launch_pdl(void (*kern)(KArgs...), dim3 grid, int threads, uint32_t smem, cudaStream_t st,
                              bool pdl, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace atf
