// RMS norm of a 128-element row held by 8 lanes, with the rotation behind it: shared by
// the norm kernel and the appends. Lane c (0..7) holds the HF pairs 8c..8c+7, elements
// x1 = dims [8c, 8c+8) and x2 = dims [64+8c, 64+8c+8).
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "rope_math.cuh"

namespace atf {
namespace normmath {

__device__ __forceinline__ float weight_at(const void* w, bool f32, int i) {
  return f32 ? static_cast<const float*>(w)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// 8 floats from a 16-byte aligned address (generic)
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// 8 bf16 to fp32
__device__ __forceinline__ void unpack(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// weights i .. i + 7, bf16 or fp32, 16-byte aligned
__device__ __forceinline__ void weights8(const void* w, bool f32, int i, float (&v)[8]) {
  if (f32)
    load8(static_cast<const float*>(w) + i, v);
  else
    unpack(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(w) + i), v);
}

// x <- (x / sqrt(mean(x^2) + eps)) w over the row of the 8 lanes; `mask` names the lanes
// that take part (whole groups of 8). fp32 throughout: the 128 squares' sum is off by at
// most 2^-20 of itself, the rest by a few units of 2^-24, far under the one rounding to
// bf16 (2^-9) that follows.
__device__ __forceinline__ void normalise(float (&x1)[8], float (&x2)[8], const float (&w1)[8], const float (&w2)[8],
                                          float eps, unsigned mask) {
  float q = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) q = fmaf(x1[e], x1[e], fmaf(x2[e], x2[e], q));
  q += __shfl_xor_sync(mask, q, 1);
  q += __shfl_xor_sync(mask, q, 2);
  q += __shfl_xor_sync(mask, q, 4);
  const float r = rsqrtf(fmaf(q, 1.0f / 128.0f, eps));
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x1[e] = x1[e] * r * w1[e];
    x2[e] = x2[e] * r * w2[e];
  }
}

// The rotation of rope_math.cuh (separately rounded products) on the lane's 8 pairs, as
// bf16 words in the order in which they are written.
__device__ __forceinline__ void rotate(const float (&x1)[8], const float (&x2)[8], const float (&cv)[8],
                                       const float (&sv)[8], bool sorted, uint32_t (&o)[8]) {
  float r1[8], r2[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    r1[e] = __fsub_rn(__fmul_rn(x1[e], cv[e]), __fmul_rn(x2[e], sv[e]));
    r2[e] = __fadd_rn(__fmul_rn(x2[e], cv[e]), __fmul_rn(x1[e], sv[e]));
  }
  if (sorted) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[7 - e] = ropemath::pack_rn(r1[e], r2[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = ropemath::pack_rn(r1[2 * e], r1[2 * e + 1]);
      o[4 + e] = ropemath::pack_rn(r2[2 * e], r2[2 * e + 1]);
    }
  }
}

// the lane's 32 bytes of a bf16 row: sorted pairs are level 7 - c, at `level` elements a
// level; rotate_half the two chunks of dims it came from
__device__ __forceinline__ void store_pairs(__nv_bfloat16* row, int c, bool sorted, long long level,
                                            const uint32_t (&o)[8]) {
  uint4* d0 = reinterpret_cast<uint4*>(sorted ? row + level * (7 - c) : row + 8 * c);
  uint4* d1 = sorted ? d0 + 1 : reinterpret_cast<uint4*>(row + 64 + 8 * c);
  *d0 = make_uint4(o[0], o[1], o[2], o[3]);
  *d1 = make_uint4(o[4], o[5], o[6], o[7]);
}

}  // namespace normmath
}  // namespace atf
