// Paged-KV append into an e4m3 cache with one scale per (page, kv head).
//
// A run is the new tokens of one request that fall into one page. Its scale is
// s = 2^e with the smallest e such that amax <= 448 * 2^e (amax over the run's
// rows of the head): with a power of two, x / s is exact and rounding to e4m3's
// 3 mantissa bits is the only error, and a row moved to a larger scale later
// loses bits only where it falls below e4m3's normal range. A run that begins
// inside a page keeps the page's scale unless its own amax needs a larger one.
//
// One warp owns a (run, kv head), K and V, so the scale's read, its update and
// the rows under it need no atomics and the result has one value. 8 lanes hold a
// row (16 elements each), so a warp reads 4 rows of 256 bytes at once and writes
// 16 bytes per lane. Runs of up to 16 rows stay in registers between the maximum
// and the rounding; longer ones (pages over 16) are read a second time, from L2.
//
// What bounds it: HBM for prompts (2 x 256 bytes read and 2 x 128 written per
// token and head); for one token per request the chain of dependent loads (token
// -> page list -> scale -> row). A CTA covers a window of tokens and hands its
// (run, head) pairs to 8 warps; the window shrinks with the token count so that a
// decode step's tokens spread over the SMs.
#include <cuda_fp16.h>

#include "atf_internal.h"
#include "rope_math.cuh"

namespace atf {
namespace append8 {

constexpr int WARPS = 8;
constexpr int THREADS = WARPS * 32;
constexpr int MAX_WINDOW = 32;
constexpr int REG_ROWS = 16;  // rows of a run kept in registers: 4 steps of 4

struct Args {
  const __nv_bfloat16* ak;
  const __nv_bfloat16* av;
  long long nnz, as_n, as_h;
  const int32_t* batch_indices;
  const int32_t* positions;
  uint8_t* kc;
  uint8_t* vc;
  long long num_pages, s_page, s_tok, s_head;
  int H, page_size, B, window;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  float* ks;
  float* vs;
  long long ss_page, ss_head;
  const float* cs;
  const float* sn;
  long long cs_stride, n_pos;
  const int64_t* rope_pos;
  int rope, sorted;
  int* err;
};

// exponent e of the smallest power of two with amax <= 448 * 2^e, in [-126, 120]:
// 448 = 1.75 * 2^8, so e = exponent(amax) - 8, one more where the mantissa is over 1.75
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = min(max(e, -126), 120);
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_to_f32(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// 16 elements of a row as 8 bf16x2 words
struct Words {
  uint32_t w[8];
};

__device__ __forceinline__ float abs_max(const Words& x, float m) {
  __nv_bfloat162 a = __float2bfloat162_rn(0.f);
#pragma unroll
  for (int i = 0; i < 8; ++i)  // a NaN loses against any number here
    a = __hmax2(a, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&x.w[i])));
  return fmaxf(m, fmaxf(__low2float(a), __high2float(a)));
}

// x / s and x * r truncated to 24 bits, with the last bit set where something was
// cut off ("round to odd"): rounding that to e4m3's 4 bits gives the same as
// rounding the exact value once, ties included
__device__ __forceinline__ float div_odd(float x, float s) {
  const float q = __fdiv_rz(x, s);
  return __fmaf_rn(-q, s, x) != 0.f ? __uint_as_float(__float_as_uint(q) | 1u) : q;
}
__device__ __forceinline__ float mul_odd(float x, float r) {
  const float q = __fmul_rz(x, r);
  return __fmaf_rn(x, r, -q) != 0.f ? __uint_as_float(__float_as_uint(q) | 1u) : q;
}

// the 16 elements under scale s: the product with 1/s is exact for a power of two
// (what this kernel writes); a scale set by another program is divided by
__device__ __forceinline__ void round_words(const Words& x, float s, uint32_t (&o)[4]) {
  const bool pow2 = (__float_as_uint(s) & 0x7fffffu) == 0;
  const float inv = __fdiv_rn(1.f, s);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f[2 * j] = ropemath::bf2f(x.w[2 * i + j] & 0xffffu);
      f[2 * j + 1] = __uint_as_float(x.w[2 * i + j] & 0xffff0000u);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = pow2 ? f[j] * inv : div_odd(f[j], s);
    o[i] = e4m3x2(f[0], f[1]) | (e4m3x2(f[2], f[3]) << 16);
  }
}

// this lane's 16 elements of a row: contiguous (16c..), or for RoPE the 8 pairs
// (8c.., 64 + 8c..) rotated, as the pairs' words in the order they are written
__device__ __forceinline__ Words load_plain(const __nv_bfloat16* row, int c) {
  Words x;
  const uint4 a = *reinterpret_cast<const uint4*>(row + 16 * c);
  const uint4 b = *reinterpret_cast<const uint4*>(row + 16 * c + 8);
  x.w[0] = a.x; x.w[1] = a.y; x.w[2] = a.z; x.w[3] = a.w;
  x.w[4] = b.x; x.w[5] = b.y; x.w[6] = b.z; x.w[7] = b.w;
  return x;
}
__device__ __forceinline__ Words load_rope(const Args& a, const __nv_bfloat16* row, long long i, int pos, int c) {
  long long rp = a.rope_pos != nullptr ? a.rope_pos[i] : pos;
  rp = rp < 0 ? 0 : (rp >= a.n_pos ? a.n_pos - 1 : rp);
  const float* cr = a.cs + rp * a.cs_stride;
  const float* sr = a.sn + rp * a.cs_stride;
  Words x;
  ropemath::rotate_chunk_sorted_words(row, cr, sr, c, x.w);
  if (!a.sorted) {
    // sorted word jl packs (x1, x2) of pair 8c + 7 - jl: back to the halves' order
    Words y;
#pragma unroll
    for (int i2 = 0; i2 < 4; ++i2) {
      const uint32_t p0 = x.w[7 - 2 * i2], p1 = x.w[6 - 2 * i2];
      y.w[i2] = (p0 & 0xffffu) | (p1 << 16);
      y.w[4 + i2] = (p0 >> 16) | (p1 & 0xffff0000u);
    }
    return y;
  }
  return x;
}

template <bool ROPE>
__device__ __forceinline__ Words load_k(const Args& a, const __nv_bfloat16* row, long long i, int pos, int c) {
  if constexpr (ROPE) return load_rope(a, row, i, pos, c);
  else return load_plain(row, c);
}
template <bool ROPE>
__device__ __forceinline__ void store_k(const Args& a, uint8_t* row, int c, const uint32_t (&o)[4]) {
  if (ROPE && !a.sorted) {
    *reinterpret_cast<uint2*>(row + 8 * c) = make_uint2(o[0], o[1]);
    *reinterpret_cast<uint2*>(row + 64 + 8 * c) = make_uint2(o[2], o[3]);
  } else {
    *reinterpret_cast<uint4*>(row + 16 * (ROPE ? 7 - c : c)) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// rows [0, n) of a page under the scale s_new instead of s_old; s_new is a power of
// two here (a scale only grows to one), so the ratio is exact
__device__ __forceinline__ void round_again(uint8_t* page_row0, long long s_tok, int n, float s_old, float s_new,
                                            int lane) {
  const float ratio = __fdiv_rn(s_old, s_new);
  for (int r = lane >> 3; r < n; r += 4) {
    uint4* at = reinterpret_cast<uint4*>(page_row0 + r * s_tok + 16 * (lane & 7));
    const uint4 v = *at;
    const uint32_t in[4] = {v.x, v.y, v.z, v.w};
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = e4m3x2_to_f32(in[i] & 0xffffu), b = e4m3x2_to_f32(in[i] >> 16);
      out[i] = e4m3x2(mul_odd(a.x, ratio), mul_odd(a.y, ratio)) | (e4m3x2(mul_odd(b.x, ratio), mul_odd(b.y, ratio)) << 16);
    }
    *at = make_uint4(out[0], out[1], out[2], out[3]);
  }
}

template <bool ROPE>
__global__ void __launch_bounds__(THREADS) append_e4m3_kernel(const Args a) {
  __shared__ int s_lead[MAX_WINDOW];
  __shared__ int s_n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long i0 = static_cast<long long>(blockIdx.x) * a.window;
  // the runs that begin in this window: a token begins one unless the token before
  // it is its predecessor in the same page
  if (warp == 0) {
    const long long i = i0 + lane;
    bool lead = false;
    if (lane < a.window && i < a.nnz) {
      const int b = a.batch_indices[i], pos = a.positions[i];
      lead = b >= 0;
      if (lead && i > 0 && pos > 0 && pos % a.page_size != 0)
        lead = !(a.batch_indices[i - 1] == b && a.positions[i - 1] == pos - 1);
    }
    const unsigned m = __ballot_sync(0xffffffffu, lead);
    if (lead) s_lead[__popc(m & ((1u << lane) - 1u))] = lane;
    if (lane == 0) s_n = __popc(m);
  }
  __syncthreads();
  const int tasks = s_n * a.H;
  for (int task = warp; task < tasks; task += WARPS) {
    const long long i = i0 + s_lead[task / a.H];
    const int h = task % a.H;
    const int b = a.batch_indices[i], pos = a.positions[i];
    bool bad = b >= a.B || pos < 0;
    long long page = -1;
    if (!bad) {
      const long long pidx = static_cast<long long>(a.kv_indptr[b]) + pos / a.page_size;
      bad = pidx >= a.kv_indptr[b + 1];
      if (!bad) {
        page = a.kv_indices[pidx];
        bad = page < 0 || page >= a.num_pages;
      }
    }
    if (bad) {  // the run is skipped
      if (a.err != nullptr && lane == 0) atomicCAS(a.err, 0, kDevErrIndex);
      continue;
    }
    const int slot = pos % a.page_size;
    // length of the run
    int n = 0;
    const int most = static_cast<int>(min(static_cast<long long>(a.page_size - slot), a.nnz - i));
    while (n < most) {
      const int j = n + lane;
      const bool in = j < most && a.batch_indices[i + j] == b && a.positions[i + j] == pos + j;
      const unsigned out = ~__ballot_sync(0xffffffffu, in);
      if (out != 0) {
        n += __ffs(out) - 1;
        break;
      }
      n += 32;
    }
    const long long src0 = i * a.as_n + static_cast<long long>(h) * a.as_h;
    const long long dst0 = page * a.s_page + static_cast<long long>(h) * a.s_head;
    const long long sc = page * a.ss_page + static_cast<long long>(h) * a.ss_head;
    const float ks_old = slot > 0 ? a.ks[sc] : 0.f, vs_old = slot > 0 ? a.vs[sc] : 0.f;
    const int c = lane & 7, r0 = lane >> 3;
    const bool in_regs = n <= REG_ROWS;
    Words kw[REG_ROWS / 4], vw[REG_ROWS / 4];
    float km = 0.f, vm = 0.f;
    for (int base = 0; base < n; base += REG_ROWS) {
#pragma unroll
      for (int u = 0; u < REG_ROWS / 4; ++u) {
        const int r = base + 4 * u + r0;
        if (r < n) {
          kw[u] = load_k<ROPE>(a, a.ak + src0 + r * a.as_n, i + r, pos + r, c);
          vw[u] = load_plain(a.av + src0 + r * a.as_n, c);
        }
      }
#pragma unroll
      for (int u = 0; u < REG_ROWS / 4; ++u)
        if (base + 4 * u + r0 < n) {
          km = abs_max(kw[u], km);
          vm = abs_max(vw[u], vm);
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      km = fmaxf(km, __shfl_xor_sync(0xffffffffu, km, off));
      vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, off));
    }
    const float ks_new = slot > 0 ? fmaxf(ks_old, scale_for(km)) : scale_for(km);
    const float vs_new = slot > 0 ? fmaxf(vs_old, scale_for(vm)) : scale_for(vm);
    if (slot > 0 && ks_new != ks_old) round_again(a.kc + dst0, a.s_tok, slot, ks_old, ks_new, lane);
    if (slot > 0 && vs_new != vs_old) round_again(a.vc + dst0, a.s_tok, slot, vs_old, vs_new, lane);
    for (int base = 0; base < n; base += REG_ROWS) {
#pragma unroll
      for (int u = 0; u < REG_ROWS / 4; ++u) {
        const int r = base + 4 * u + r0;
        if (r < n) {
          if (!in_regs) {
            kw[u] = load_k<ROPE>(a, a.ak + src0 + r * a.as_n, i + r, pos + r, c);
            vw[u] = load_plain(a.av + src0 + r * a.as_n, c);
          }
          const long long dst = dst0 + static_cast<long long>(slot + r) * a.s_tok;
          uint32_t o[4];
          round_words(kw[u], ks_new, o);
          store_k<ROPE>(a, a.kc + dst, c, o);
          round_words(vw[u], vs_new, o);
          *reinterpret_cast<uint4*>(a.vc + dst + 16 * c) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
    }
    if (lane == 0) {
      a.ks[sc] = ks_new;
      a.vs[sc] = vs_new;
    }
  }
}

}  // namespace append8
}  // namespace atf

using namespace atf;

extern "C" int atf_paged_kv_append_e4m3(const AtfAppendParams* p, const AtfKvScales* s, atf_stream_t stream) {
  if (p == nullptr || s == nullptr || p->append_k == nullptr || p->append_v == nullptr ||
      p->batch_indices == nullptr || p->positions == nullptr || p->k_cache == nullptr || p->v_cache == nullptr ||
      p->kv_indptr == nullptr || p->kv_indices == nullptr || s->k_scale == nullptr || s->v_scale == nullptr)
    return ATF_ERR_INVALID_ARG;
  if (p->head_dim != ATF_HEAD_DIM || p->k_level_major) return ATF_ERR_UNSUPPORTED;
  if (p->nnz < 0 || p->num_kv_heads < 1 || p->page_size < 1 || p->batch_size < 1 || p->num_pages < 1)
    return ATF_ERR_INVALID_ARG;
  const bool rope = p->cos != nullptr;
  if (rope != (p->sin != nullptr)) return ATF_ERR_INVALID_ARG;
  if (rope && (p->n_pos < 1 || p->cs_stride_pos < 64)) return ATF_ERR_INVALID_ARG;
  if (p->out_layout != ATF_LAYOUT_SORTED_PAIR && p->out_layout != ATF_LAYOUT_ROTATE_HALF)
    return ATF_ERR_INVALID_ARG;
  if (!aligned16(p->append_k) || !aligned16(p->append_v) || !aligned16(p->k_cache) || !aligned16(p->v_cache) ||
      (p->a_stride_n & 7) || (p->a_stride_h & 7) || (p->kv_stride_page & 15) || (p->kv_stride_token & 15) ||
      (p->kv_stride_head & 15))
    return ATF_ERR_ALIGNMENT;
  if (p->nnz == 0) return ATF_OK;
  int dev = 0;
  int rc = check_device(&dev);
  if (rc != ATF_OK) return rc;
  append8::Args a;
  a.ak = static_cast<const __nv_bfloat16*>(p->append_k);
  a.av = static_cast<const __nv_bfloat16*>(p->append_v);
  a.nnz = p->nnz;
  a.as_n = p->a_stride_n;
  a.as_h = p->a_stride_h;
  a.batch_indices = p->batch_indices;
  a.positions = p->positions;
  a.kc = static_cast<uint8_t*>(p->k_cache);
  a.vc = static_cast<uint8_t*>(p->v_cache);
  a.num_pages = p->num_pages;
  a.s_page = p->kv_stride_page;
  a.s_tok = p->kv_stride_token;
  a.s_head = p->kv_stride_head;
  a.H = p->num_kv_heads;
  a.page_size = p->page_size;
  a.B = p->batch_size;
  a.kv_indptr = p->kv_indptr;
  a.kv_indices = p->kv_indices;
  a.ks = s->k_scale;
  a.vs = s->v_scale;
  a.ss_page = s->stride_page;
  a.ss_head = s->stride_head;
  a.cs = p->cos;
  a.sn = p->sin;
  a.cs_stride = p->cs_stride_pos;
  a.n_pos = p->n_pos;
  a.rope_pos = p->rope_positions;
  a.rope = rope ? 1 : 0;
  a.sorted = p->out_layout == ATF_LAYOUT_SORTED_PAIR ? 1 : 0;
  a.err = p->error_flag;
  // tokens per CTA: about four CTAs per SM, between 1 and 32 tokens
  a.window = append8::MAX_WINDOW;
  while (a.window > 1 && (a.nnz + a.window - 1) / a.window < 4 * 148) a.window >>= 1;
  const long long blocks = (a.nnz + a.window - 1) / a.window;
  if (blocks > 0x7fffffffLL) return ATF_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (rope)
    append8::append_e4m3_kernel<true><<<static_cast<unsigned>(blocks), append8::THREADS, 0, st>>>(a);
  else
    append8::append_e4m3_kernel<false><<<static_cast<unsigned>(blocks), append8::THREADS, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? ATF_OK : ATF_ERR_CUDA;
}
