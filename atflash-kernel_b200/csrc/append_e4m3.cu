// Paged-KV append into an e4m3 cache with one scale per (page, kv head).
//
// A run is the new tokens of one request that fall into one page. Its scale is
// s = 2^e with the smallest e such that amax <= 448 * 2^e (amax over the run's
// rows of the head): with a power of two, x / s is exact and rounding to e4m3's
// 3 mantissa bits is the only error, and a row moved to a larger scale later
// loses bits only where it falls below e4m3's normal range. A run that begins
// inside a page keeps the page's scale unless its own amax needs a larger one.
//
// A task is (run, kv head, K or V). Up to 8 warps share a task, 16 rows each, so
// that runs of large pages are as parallel as those of small ones; they exchange
// their maxima through shared memory, and the scale's read, its update and the rows
// under it need no atomics: the result has one value. 8 lanes hold a row (16
// elements each), so a warp reads 4 rows of 256 bytes at once and writes 16 bytes
// per lane. Rows stay in registers between the maximum and the rounding (a run over
// 128 rows, in pages of 256, is read a second time, from L2).
//
// What bounds it: HBM for prompts (2 x 256 bytes read and 2 x 128 written per
// token and head); for one token per request the chain of dependent loads (token
// -> page list -> row). A CTA covers a window of tokens: its first warp finds the
// runs that begin there, their pages and lengths once, while the others fetch the
// tokens' rows of angles for all heads (RoPE); then all warps go through the tasks.
// The window shrinks with the token count so that a decode step's tokens spread over
// the SMs.
//
// Measured: 64K tokens x 8 heads in pages of 16 74 us (90% of HBM), with RoPE 98: no
// loads are in flight while rows are rotated and rounded (62% of HBM, 58% of the issue
// slots; 107 with the angles read from L2 for every head); 64 tokens
// x 8 heads 4.5 us. What cost most on the way: rows loaded one after another behind
// their bounds checks (170 us), and a division per element in the unrolled rounding
// (130). CTAs of 4 warps: 96-102 us, but 18-19 instead of 13 for pages of 64.
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "atf_internal.h"
#include "rope_math.cuh"

namespace atf {
namespace append8 {

constexpr int WARPS = 8;
constexpr int THREADS = WARPS * 32;
constexpr int MAX_WINDOW = 32;
constexpr int WARP_ROWS = 16;  // rows of a run that a warp keeps in registers: 4 steps of 4

struct Args {
  const __nv_bfloat16* ak;
  const __nv_bfloat16* av;
  long long nnz, as_n, as_h;
  const int32_t* batch_indices;
  const int32_t* positions;
  uint8_t* kc;
  uint8_t* vc;
  long long num_pages, s_page, s_tok, s_head;
  int H, page_size, B, window, share, heads;  // share: warps of a task (1, 2, 4 or 8)
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  float* ks;
  float* vs;
  long long ss_page, ss_head;
  const float* cs;
  const float* sn;
  long long cs_stride, n_pos;
  const int64_t* rope_pos;
  int sorted;
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

// the 16 elements under a scale that is no such power of two (another program's), divided
// by it; out of line, since this kernel writes powers of two only
__device__ __noinline__ uint4 divide_words(uint4 lo, uint4 hi, float s) {
  const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  uint32_t o[4];
  for (int i = 0; i < 4; ++i) {
    float f[4];
    for (int j = 0; j < 2; ++j) {
      f[2 * j] = div_odd(ropemath::bf2f(w[2 * i + j] & 0xffffu), s);
      f[2 * j + 1] = div_odd(__uint_as_float(w[2 * i + j] & 0xffff0000u), s);
    }
    o[i] = e4m3x2(f[0], f[1]) | (e4m3x2(f[2], f[3]) << 16);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
// the 16 elements under scale s: for a power of two up to 2^126 the product with 1/s is
// exact (the inverse of 2^127 is no normal number)
__device__ __forceinline__ void round_words(const Words& x, float s, uint32_t (&o)[4]) {
  if ((__float_as_uint(s) & 0x7fffffu) != 0 || __float_as_uint(s) >= 0x7f000000u) {
    const uint4 v = divide_words(make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]),
                                 make_uint4(x.w[4], x.w[5], x.w[6], x.w[7]), s);
    o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
    return;
  }
  const float inv = __uint_as_float(0x7f000000u - __float_as_uint(s));  // 2^-e of 2^e, |e| <= 126
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f[2 * j] = __uint_as_float(x.w[2 * i + j] << 16) * inv;
      f[2 * j + 1] = __uint_as_float(x.w[2 * i + j] & 0xffff0000u) * inv;
    }
    o[i] = e4m3x2(f[0], f[1]) | (e4m3x2(f[2], f[3]) << 16);
  }
}

// this lane's 16 elements of a row: contiguous (16c..), or for RoPE the 8 pairs
// (8c.., 64 + 8c..)
__device__ __forceinline__ Words load_row(const __nv_bfloat16* row, int c, bool pairs) {
  Words x;
  const uint4 a = *reinterpret_cast<const uint4*>(row + (pairs ? 8 * c : 16 * c));
  const uint4 b = *reinterpret_cast<const uint4*>(row + (pairs ? 64 + 8 * c : 16 * c + 8));
  x.w[0] = a.x; x.w[1] = a.y; x.w[2] = a.z; x.w[3] = a.w;
  x.w[4] = b.x; x.w[5] = b.y; x.w[6] = b.z; x.w[7] = b.w;
  return x;
}
// the 8 pairs rotated as in rope_math.cuh (separately rounded products, then bf16),
// as words in the order they are written; row(f): the position's table rows, cos in
// the 16-byte words 0 .. 15 and sin in 16 .. 31
template <typename Row>
__device__ __forceinline__ Words rotate(const Words& in, Row row, int c, bool sorted) {
  float cv[8], sv[8];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const float4 c4 = row(2 * c + q);
    const float4 s4 = row(16 + 2 * c + q);
    cv[4 * q] = c4.x; cv[4 * q + 1] = c4.y; cv[4 * q + 2] = c4.z; cv[4 * q + 3] = c4.w;
    sv[4 * q] = s4.x; sv[4 * q + 1] = s4.y; sv[4 * q + 2] = s4.z; sv[4 * q + 3] = s4.w;
  }
  float r1[8], r2[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t l2 = in.w[e >> 1], h2 = in.w[4 + (e >> 1)];
    const float x1 = (e & 1) ? __uint_as_float(l2 & 0xffff0000u) : __uint_as_float(l2 << 16);
    const float x2 = (e & 1) ? __uint_as_float(h2 & 0xffff0000u) : __uint_as_float(h2 << 16);
    r1[e] = __fsub_rn(__fmul_rn(x1, cv[e]), __fmul_rn(x2, sv[e]));
    r2[e] = __fadd_rn(__fmul_rn(x2, cv[e]), __fmul_rn(x1, sv[e]));
  }
  Words x;
  if (sorted) {  // pairs in falling order, (x1, x2) adjacent
#pragma unroll
    for (int e = 0; e < 8; ++e) x.w[7 - e] = ropemath::pack_rn(r1[e], r2[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x.w[e] = ropemath::pack_rn(r1[2 * e], r1[2 * e + 1]);
      x.w[4 + e] = ropemath::pack_rn(r2[2 * e], r2[2 * e + 1]);
    }
  }
  return x;
}

// rows [0, n) of a page under the scale s_new instead of s_old; s_new is a power of
// two here (a scale only grows to one), so the ratio is exact
__device__ __forceinline__ void round_again(uint8_t* page_row0, long long s_tok, int first, int step, int n,
                                            float s_old, float s_new, int c) {
  const float ratio = __fdiv_rn(s_old, s_new);
  for (int r = first; r < n; r += step) {
    uint4* at = reinterpret_cast<uint4*>(page_row0 + r * s_tok + 16 * c);
    const uint4 v = *at;
    const uint32_t in[4] = {v.x, v.y, v.z, v.w};
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = e4m3x2_to_f32(in[i] & 0xffffu), b = e4m3x2_to_f32(in[i] >> 16);
      out[i] = e4m3x2(mul_odd(a.x, ratio), mul_odd(a.y, ratio)) |
               (e4m3x2(mul_odd(b.x, ratio), mul_odd(b.y, ratio)) << 16);
    }
    *at = make_uint4(out[0], out[1], out[2], out[3]);
  }
}

// A run: the tokens i .. i + n - 1 of the window, from slot `slot` of page `page` on
struct Run {
  long long page;
  int i, n, slot, pos;
};

// The runs that begin in the CTA's window of tokens, by its first warp. A token
// begins one unless the token before it is its predecessor in the same page; a run
// ends before the next one, a padding token or the page's end. Runs with a page
// that is not the request's or the cache's are reported and left out.
__device__ __forceinline__ int find_runs(const Args& a, long long i0, Run* runs, int lane) {
  const long long i = i0 + lane;
  const bool in = lane < a.window && i < a.nnz;
  int b = -1, pos = 0;
  if (in) {
    b = a.batch_indices[i];
    pos = a.positions[i];
  }
  bool lead = in && b >= 0;
  if (lead && i > 0 && pos > 0 && pos % a.page_size != 0)
    lead = !(a.batch_indices[i - 1] == b && a.positions[i - 1] == pos - 1);
  const unsigned leads = __ballot_sync(0xffffffffu, lead);
  const unsigned stops = __ballot_sync(0xffffffffu, lead || (in && b < 0));
  bool good = lead && b < a.B && pos >= 0;
  long long page = -1;
  if (good) {
    const long long pidx = static_cast<long long>(a.kv_indptr[b]) + pos / a.page_size;
    good = pidx < a.kv_indptr[b + 1];
    if (good) {
      page = a.kv_indices[pidx];
      good = page >= 0 && page < a.num_pages;
    }
  }
  if (lead && !good && a.err != nullptr) atomicCAS(a.err, 0, kDevErrIndex);
  const int tokens = static_cast<int>(min(static_cast<long long>(a.window), a.nnz - i0));
  // inside the window a run ends at the next stop
  const unsigned later = lane < 31 ? stops >> (lane + 1) : 0u;
  int n = later != 0 ? __ffs(later) : tokens - lane;
  // the last run may go on past the window
  const unsigned open = __ballot_sync(0xffffffffu, lead && later == 0);
  if (open != 0) {
    const int l = __ffs(open) - 1;
    const int ob = __shfl_sync(0xffffffffu, b, l), opos = __shfl_sync(0xffffffffu, pos, l);
    const int most = a.page_size - (opos >= 0 ? opos % a.page_size : 0);
    int on = tokens - l;
    while (on < most) {
      const long long j = i0 + l + on + lane;
      const bool same = on + lane < most && j < a.nnz && a.batch_indices[j] == ob && a.positions[j] == opos + on + lane;
      const unsigned out = ~__ballot_sync(0xffffffffu, same);
      if (out != 0) {
        on += __ffs(out) - 1;
        break;
      }
      on += 32;
    }
    if (lane == l) n = on;
  }
  const unsigned goods = __ballot_sync(0xffffffffu, good);
  if (good) {
    Run r;
    r.page = page;
    r.i = lane;
    r.slot = pos % a.page_size;
    r.n = min(n, a.page_size - r.slot);
    r.pos = pos;
    runs[__popc(goods & ((1u << lane) - 1u))] = r;
  }
  return __popc(goods);
}

// position of a token in the tables, inside them
__device__ __forceinline__ long long angle_row(const Args& a, long long i) {
  const long long rp = a.rope_pos != nullptr ? a.rope_pos[i] : a.positions[i];
  return rp < 0 ? 0 : (rp >= a.n_pos ? a.n_pos - 1 : rp);
}
// word f of a staged row: even words of the two halves of cos (or sin) would share
// banks, so the second half's are swapped with their neighbours
__device__ __forceinline__ int angle_slot(int f) { return f ^ ((f >> 3) & 1); }

// The angles of the window's tokens, read once for all heads, by the warps that
// wait for find_runs meanwhile
__device__ __forceinline__ void stage_angles(const Args& a, long long i0, float4 (*rows)[32], int warp, int lane) {
  const int tokens = static_cast<int>(min(static_cast<long long>(a.window), a.nnz - i0));
  // lane k holds the row of this warp's k-th token
  const int mine = (warp - 1) + lane * (WARPS - 1);
  const long long rp = mine < tokens ? angle_row(a, i0 + mine) : 0;
  for (int k = 0, t = warp - 1; t < tokens; ++k, t += WARPS - 1) {
    const long long at = __shfl_sync(0xffffffffu, rp, k) * a.cs_stride + 4 * (lane & 15);
    const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(&rows[t][angle_slot(lane)]));
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"((lane < 16 ? a.cs : a.sn) + at) : "memory");
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <bool ROPE>
__global__ void __launch_bounds__(THREADS, 3) append_e4m3_kernel(const Args a) {
  __shared__ Run s_run[MAX_WINDOW];
  __shared__ int s_n;
  __shared__ float s_max[2][WARPS];
  __shared__ __align__(16) float4 s_angle[ROPE ? MAX_WINDOW : 1][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long i0 = static_cast<long long>(blockIdx.x) * a.window;
  if (warp == 0) {
    const int n = find_runs(a, i0, s_run, lane);
    if (lane == 0) s_n = n;
  } else if (ROPE) {
    stage_angles(a, i0, s_angle, warp, lane);
  }
  __syncthreads();
  // this CTA's heads: a block's y takes `heads` of them
  const int h0 = static_cast<int>(blockIdx.y) * a.heads, nh = min(a.heads, a.H - h0);
  const int tasks = s_n * nh * 2;
  const int W = a.share, wi = warp & (W - 1), slots = WARPS / W;
  const int c = lane & 7, r0 = wi * WARP_ROWS + (lane >> 3), step = W * WARP_ROWS;
  int turn = 0;
  for (int base = 0; base < tasks; base += slots, turn ^= 1) {
    const int task = base + warp / W;
    const bool live = task < tasks;
    // K and V of a (run, head) are neighbouring tasks; idle warps repeat the last
    const int t = live ? task : tasks - 1;
    const bool is_v = t & 1;
    const int h = h0 + (t >> 1) % nh;
    const Run run = s_run[(t >> 1) / nh];
    const int n = live ? run.n : 0;
    const __nv_bfloat16* src = (is_v ? a.av : a.ak) + (i0 + run.i) * a.as_n + static_cast<long long>(h) * a.as_h;
    uint8_t* page0 = (is_v ? a.vc : a.kc) + run.page * a.s_page + static_cast<long long>(h) * a.s_head;
    float* scale = (is_v ? a.vs : a.ks) + run.page * a.ss_page + static_cast<long long>(h) * a.ss_head;
    const bool rot = ROPE && !is_v;
    const float s_old = run.slot > 0 && live ? *scale : 0.f;
    Words w[WARP_ROWS / 4];
    // Rows b0 + r0 + 4 u: all loads are issued before the first is used, without a
    // branch between them; rows past the run's end read its last row again, which
    // changes no maximum, and are not written.
    auto load = [&](int b0, auto steps) {
      constexpr int U = decltype(steps)::value;
      int r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        r[u] = min(b0 + r0 + 4 * u, n - 1);
        w[u] = load_row(src + r[u] * a.as_n, c, rot);
      }
      if (rot) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int t = run.i + r[u];
          if (t < a.window) {
            w[u] = rotate(w[u], [&](int f) { return s_angle[t][angle_slot(f)]; }, c, a.sorted != 0);
          } else {  // the run goes on past the window
            const long long at = angle_row(a, i0 + t) * a.cs_stride;
            w[u] = rotate(w[u], [&](int f) {
              return *reinterpret_cast<const float4*>((f < 16 ? a.cs : a.sn) + at + 4 * (f & 15));
            }, c, a.sorted != 0);
          }
        }
      }
    };
    const std::integral_constant<int, 1> one{};
    const std::integral_constant<int, WARP_ROWS / 4> all{};
    const bool few = n <= 4 && W == 1;  // a step of a decode: one row of the four
    float m = 0.f;
    if (few) {
      if (n > 0) {
        load(0, one);
        m = abs_max(w[0], m);
      }
    } else {
      for (int b0 = 0; b0 < n; b0 += step) {
        load(b0, all);
#pragma unroll
        for (int u = 0; u < WARP_ROWS / 4; ++u) m = abs_max(w[u], m);
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    if (W > 1) {
      if (lane == 0) s_max[turn][warp] = m;
      __syncthreads();  // also: every warp of the task has read the old scale
      for (int k = 0; k < W; ++k) m = fmaxf(m, s_max[turn][(warp & ~(W - 1)) + k]);
    }
    const float s_new = run.slot > 0 ? fmaxf(s_old, scale_for(m)) : scale_for(m);
    if (!live) continue;
    if (run.slot > 0 && s_new != s_old)
      round_again(page0, a.s_tok, wi * 4 + (lane >> 3), 4 * W, run.slot, s_old, s_new, c);
    auto store = [&](int b0, auto steps) {
      constexpr int U = decltype(steps)::value;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = b0 + r0 + 4 * u;
        uint32_t o[4];
        round_words(w[u], s_new, o);
        if (r < n) {
          uint8_t* dst = page0 + static_cast<long long>(run.slot + r) * a.s_tok;
          if (rot && !a.sorted) {
            *reinterpret_cast<uint2*>(dst + 8 * c) = make_uint2(o[0], o[1]);
            *reinterpret_cast<uint2*>(dst + 64 + 8 * c) = make_uint2(o[2], o[3]);
          } else {
            *reinterpret_cast<uint4*>(dst + 16 * (rot ? 7 - c : c)) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
      }
    };
    if (few) {
      store(0, one);
    } else {
      for (int b0 = 0; b0 < n; b0 += step) {
        if (n > step) load(b0, all);
        store(b0, all);
      }
    }
    if (lane == 0 && wi == 0) *scale = s_new;
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
  if (p->head_dim != ATF_HEAD_DIM || p->k_level_major || p->num_kv_heads > 65535) return ATF_ERR_UNSUPPORTED;
  if (p->nnz < 0 || p->num_kv_heads < 1 || p->page_size < 1 || p->batch_size < 1 || p->num_pages < 1)
    return ATF_ERR_INVALID_ARG;
  const bool rope = p->cos != nullptr;
  if (rope != (p->sin != nullptr)) return ATF_ERR_INVALID_ARG;
  if (rope && (p->n_pos < 1 || p->cs_stride_pos < 64)) return ATF_ERR_INVALID_ARG;
  if (p->out_layout != ATF_LAYOUT_SORTED_PAIR && p->out_layout != ATF_LAYOUT_ROTATE_HALF)
    return ATF_ERR_INVALID_ARG;
  if (rope && (!aligned16(p->cos) || !aligned16(p->sin) || (p->cs_stride_pos & 3))) return ATF_ERR_ALIGNMENT;
  if (!aligned16(p->append_k) || !aligned16(p->append_v) || !aligned16(p->k_cache) || !aligned16(p->v_cache) ||
      (p->a_stride_n & 7) || (p->a_stride_h & 7) || (p->kv_stride_page & 15) || (p->kv_stride_token & 15) ||
      (p->kv_stride_head & 15))
    return ATF_ERR_ALIGNMENT;
  // pages and scales are written: one element that stands for several (a broadcast
  // axis) would take whichever task came last
  if ((p->num_pages > 1 && (s->stride_page == 0 || p->kv_stride_page == 0)) ||
      (p->num_kv_heads > 1 && (s->stride_head == 0 || p->kv_stride_head == 0)) ||
      (p->page_size > 1 && p->kv_stride_token == 0))
    return ATF_ERR_INVALID_ARG;
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
  a.sorted = p->out_layout == ATF_LAYOUT_SORTED_PAIR ? 1 : 0;
  a.err = p->error_flag;
  // warps per task: a page's rows, 16 each
  a.share = 1;
  while (a.share < append8::WARPS && a.share * append8::WARP_ROWS < a.page_size) a.share <<= 1;
  // tokens per CTA: the most, up to 32, that give every SM a CTA
  a.window = append8::MAX_WINDOW;
  while (a.window > 1 && (a.nnz + a.window - 1) / a.window < 148) a.window >>= 1;
  const long long blocks = (a.nnz + a.window - 1) / a.window;
  if (blocks > 0x7fffffffLL) return ATF_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // Few CTAs that begin a run (pages longer than the window: not all do) with more
  // tasks than warps: the heads go to several (13 prompts in pages of 64, 4 heads:
  // 13.4 us undivided, 10.0 divided; dividing further, or more CTAs than this, gave
  // nothing or cost 1.8 us at pages of 16)
  const long long runs = a.window / p->page_size + 1;  // that a window may begin, for one request
  const long long at_once = append8::WARPS / a.share;
  int split = 1;
  const long long busy = (blocks * std::min(a.window, p->page_size) + p->page_size - 1) / p->page_size;
  while (split < a.H && busy * split < 2 * 148 && runs * ((a.H + split - 1) / split) * 2 > at_once) split <<= 1;
  a.heads = (a.H + split - 1) / split;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((a.H + a.heads - 1) / a.heads));
  if (rope)
    append8::append_e4m3_kernel<true><<<grid, append8::THREADS, 0, st>>>(a);
  else
    append8::append_e4m3_kernel<false><<<grid, append8::THREADS, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? ATF_OK : ATF_ERR_CUDA;
}
