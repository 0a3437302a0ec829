// Paged-KV append into an e4m3 cache with one scale per (page, kv head).
//
// A run is the new tokens of one request that fall into one page. Its scale is
// s = 2^e with the smallest e such that amax <= 448 * 2^e (amax over the run's
// rows of the head): with a power of two, x / s is exact and rounding to e4m3's
// 3 mantissa bits is the only error, and a row moved to a larger scale later
// loses bits only where it falls below e4m3's normal range. A run that begins
// inside a page keeps the page's scale unless its own amax needs a larger one.
//
// A task is (run, kv head, K or V). What works on it goes by the run's length: one row 8
// lanes, up to 16 rows a warp, more rows up to 8 warps, 16 rows each, so that runs of
// large pages are as parallel as those of small ones; these exchange their maxima through
// shared memory. The scale's read, its update and the rows under it need no atomics: the
// result has one value. 8 lanes hold a row (16 elements each), so a warp reads 4 rows of
// 256 bytes at once and writes 16 bytes per lane. Rows stay in registers between the
// maximum and the rounding (a run over 128 rows, in pages of 256, is read a second time,
// from L2).
//
// What bounds it: HBM for prompts (2 x 256 bytes read and 2 x 128 written per
// token and head); for one token per request the chain of dependent loads (token
// -> page list -> row). A CTA covers a window of tokens: its first warp finds the
// runs that begin there, their pages and lengths once, while the others fetch the
// tokens' rows of angles for all heads (RoPE); then all warps go through the tasks. (A CTA
// where no run begins, as every second one for pages of 64, ends after its first loads.)
// The window shrinks with the token count so that a decode step's tokens spread over
// the SMs.
//
// Measured: 64K tokens x 8 heads in pages of 16 74 us (90% of HBM), with RoPE 98: no
// loads are in flight while rows are rotated and rounded (62% of HBM, 58% of the issue
// slots; 107 with the angles read from L2 for every head); 64 tokens
// x 8 heads 4.5 us. What cost most on the way: rows loaded one after another behind
// their bounds checks (170 us), and a division per element in the unrolled rounding
// (130). CTAs of 4 warps: 96-102 us, but 18-19 instead of 13 for pages of 64. From cold
// memory, with as many warps to every run as the page has rows and with them by the run:
// 512 single tokens x 8 heads in pages of 64 51 and 10 us (pages of 16: 16.4 and 10), 200
// single tokens beside 2 prompts of 3000 x 4 heads 107 and 21. Prompts alone pay for that where a
// CTA has little to do (64K tokens x 8 heads with RoPE in pages of 64 145 and 149, 63486 x 1 head
// in pages of 32, replayed from a graph, 18 and 20) and gain 4 to 6% in pages of 128 and 256.
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "atf_internal.h"
#include "norm_math.cuh"
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
  int H, page_size, B, window, heads;
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
  const void* norm_w;
  int norm_f32;
  float eps;
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
// the 16-byte words 0 .. 15 and sin in 16 .. 31. With a norm, the pairs are normed first
// over the 8 lanes of the row, under weights w1 and w2.
template <bool NORM, typename Row>
__device__ __forceinline__ Words rotate(const Words& in, Row row, int c, bool sorted, const float (&w1)[NORM ? 8 : 1],
                                        const float (&w2)[NORM ? 8 : 1], float eps) {
  float cv[8], sv[8];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const float4 c4 = row(2 * c + q);
    const float4 s4 = row(16 + 2 * c + q);
    cv[4 * q] = c4.x; cv[4 * q + 1] = c4.y; cv[4 * q + 2] = c4.z; cv[4 * q + 3] = c4.w;
    sv[4 * q] = s4.x; sv[4 * q + 1] = s4.y; sv[4 * q + 2] = s4.z; sv[4 * q + 3] = s4.w;
  }
  float x1[8], x2[8];
  normmath::unpack(make_uint4(in.w[0], in.w[1], in.w[2], in.w[3]), x1);
  normmath::unpack(make_uint4(in.w[4], in.w[5], in.w[6], in.w[7]), x2);
  if constexpr (NORM) normmath::normalise(x1, x2, w1, w2, eps, 0xffu << (threadIdx.x & 24));
  Words x;
  normmath::rotate(x1, x2, cv, sv, sorted, x.w);
  return x;
}

// rows [0, n) of a page under the scale s_new instead of s_old, U of a lane's in flight;
// s_new is a power of two here (a scale only grows to one), so the ratio is exact
template <int U>
__device__ __forceinline__ void round_again(uint8_t* page_row0, long long s_tok, int first, int step, int n,
                                            float s_old, float s_new, int c) {
  const float ratio = __fdiv_rn(s_old, s_new);
  for (int r0 = first; r0 < n; r0 += U * step) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = *reinterpret_cast<const uint4*>(page_row0 + min(r0 + u * step, n - 1) * s_tok + 16 * c);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * step;
      if (r >= n) break;
      const uint32_t in[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
      uint32_t out[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = e4m3x2_to_f32(in[i] & 0xffffu), b = e4m3x2_to_f32(in[i] >> 16);
        out[i] = e4m3x2(mul_odd(a.x, ratio), mul_odd(a.y, ratio)) |
                 (e4m3x2(mul_odd(b.x, ratio), mul_odd(b.y, ratio)) << 16);
      }
      *reinterpret_cast<uint4*>(page_row0 + r * s_tok + 16 * c) = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
}

// A run: the tokens i .. i + n - 1 of the window, from slot `slot` of page `page` on
struct Run {
  long long page;
  int i, n, slot;
};

// A lane's token of the window, and the window's lanes where a run begins. A token
// begins one unless the token before it is its predecessor in the same page.
struct Tokens {
  int b, pos;
  bool lead;
  unsigned leads, stops;
};
__device__ __forceinline__ Tokens read_tokens(const Args& a, long long i0, int lane) {
  const long long i = i0 + lane;
  const bool in = lane < a.window && i < a.nnz;
  Tokens t = {-1, 0, false, 0u, 0u};
  if (in) {
    t.b = a.batch_indices[i];
    t.pos = a.positions[i];
  }
  int first_b = -1, first_pos = -1;  // of the token before the window
  if (lane == 0 && i0 > 0) {
    first_b = a.batch_indices[i0 - 1];
    first_pos = a.positions[i0 - 1];
  }
  int before_b = __shfl_up_sync(0xffffffffu, t.b, 1), before_pos = __shfl_up_sync(0xffffffffu, t.pos, 1);
  if (lane == 0) {
    before_b = first_b;
    before_pos = first_pos;
  }
  t.lead = in && t.b >= 0;
  if (t.lead && i > 0 && t.pos > 0 && t.pos % a.page_size != 0) t.lead = !(before_b == t.b && before_pos == t.pos - 1);
  t.leads = __ballot_sync(0xffffffffu, t.lead);
  t.stops = __ballot_sync(0xffffffffu, t.lead || (in && t.b < 0));
  return t;
}

// What a CTA goes through: runs of one row [0, single), of up to 16 [single, few), of
// more [few, all), with `share` warps to a task of these
struct Work {
  int single, few, all, share;
};

// The runs that begin in the CTA's window of tokens, by its first warp. A run ends
// before the next one, a padding token or the page's end. Runs with a page that is not
// the request's or the cache's are reported and left out.
__device__ __forceinline__ Work find_runs(const Args& a, long long i0, const Tokens& t, Run* runs, int lane) {
  const int tokens = static_cast<int>(min(static_cast<long long>(a.window), a.nnz - i0));
  // inside the window a run ends at the next stop
  const unsigned later = lane < 31 ? t.stops >> (lane + 1) : 0u;
  int n = later != 0 ? __ffs(later) : tokens - lane;
  // the last run may go on past the window: the first tokens that it may have there are
  // read side by side with the page list's bounds
  const unsigned open = __ballot_sync(0xffffffffu, t.lead && later == 0);
  const int l = open != 0 ? __ffs(open) - 1 : 0;
  const int ob = __shfl_sync(0xffffffffu, t.b, l), opos = __shfl_sync(0xffffffffu, t.pos, l);
  const int most = open != 0 ? a.page_size - (opos >= 0 ? opos % a.page_size : 0) : 0;
  int on = tokens - l;
  int next_b = -1, next_pos = 0;
  auto read_next = [&]() {
    const long long j = i0 + l + on + lane;
    next_b = -1;
    if (on + lane < most && j < a.nnz) {
      next_b = a.batch_indices[j];
      next_pos = a.positions[j];
    }
  };
  read_next();
  bool good = t.lead && t.b < a.B && t.pos >= 0;
  int list0 = 0, list1 = 0;
  if (good) {
    list0 = a.kv_indptr[t.b];
    list1 = a.kv_indptr[t.b + 1];
  }
  const long long pidx = static_cast<long long>(list0) + (t.pos >= 0 ? t.pos : 0) / a.page_size;
  good = good && pidx < list1;
  const long long page = good ? a.kv_indices[pidx] : -1;
  while (on < most) {
    const unsigned out = ~__ballot_sync(0xffffffffu, next_b == ob && next_pos == opos + on + lane);
    if (out != 0) {
      on += __ffs(out) - 1;
      break;
    }
    on += 32;
    read_next();
  }
  if (open != 0 && lane == l) n = on;
  good = good && page >= 0 && page < a.num_pages;
  if (t.lead && !good && a.err != nullptr) atomicCAS(a.err, 0, kDevErrIndex);
  n = good ? min(n, a.page_size - t.pos % a.page_size) : 0;
  const int longest = __reduce_max_sync(0xffffffffu, n);
  const unsigned one = __ballot_sync(0xffffffffu, n == 1), more = __ballot_sync(0xffffffffu, n > WARP_ROWS);
  const unsigned some = __ballot_sync(0xffffffffu, n > 1 && n <= WARP_ROWS);
  Work work;
  work.single = __popc(one);
  work.few = work.single + __popc(some);
  work.all = work.few + __popc(more);
  work.share = longest > 4 * WARP_ROWS ? 8 : longest > 2 * WARP_ROWS ? 4 : 2;
  if (good) {
    Run r;
    r.page = page;
    r.i = lane;
    r.slot = t.pos % a.page_size;
    r.n = n;
    const unsigned before = (1u << lane) - 1u;
    const int at = n == 1 ? __popc(one & before)
                          : n <= WARP_ROWS ? work.single + __popc(some & before) : work.few + __popc(more & before);
    runs[at] = r;
  }
  return work;
}

// position of a token in the tables, inside them
__device__ __forceinline__ long long inside(const Args& a, long long rp) {
  return rp < 0 ? 0 : (rp >= a.n_pos ? a.n_pos - 1 : rp);
}
__device__ __forceinline__ long long angle_row(const Args& a, long long i) {
  return inside(a, a.rope_pos != nullptr ? a.rope_pos[i] : a.positions[i]);
}
// word f of a staged row: even words of the two halves of cos (or sin) would share
// banks, so the second half's are swapped with their neighbours
__device__ __forceinline__ int angle_slot(int f) { return f ^ ((f >> 3) & 1); }

// The angles of the window's tokens, read once for all heads, by the warps that
// wait for find_runs meanwhile
__device__ __forceinline__ void stage_angles(const Args& a, long long i0, int pos, float4 (*rows)[32], int warp,
                                             int lane) {
  const int tokens = static_cast<int>(min(static_cast<long long>(a.window), a.nnz - i0));
  // lane k holds the row of this warp's k-th token
  const int mine = (warp - 1) + lane * (WARPS - 1);
  const int mine_pos = __shfl_sync(0xffffffffu, pos, mine & 31);
  const long long rp = mine < tokens ? inside(a, a.rope_pos != nullptr ? a.rope_pos[i0 + mine] : mine_pos) : 0;
  for (int k = 0, t = warp - 1; t < tokens; ++k, t += WARPS - 1) {
    const long long at = __shfl_sync(0xffffffffu, rp, k) * a.cs_stride + 4 * (lane & 15);
    const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(&rows[t][angle_slot(lane)]));
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"((lane < 16 ? a.cs : a.sn) + at) : "memory");
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// The norm's weights stay in registers, with two CTAs an SM instead of three: 64K tokens x 8
// heads in pages of 16 125 us (98 with the rotation alone; in pages of 64 165 and 141); from
// shared memory 135, and 157 with three CTAs (spills).
template <bool ROPE, bool NORM>
__global__ void __launch_bounds__(THREADS, NORM ? 2 : 3) append_e4m3_kernel(const Args a) {
  __shared__ Run s_run[MAX_WINDOW];
  __shared__ Work s_work;
  __shared__ float s_max[2][WARPS];
  __shared__ __align__(16) float4 s_angle[ROPE ? MAX_WINDOW : 1][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long i0 = static_cast<long long>(blockIdx.x) * a.window;
  const int c = lane & 7;
  float w1[NORM ? 8 : 1] = {}, w2[NORM ? 8 : 1] = {};  // of this lane's pairs
  const Tokens tokens = read_tokens(a, i0, lane);  // by every warp, alike
  if (tokens.leads == 0) return;
  if constexpr (NORM) {
    normmath::weights8(a.norm_w, a.norm_f32 != 0, 8 * c, w1);
    normmath::weights8(a.norm_w, a.norm_f32 != 0, 64 + 8 * c, w2);
  }
  if (warp == 0) {
    const Work work = find_runs(a, i0, tokens, s_run, lane);
    if (lane == 0) s_work = work;
  } else if (ROPE) {
    stage_angles(a, i0, tokens.pos, s_angle, warp, lane);
  }
  __syncthreads();
  // this CTA's heads: a block's y takes `heads` of them
  const int h0 = static_cast<int>(blockIdx.y) * a.heads, nh = min(a.heads, a.H - h0);
  // Runs of several rows: a warp each up to 16 rows, then those that warps share
  int turn = 0;
  for (int part = 0; part < 2; ++part) {
    const int q0 = part == 0 ? s_work.single : s_work.few;
    const int tasks = ((part == 0 ? s_work.few : s_work.all) - q0) * nh * 2;
    const int W = part == 0 ? 1 : s_work.share, wi = warp & (W - 1), slots = WARPS / W;
    const int r0 = wi * WARP_ROWS + (lane >> 3), step = W * WARP_ROWS;
    for (int base = 0; base < tasks; base += slots, turn ^= 1) {
      const int task = base + warp / W;
      const bool live = task < tasks;
      // K and V of a (run, head) are neighbouring tasks; idle warps repeat the last
      const int t = live ? task : tasks - 1;
      const bool is_v = t & 1;
      const int h = h0 + (t >> 1) % nh;
      const Run run = s_run[q0 + (t >> 1) / nh];
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
              w[u] = rotate<NORM>(w[u], [&](int f) { return s_angle[t][angle_slot(f)]; }, c, a.sorted != 0, w1, w2, a.eps);
            } else {  // the run goes on past the window
              const long long at = angle_row(a, i0 + t) * a.cs_stride;
              w[u] = rotate<NORM>(w[u], [&](int f) {
                return *reinterpret_cast<const float4*>((f < 16 ? a.cs : a.sn) + at + 4 * (f & 15));
              }, c, a.sorted != 0, w1, w2, a.eps);
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
      if (run.slot > 0 && s_new != s_old) {
        if (few)
          round_again<4>(page0, a.s_tok, lane >> 3, 4, run.slot, s_old, s_new, c);
        else
          round_again<1>(page0, a.s_tok, wi * 4 + (lane >> 3), 4 * W, run.slot, s_old, s_new, c);
      }
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
  // Single rows: 8 lanes each, first those of K, then those of V. (With these first the
  // registers of the part above are spilled: 64K tokens with RoPE 115 us instead of 105.)
  const int n1 = s_work.single * nh;
  for (int base = 4 * warp; base < 2 * n1; base += 4 * WARPS) {
    const int task = base + (lane >> 3);
    const bool live = task < 2 * n1;
    const int t = live ? task : 2 * n1 - 1;
    const bool is_v = t >= n1, rot = ROPE && !is_v;
    const int k = is_v ? t - n1 : t, h = h0 + k % nh;
    const Run run = s_run[k / nh];
    const __nv_bfloat16* src = (is_v ? a.av : a.ak) + (i0 + run.i) * a.as_n + static_cast<long long>(h) * a.as_h;
    uint8_t* page0 = (is_v ? a.vc : a.kc) + run.page * a.s_page + static_cast<long long>(h) * a.s_head;
    float* scale = (is_v ? a.vs : a.ks) + run.page * a.ss_page + static_cast<long long>(h) * a.ss_head;
    const float s_old = run.slot > 0 && live ? *scale : 0.f;
    Words w = load_row(src, c, rot);
    if (rot)
      w = rotate<NORM>(w, [&](int f) { return s_angle[run.i][angle_slot(f)]; }, c, a.sorted != 0, w1, w2, a.eps);
    float m = abs_max(w, 0.f);
    __syncwarp();
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    const float s_new = fmaxf(s_old, scale_for(m));  // (a scale is above 0)
    // pages whose scale grows, by the whole warp one after another
    unsigned grown = __ballot_sync(0xffffffffu, live && run.slot > 0 && s_new != s_old && c == 0);
    for (; grown != 0; grown &= grown - 1) {
      const int l = __ffs(grown) - 1;
      uint8_t* page = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<uintptr_t>(page0), l));
      round_again<8>(page, a.s_tok, lane >> 3, 4, __shfl_sync(0xffffffffu, run.slot, l),
                     __shfl_sync(0xffffffffu, s_old, l), __shfl_sync(0xffffffffu, s_new, l), c);
    }
    if (!live) continue;
    uint32_t o[4];
    round_words(w, s_new, o);
    uint8_t* dst = page0 + static_cast<long long>(run.slot) * a.s_tok;
    if (rot && !a.sorted) {
      *reinterpret_cast<uint2*>(dst + 8 * c) = make_uint2(o[0], o[1]);
      *reinterpret_cast<uint2*>(dst + 64 + 8 * c) = make_uint2(o[2], o[3]);
    } else {
      *reinterpret_cast<uint4*>(dst + 16 * (rot ? 7 - c : c)) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    if (c == 0) *scale = s_new;
  }
}

}  // namespace append8
}  // namespace atf

using namespace atf;

extern "C" int atf_paged_kv_append_e4m3(const AtfAppendParams* p, const AtfKvScales* s, atf_stream_t stream) {
  return append_e4m3(p, s, nullptr, stream);
}

int atf::append_e4m3(const AtfAppendParams* p, const AtfKvScales* s, const AtfKNorm* norm, atf_stream_t stream) {
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
  int rc = norm_args_ok(p, norm);
  if (rc != ATF_OK) return rc;
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
  rc = check_device(&dev);
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
  // tokens per CTA: the most, up to 32, that give every SM a CTA, but as many as a run is
  // long, up to 16 (2048 tokens of one request, 8 heads, pages of 64 with norm: windows of 8
  // 20.6 us, of 16 16.5, of 32 14.3; but of a batch of 13 uneven prompts 20.8, 20.5, 22.5)
  const long long run = std::min<long long>(p->page_size, std::max<long long>(a.nnz / p->batch_size, 1));
  a.window = append8::MAX_WINDOW;
  while (a.window > std::min<long long>(run, 16) && (a.nnz + a.window - 1) / a.window < 148) a.window >>= 1;
  const long long blocks = (a.nnz + a.window - 1) / a.window;
  if (blocks > 0x7fffffffLL) return ATF_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // Fewer CTAs that begin a run (where runs are longer than the window, not all do) than
  // the SMs hold, with more tasks than their warps take at once: the heads go to several
  // (13 prompts in pages of 64, 4 heads: 24.7 us undivided, 15.3 divided by 4; 2048 tokens of
  // one request in pages of 16, 8 heads: 14.4, by two 12.2, by four, past what the SMs
  // hold, 16.4). Requests may be longer than the mean: up to 4 times its warps are counted.
  const long long runs = run == 1 ? a.window : a.window / run + 1;  // of a window
  const long long warps = (std::min<long long>(p->page_size, 4 * run) + append8::WARP_ROWS - 1) / append8::WARP_ROWS;
  const long long at_once = run == 1 ? 4 * append8::WARPS : append8::WARPS / std::min<long long>(warps, append8::WARPS);
  int split = 1;
  const long long busy = (blocks * std::min<long long>(a.window, run) + run - 1) / run;
  while (split < a.H && 2 * busy * split <= (norm != nullptr ? 2 : 3) * 148 &&
         runs * ((a.H + split - 1) / split) * 2 > at_once)
    split <<= 1;
  a.heads = (a.H + split - 1) / split;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((a.H + a.heads - 1) / a.heads));
  a.norm_w = norm != nullptr ? norm->weight : nullptr;
  a.norm_f32 = norm != nullptr && norm->weight_dtype == ATF_DTYPE_F32 ? 1 : 0;
  a.eps = norm != nullptr ? norm->eps : 0.f;
  if (a.norm_w != nullptr)
    append8::append_e4m3_kernel<true, true><<<grid, append8::THREADS, 0, st>>>(a);
  else if (rope)
    append8::append_e4m3_kernel<true, false><<<grid, append8::THREADS, 0, st>>>(a);
  else
    append8::append_e4m3_kernel<false, false><<<grid, append8::THREADS, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? ATF_OK : ATF_ERR_CUDA;
}
