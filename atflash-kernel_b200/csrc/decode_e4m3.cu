// Paged GQA split-KV decode over an e4m3 cache with one scale per (page, kv head).
//
// Per query head, over the keys n of its request (page(n) = the key's page):
//   s_n = sm_scale * ks[page(n)] * sum_{d in window(n)} q_d k_nd
//   o   = sum_n softmax(s)_n * vs[page(n)] * v_n
// with k, v the stored e4m3 values. A key at distance z from the query reads the
// first 16 * #{i : zhi16[i] >= z} dims of its row (sorted pairs; level 0 always),
// as in the bf16 decode.
//
// What bounds it: HBM, at 256 bytes per key and kv head (half the bf16 cache's).
// At the measured copy bandwidth an SM takes in about 23 bytes, i.e. 23 elements,
// per clock, so what counts is instructions per element:
//   - e4m3 goes to f16 in the fragments (cvt: two elements an instruction, exact)
//     and both products run as f16 MMAs with fp32 sums. q is scaled by a power of
//     two per head so that its largest element lies in [2^14, 2^15): every bf16 q
//     keeps its bits down to 2^-28 of that.
//   - keys are the MMA rows (S^T = K Q^T, O^T = V^T P^T), heads the 8 columns: a
//     16-key, 32-dim ldmatrix of K is two MMA operands as it stands, since the
//     order of the dims in the sum is free as long as q has the same; the
//     transposed load of V pairs two dims per 16-bit unit, one byte permute per
//     register splits them.
//   - a group of 16 keys lies in one page, so its two scales are two values per
//     group: ks goes into the factor that brings a score to log2 units, log2(vs)
//     is added to the scores for P V.
// The scale of V in the exponent keeps P V free of its range: with m the running
// maximum of s and M that of s + log2 vs (both log2 units), l = sum 2^(s - m) and
// O = sum 2^(s + log2 vs - M) v; the row is O / l * 2^(M - m). The second
// exponential costs 4 ex2 per thread and group. P is rounded to f16 (11 bits,
// where the bf16 decode keeps 8). m and M move only when a score exceeds them by
// more than 8, so most stages need no maximum over lanes and no pass over O.
//
// CTA = (work item of atf_decode_plan, kv head): one producer warp with TMA boxes
// per page slice (K as 32-byte slabs of two window levels each, only those in the
// window; V rows of 128 bytes), 8 consumer warps with 16 keys each of a 128-key
// stage. Two CTAs per SM.
#include <cuda_fp16.h>
#include <limits.h>
#include <math.h>

#include "atf_internal.h"
#include "atf_ptx.cuh"
#include "decode_common.cuh"
#include "merge.cuh"

namespace atf {
namespace decode8 {

using decode::ex2f;
using decode::key_limit;
using decode::ldsm_x4;
using decode::ldsm_x4_t;
using decode::levels_of;
using decode::movmatrix_t;

constexpr int STAGE_KEYS = 128;
constexpr int CONSUMERS = 8;
constexpr int THREADS = (CONSUMERS + 1) * 32;
constexpr int NSTAGE_MAX = 4;
constexpr int SLABS = 4;                              // 32-byte slabs of a K row
constexpr uint32_t SLAB_BYTES = STAGE_KEYS * 32;
constexpr uint32_t V_BYTES = STAGE_KEYS * 128;
constexpr uint32_t RING_BYTES = 3 * (SLABS * SLAB_BYTES + V_BYTES);  // 96 KB
constexpr int MAX_ITEM_KEYS = 16384;  // atf_decode_plan never makes longer items
constexpr int MAX_ITEM_PAGES = MAX_ITEM_KEYS / 16 + 2;
constexpr uint32_t OFF_BAR = RING_BYTES;
constexpr uint32_t OFF_ABORT = OFF_BAR + 8 * 2 * NSTAGE_MAX;
constexpr uint32_t OFF_ZB = OFF_ABORT + 8;
constexpr uint32_t OFF_PAGES = OFF_BAR + 128;
constexpr uint32_t OFF_SCALES = OFF_PAGES + 4 * MAX_ITEM_PAGES;
constexpr uint32_t SMEM_BYTES = OFF_SCALES + 8 * MAX_ITEM_PAGES + 1024;
constexpr uint32_t FULLMASK = 0xffffffffu;
constexpr float LAZY = 8.f;  // P <= 2^8: exact enough in f16, far from its largest value
static_assert(OFF_ZB + 8 <= OFF_PAGES && (OFF_SCALES & 7) == 0, "shared memory layout");

struct Args {
  const __nv_bfloat16* q;
  long long q_sb, q_sh;
  const int* indptr;
  const int* indices;
  const int* last_page_len;
  const int* items;
  const int64_t* q_pos;
  const int64_t* kv_pos0;
  const float* ks;
  const float* vs;
  long long ss_page, ss_head;
  long long num_pages;
  int Hq, G, page_size, page_shift, rows;
  float scale_log2;
  int window;
  int zhi16[ATF_MAX_LEVELS];
  float* part_o;
  float* part_lse;
  int* err;
};

// K tensor maps over (32 bytes of a slab, token, slab, kv head, page); map n-1
// has the box {32, rows, n, 1, 1}
struct KMaps {
  CUtensorMap n[SLABS];
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// four e4m3 bytes as two f16x2 words (bytes 0, 1 and bytes 2, 3)
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t x, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(x));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// NT: tiles of 8 query heads (the group's size is at most 8 NT)
template <int NT>
__global__ void __launch_bounds__(THREADS, NT == 1 ? 2 : 1)
    decode_e4m3_kernel(const __grid_constant__ KMaps tmK, const __grid_constant__ CUtensorMap tmV, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  // the split merge that follows on the stream may be scheduled now; it waits
  // for this grid's completion before reading the partial states
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sb = (raw + 1023u) & ~1023u;
  uint8_t* sp = smem_raw + (sb - raw);
  auto full_bar = [&](int s) { return sb + OFF_BAR + 8u * s; };
  auto empty_bar = [&](int s) { return sb + OFF_BAR + 8u * (NSTAGE_MAX + s); };
  volatile int* s_abort = reinterpret_cast<volatile int*>(sp + OFF_ABORT);
  volatile long long* s_zb = reinterpret_cast<volatile long long*>(sp + OFF_ZB);
  int* s_pages = reinterpret_cast<int*>(sp + OFF_PAGES);
  float2* s_scale = reinterpret_cast<float2*>(sp + OFF_SCALES);  // (ks, log2 vs) of the item's pages

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int item = blockIdx.x, hk = blockIdx.y;
  // Prologue, part 1: only the plan and the page table, which no kernel of this
  // step writes (it runs before the previous kernel's end under programmatic
  // dependent launch).
  const int b = a.items[4 * item + 0];
  const int k_beg = a.items[4 * item + 1];
  const int k_end = a.items[4 * item + 2];
  const int pg0 = a.indptr[b];
  const int npages = a.indptr[b + 1] - pg0;
  const long long kv_len =
      npages > 0 ? static_cast<long long>(npages - 1) * a.page_size + a.last_page_len[b] : 0;
  // an item starts on a 64-key boundary, lies inside its request and holds at
  // most MAX_ITEM_KEYS keys; any other is reported and skipped
  if (k_beg < 0 || k_end < k_beg || (k_beg & 63) || k_end > kv_len || k_end - k_beg > MAX_ITEM_KEYS) {
    if (tid == 0 && a.err != nullptr) atomicCAS(a.err, 0, kDevErrIndex);
    return;
  }
  const int G = a.G, hq0 = hk * G;
  const int nst = (k_end - k_beg + STAGE_KEYS - 1) / STAGE_KEYS;
  if (tid == 0) {
    *s_abort = (a.err != nullptr && *reinterpret_cast<volatile int*>(a.err) != 0) ? 1 : 0;
    for (int s = 0; s < NSTAGE_MAX; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), CONSUMERS);
    }
    fence_mbar_init();
  }
  const int first_page = k_beg >> a.page_shift;
  const int n_item_pages = k_end > k_beg ? ((k_end - 1) >> a.page_shift) - first_page + 1 : 0;
  if (warp == CONSUMERS) {
    if (lane < SLABS) tma_prefetch_desc(&tmK.n[lane]);
    if (lane == SLABS) tma_prefetch_desc(&tmV);
  }
  for (int i = tid; i < n_item_pages; i += THREADS) s_pages[i] = a.indices[pg0 + first_page + i];
  // Part 2: what a preceding kernel may have written (positions, query, pages,
  // scales) is read from here on.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (tid == 0) {
    const long long q_pos = a.q_pos != nullptr ? a.q_pos[b] : kv_len - 1;
    const long long pos0 = a.kv_pos0 != nullptr ? a.kv_pos0[b] : 0;
    *s_zb = q_pos - pos0;
  }
  __syncthreads();
  const long long zb = *s_zb;
  int lim[ATF_MAX_LEVELS];  // level i is read by local keys n >= lim[i]
#pragma unroll
  for (int i = 0; i < ATF_MAX_LEVELS; ++i)
    lim[i] = (!a.window || i == 0) ? INT_MIN : key_limit(zb, a.zhi16[i]);
  // ring geometry of this item: the slabs that its newest key reads
  const int Sc = k_end > k_beg ? (levels_of(lim, k_end - 1) + 1) >> 1 : SLABS;
  const uint32_t K_BYTES = static_cast<uint32_t>(Sc) * SLAB_BYTES;
  const uint32_t STAGE_BYTES = K_BYTES + V_BYTES;
  const int NSTAGE = min(NSTAGE_MAX, static_cast<int>(RING_BYTES / STAGE_BYTES));
  const AbortCtl ab{s_abort, a.err};
  const bool start_ok = (*s_abort == 0);
  const int g = lane >> 2, t4 = lane & 3;

  // this thread's heads: 8 nt + 2 t4 + {0, 1}
  float m_s[NT][2], m_u[NT][2], l_run[NT][2], o[NT][8][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m_s[nt][0] = m_s[nt][1] = m_u[nt][0] = m_u[nt][1] = -INFINITY;
    l_run[nt][0] = l_run[nt][1] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
  }

  if (start_ok && warp == CONSUMERS) {
    // ------------------------------------------------------------ producer
    const int R = a.rows;
    const int slice = lane >> 1, is_v = lane & 1;  // one lane per box
    const int r0 = slice * R;
    int issued = 0;
    for (int s = 0; s < nst; ++s) {
      const int buf = s % NSTAGE;
      if (!__all_sync(FULLMASK, mbar_wait(empty_bar(buf), ((s / NSTAGE) & 1) ^ 1, ab, kDevErrTimeout))) break;
      const int k0 = k_beg + s * STAGE_KEYS;
      const int nkeys = min(STAGE_KEYS, k_end - k0);
      const bool live = r0 < nkeys && r0 < STAGE_KEYS;
      int n_slab = 0;
      if (live) n_slab = (levels_of(lim, min(k0 + r0 + R, k_end) - 1) + 1) >> 1;
      uint32_t bytes = live ? static_cast<uint32_t>(R) * (is_v ? 128u : 32u * n_slab) : 0u;
      const uint32_t mine = bytes;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) bytes += __shfl_xor_sync(FULLMASK, bytes, off);
      mbar_arrive_expect_tx_elect(full_bar(buf), bytes);
      __syncwarp();
      if (mine != 0) {
        const int n = k0 + r0;
        const int page = s_pages[(n >> a.page_shift) - first_page];
        const int tok = n & (a.page_size - 1);
        const uint32_t st = sb + buf * STAGE_BYTES;
        if (is_v)
          tma_load_4d(st + K_BYTES + static_cast<uint32_t>(r0) * 128u, &tmV, full_bar(buf), 0, tok, hk, page);
        else
          tma_load_5d(st + static_cast<uint32_t>(r0 * Sc) * 32u, &tmK.n[n_slab - 1], full_bar(buf), 0, tok, 0, hk,
                      page);
      }
      __syncwarp();
      issued = s + 1;
    }
    // every copy in flight lands before shared memory is used again
    for (int s = issued - NSTAGE; s < issued; ++s)
      if (s >= 0) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(full_bar(s % NSTAGE), (s / NSTAGE) & 1))
          if (globaltimer_ns() - t0 > kWaitLimitNs) break;
      }
  } else if (start_ok) {
    // ------------------------------------------------------------ consumers
    // the item's scales, once, while the first pages are on their way
    for (int i = tid; i < n_item_pages; i += CONSUMERS * 32) {
      const int page = s_pages[i];
      float2 v = make_float2(0.f, -INFINITY);
      if (page >= 0 && page < a.num_pages) {
        const long long at = page * a.ss_page + hk * a.ss_head;
        v = make_float2(a.ks[at], log2f(a.vs[at]));
      } else if (a.err != nullptr) {
        atomicCAS(a.err, 0, kDevErrIndex);
      }
      s_scale[i] = v;
    }
    // q as the B operand, heads as columns: in the MMA of level i, k-rows 2 t4,
    // 2 t4 + 1 are dims 16 i + 4 t4 + {0, 1} and k-rows 2 t4 + {8, 9} dims + {2, 3}
    uint32_t qb[NT][8][2];
    float qsl[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = 8 * nt + g;
      const bool v0 = h < G;
      const __nv_bfloat16* qrow =
          a.q + static_cast<long long>(b) * a.q_sb + static_cast<long long>(hq0 + (v0 ? h : 0)) * a.q_sh;
      float mx = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t w = v0 ? *reinterpret_cast<const uint32_t*>(qrow + 16 * i + 4 * t4 + 2 * e) : 0u;
          qb[nt][i][e] = w;
          mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u))));
        }
      mx = fmaxf(mx, __shfl_xor_sync(FULLMASK, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(FULLMASK, mx, 2));
      // 2^sh with mx * 2^sh in [2^14, 2^15); 1 for a row of zeros or with an infinity
      const int ex = static_cast<int>(__float_as_uint(mx) >> 23);  // biased
      const int sh = (mx > 0.f && ex < 255) ? min(14 + 127 - ex, 126) : 0;
      const float up = __uint_as_float(static_cast<uint32_t>(sh + 127) << 23);
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t w = qb[nt][i][e];
          qb[nt][i][e] = pack_f16(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up);
        }
      // log2-domain factor of this lane's column head, then of this thread's heads
      const float f = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - sh) << 23);
      qsl[nt][0] = __shfl_sync(FULLMASK, f, 8 * t4);
      qsl[nt][1] = __shfl_sync(FULLMASK, f, 8 * t4 + 4);
    }
    asm volatile("bar.sync 1, %0;" ::"n"(CONSUMERS * 32) : "memory");  // s_scale is complete

    // this warp's 16 keys of a stage lie in slice 16 warp / R
    const uint32_t R = static_cast<uint32_t>(a.rows);
    const uint32_t slice = static_cast<uint32_t>(warp * 16) / R, in_slice = static_cast<uint32_t>(warp * 16) % R;
    const int mi = lane >> 3, mr = lane & 7;
    // ldmatrix rows. K: matrices (keys 0-7, level 2p), (keys 8-15, 2p), (0-7, 2p+1),
    // (8-15, 2p+1) in 32-byte rows, 16-byte halves swapped by bit 2 of the row
    const uint32_t krow = in_slice + ((mi & 1) << 3) + mr;
    const uint32_t k_off = slice * R * 32u * static_cast<uint32_t>(Sc) + krow * 32u +
                           16u * (static_cast<uint32_t>(mi >> 1) ^ ((krow >> 2) & 1u));
    const uint32_t slab_stride = 32u * R;
    // V: matrices (keys 0-7, 16 dims), (8-15, same), (0-7, next 16 dims), (8-15, next)
    // in 128-byte rows whose 16-byte chunks are XORed with the row
    const uint32_t vrow = static_cast<uint32_t>(warp * 16) + ((mi & 1) << 3) + mr;
    const uint32_t v_off = vrow * 128u;
    const uint32_t vx = vrow & 7u;

    for (int s = 0; s < nst; ++s) {
      const int buf = s % NSTAGE;
      if (!__all_sync(FULLMASK, mbar_wait(full_bar(buf), (s / NSTAGE) & 1, ab, kDevErrTimeout))) break;
      const uint32_t kb = sb + buf * STAGE_BYTES + k_off;
      const uint32_t vb = sb + buf * STAGE_BYTES + K_BYTES + v_off;
      const int key0 = k_beg + s * STAGE_KEYS + warp * 16;
      if (key0 < k_end) {
        const int last = min(key0 + 15, k_end - 1);
        const int Lmax = levels_of(lim, last), Lmin = levels_of(lim, key0);
        const float2 sc = s_scale[(key0 >> a.page_shift) - first_page];
        // this thread's keys: key0 + g (c[0], c[1]) and key0 + g + 8 (c[2], c[3])
        const int key_a = key0 + g, key_b = key0 + g + 8;
        float c[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.f;
#pragma unroll
        for (int p = 0; p < SLABS; ++p) {
          if (2 * p < Lmax) {
            uint32_t r[4];
            ldsm_x4(kb + p * slab_stride, r[0], r[1], r[2], r[3]);
#pragma unroll
            for (int hl = 0; hl < 2; ++hl) {
              const int i = 2 * p + hl;
              uint32_t a0, a1, a2, a3;
              e4m3x4_to_f16(r[2 * hl], a0, a2);
              e4m3x4_to_f16(r[2 * hl + 1], a1, a3);
              if (i < Lmin) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_f16(c[nt], a0, a1, a2, a3, qb[nt][i][0], qb[nt][i][1]);
              } else if (i < Lmax) {
                // a level that only the newer keys of the group read
                const bool in_a = key_a >= lim[i], in_b = key_b >= lim[i];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  float t[4] = {0.f, 0.f, 0.f, 0.f};
                  mma_f16(t, a0, a1, a2, a3, qb[nt][i][0], qb[nt][i][1]);
                  if (in_a) {
                    c[nt][0] += t[0];
                    c[nt][1] += t[1];
                  }
                  if (in_b) {
                    c[nt][2] += t[2];
                    c[nt][3] += t[3];
                  }
                }
              }
            }
          }
        }
        const bool ok_a = key_a <= last, ok_b = key_b <= last;
        bool need = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float f0 = qsl[nt][0] * sc.x, f1 = qsl[nt][1] * sc.x;
          c[nt][0] = ok_a ? c[nt][0] * f0 : -INFINITY;
          c[nt][1] = ok_a ? c[nt][1] * f1 : -INFINITY;
          c[nt][2] = ok_b ? c[nt][2] * f0 : -INFINITY;
          c[nt][3] = ok_b ? c[nt][3] * f1 : -INFINITY;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mx = fmaxf(c[nt][e], c[nt][e + 2]);
            need |= mx > m_s[nt][e] + LAZY || mx + sc.y > m_u[nt][e] + LAZY;
          }
        }
        if (__any_sync(FULLMASK, need)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mh = fmaxf(c[nt][e], c[nt][e + 2]);  // over the group's 16 keys
#pragma unroll
              for (int off = 4; off < 32; off <<= 1) mh = fmaxf(mh, __shfl_xor_sync(FULLMASK, mh, off));
              const float ns = fmaxf(m_s[nt][e], mh), nu = fmaxf(m_u[nt][e], mh + sc.y);
              l_run[nt][e] *= m_s[nt][e] == -INFINITY ? 0.f : ex2f(m_s[nt][e] - ns);
              const float al = m_u[nt][e] == -INFINITY ? 0.f : ex2f(m_u[nt][e] - nu);
              m_s[nt][e] = ns;
              m_u[nt][e] = nu;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                o[nt][j][e] *= al;
                o[nt][j][e + 2] *= al;
              }
            }
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float ms = m_s[nt][e] == -INFINITY ? 0.f : m_s[nt][e];
            const float mu = sc.y - (m_u[nt][e] == -INFINITY ? 0.f : m_u[nt][e]);
            l_run[nt][e] += ex2f(c[nt][e] - ms) + ex2f(c[nt][e + 2] - ms);
            w[e] = ex2f(c[nt][e] + mu);
            w[e + 2] = ex2f(c[nt][e + 2] + mu);
          }
          // P^T (keys x heads) as the B operand: transpose the blocks of 8 keys
          pb[nt][0] = movmatrix_t(pack_f16(w[0], w[1]));
          pb[nt][1] = movmatrix_t(pack_f16(w[2], w[3]));
        }
        // rows past the item's end may hold anything: their P is 0, so that their V
        // must be a number (this thread's V elements are keys 2 t4, 2 t4 + 1 of each 8)
        uint32_t keep0 = FULLMASK, keep1 = FULLMASK;
        if (last < key0 + 15) {
          const int k = key0 + 2 * t4;
          keep0 = (k <= last ? 0x00ff00ffu : 0u) | (k + 1 <= last ? 0xff00ff00u : 0u);
          keep1 = (k + 8 <= last ? 0x00ff00ffu : 0u) | (k + 9 <= last ? 0xff00ff00u : 0u);
        }
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          uint32_t r[4];
          ldsm_x4_t(vb + 16u * ((2u * jj + static_cast<uint32_t>(mi >> 1)) ^ vx), r[0], r[1], r[2], r[3]);
#pragma unroll
          for (int hl = 0; hl < 2; ++hl) {
            // bytes (key, dim 2g), (key, dim 2g + 1), (next key, 2g), (next key, 2g + 1):
            // sort by dim; MMA rows g and g + 8 are dims 2g and 2g + 1 of the chunk
            uint32_t a0, a1, a2, a3;
            e4m3x4_to_f16(__byte_perm(r[2 * hl], 0, 0x3120) & keep0, a0, a1);
            e4m3x4_to_f16(__byte_perm(r[2 * hl + 1], 0, 0x3120) & keep1, a2, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_f16(o[nt][2 * jj + hl], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty_bar(buf));
    }
  }
  __syncthreads();

  // merge the consumer warps' states (the ring is free now)
  constexpr int ROWS = 8 * NT;
  float* sm_o = reinterpret_cast<float*>(sp);        // [CONSUMERS][ROWS][128]
  float* sm_s = sm_o + CONSUMERS * ROWS * 128;       // [CONSUMERS][ROWS] each
  float* sm_u = sm_s + CONSUMERS * ROWS;
  float* sm_l = sm_u + CONSUMERS * ROWS;
  if (warp < CONSUMERS) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // the sums are per thread (its two keys of each group): add the 8 key rows
        float l = l_run[nt][e];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(FULLMASK, l, off);
        const int row = warp * ROWS + 8 * nt + 2 * t4 + e;
        float2* dst = reinterpret_cast<float2*>(sm_o + row * 128);
#pragma unroll
        for (int j = 0; j < 8; ++j) dst[8 * j + g] = make_float2(o[nt][j][e], o[nt][j][e + 2]);
        if (g == 0) {
          sm_s[row] = m_s[nt][e];
          sm_u[row] = m_u[nt][e];
          sm_l[row] = l;
        }
      }
  }
  __syncthreads();
  if (!start_ok || *s_abort) return;
  for (int e = tid; e < G * 32; e += THREADS) {
    const int row = e >> 5, d = 4 * (e & 31);
    float ms = -INFINITY, mu = -INFINITY;
#pragma unroll
    for (int w = 0; w < CONSUMERS; ++w) {
      ms = fmaxf(ms, sm_s[w * ROWS + row]);
      mu = fmaxf(mu, sm_u[w * ROWS + row]);
    }
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < CONSUMERS; ++w) {
      const float s = sm_s[w * ROWS + row], u = sm_u[w * ROWS + row];
      L += s == -INFINITY ? 0.f : ex2f(s - ms) * sm_l[w * ROWS + row];
      if (u != -INFINITY) {
        const float f = ex2f(u - mu);
        const float4 x = *reinterpret_cast<const float4*>(sm_o + (w * ROWS + row) * 128 + d);
        acc.x += f * x.x;
        acc.y += f * x.y;
        acc.z += f * x.z;
        acc.w += f * x.w;
      }
    }
    const float f = (L > 0.f && mu != -INFINITY) ? ex2f(mu - ms) / L : 0.f;
    const long long at = static_cast<long long>(item) * a.Hq + hq0 + row;
    *reinterpret_cast<float4*>(a.part_o + at * 128 + d) = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
    if (d == 0) a.part_lse[at] = L > 0.f ? ms + log2f(L) : -INFINITY;
  }
}

}  // namespace decode8
}  // namespace atf

using namespace atf;

extern "C" int atf_decode_run_e4m3(const AtfDecodeParams* p, const AtfKvScales* sc, atf_stream_t stream) {
  if (p == nullptr || sc == nullptr || p->q == nullptr || p->k_cache == nullptr || p->v_cache == nullptr ||
      sc->k_scale == nullptr || sc->v_scale == nullptr || p->indptr == nullptr || p->indices == nullptr ||
      p->last_page_len == nullptr || p->items == nullptr || p->item_indptr == nullptr || p->partial_o == nullptr ||
      p->partial_lse == nullptr || p->out == nullptr)
    return ATF_ERR_INVALID_ARG;
  if (p->head_dim != ATF_HEAD_DIM) return ATF_ERR_UNSUPPORTED;
  if (p->batch_size < 1 || p->num_kv_heads < 1 || p->num_qo_heads < 1 || p->num_qo_heads % p->num_kv_heads != 0 ||
      p->page_size < 1 || p->num_items < 0 || p->num_pages < 1)
    return ATF_ERR_INVALID_ARG;
  const int G = p->num_qo_heads / p->num_kv_heads, ps = p->page_size;
  if (G > 16 || p->num_kv_heads > 65535) return ATF_ERR_UNSUPPORTED;
  if (ps != 16 && ps != 32 && ps != 64 && ps != 128 && ps != 256) return ATF_ERR_UNSUPPORTED;
  if (p->k_level_major) return ATF_ERR_UNSUPPORTED;
  if (p->qk_layout != ATF_LAYOUT_SORTED_PAIR && p->qk_layout != ATF_LAYOUT_ROTATE_HALF) return ATF_ERR_INVALID_ARG;
  if (p->window < ATF_WINDOW_OFF || p->window > ATF_WINDOW_VEC8) return ATF_ERR_INVALID_ARG;
  // a window's levels are prefixes of the row in sorted-pair order only
  if (p->window == ATF_WINDOW_VEC8 || (p->window != ATF_WINDOW_OFF && p->qk_layout != ATF_LAYOUT_SORTED_PAIR))
    return ATF_ERR_UNSUPPORTED;
  if (p->window == ATF_WINDOW_SNAP16)
    for (int i = 0; i < ATF_MAX_LEVELS; ++i)
      if (p->zhi16[i] < 0 || (i > 0 && p->zhi16[i] > p->zhi16[i - 1])) return ATF_ERR_INVALID_ARG;
  if (!aligned16(p->k_cache) || !aligned16(p->v_cache) || (p->kv_stride_page & 15) || (p->kv_stride_token & 15) ||
      (p->kv_stride_head & 15))
    return ATF_ERR_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(p->q) & 3) || (p->q_stride_b & 1) || (p->q_stride_h & 1) ||
      !aligned16(p->partial_o) || (reinterpret_cast<uintptr_t>(p->partial_lse) & 3) ||
      (p->out_dtype == ATF_DTYPE_F32 && !aligned16(p->out)) || (reinterpret_cast<uintptr_t>(p->out) & 7) ||
      (p->o_stride_b & 3) || (p->o_stride_h & 3))
    return ATF_ERR_ALIGNMENT;
  int dev = 0;
  int rc = check_device(&dev);
  if (rc != ATF_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (p->num_items > 0) {
    decode8::Args a;
    a.q = static_cast<const __nv_bfloat16*>(p->q);
    a.q_sb = p->q_stride_b;
    a.q_sh = p->q_stride_h;
    a.indptr = p->indptr;
    a.indices = p->indices;
    a.last_page_len = p->last_page_len;
    a.items = p->items;
    a.q_pos = p->q_pos;
    a.kv_pos0 = p->kv_pos0;
    a.ks = sc->k_scale;
    a.vs = sc->v_scale;
    a.ss_page = sc->stride_page;
    a.ss_head = sc->stride_head;
    a.num_pages = p->num_pages;
    a.Hq = p->num_qo_heads;
    a.G = G;
    a.page_size = ps;
    a.page_shift = 0;
    while ((1 << a.page_shift) < ps) ++a.page_shift;
    a.rows = ps < 64 ? ps : 64;
    a.scale_log2 = p->sm_scale * 1.4426950408889634f;
    a.window = p->window == ATF_WINDOW_SNAP16 ? 1 : 0;
    for (int i = 0; i < ATF_MAX_LEVELS; ++i) a.zhi16[i] = p->zhi16[i];
    a.part_o = p->partial_o;
    a.part_lse = p->partial_lse;
    a.err = p->error_flag;
    // a size-1 axis gets a placeholder stride (it is never used)
    auto stride_b = [](uint64_t size, int64_t bytes) { return size == 1 ? 128ull : static_cast<uint64_t>(bytes); };
    const uint64_t hkv = static_cast<uint64_t>(p->num_kv_heads), npg = static_cast<uint64_t>(p->num_pages);
    const uint32_t rows = static_cast<uint32_t>(a.rows);
    const uint64_t s_tok = static_cast<uint64_t>(p->kv_stride_token), s_head = stride_b(hkv, p->kv_stride_head),
                   s_page = stride_b(npg, p->kv_stride_page);
    const uint64_t kdims[5] = {32, static_cast<uint64_t>(ps), decode8::SLABS, hkv, npg};
    const uint64_t kstr[4] = {s_tok, 32, s_head, s_page};
    const uint64_t vdims[4] = {128, static_cast<uint64_t>(ps), hkv, npg};
    const uint64_t vstr[3] = {s_tok, s_head, s_page};
    decode8::KMaps tk;
    CUtensorMap tv;
    for (uint32_t n = 1; n <= decode8::SLABS; ++n) {
      const uint32_t box[5] = {32, rows, n, 1, 1};
      // under a window no promotion: the slabs out of the window are not fetched
      if ((rc = encode_tiled_u8(&tk.n[n - 1], p->k_cache, 5, kdims, kstr, box, CU_TENSOR_MAP_SWIZZLE_32B,
                                a.window ? CU_TENSOR_MAP_L2_PROMOTION_NONE : CU_TENSOR_MAP_L2_PROMOTION_L2_128B)) !=
          ATF_OK)
        return rc;
    }
    const uint32_t vbox[4] = {128, rows, 1, 1};
    if ((rc = encode_tiled_u8(&tv, p->v_cache, 4, vdims, vstr, vbox, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_128B)) != ATF_OK)
      return rc;
    auto kern = G > 8 ? decode8::decode_e4m3_kernel<2> : decode8::decode_e4m3_kernel<1>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, decode8::SMEM_BYTES) != cudaSuccess)
      return ATF_ERR_CUDA;
    const dim3 grid(static_cast<unsigned>(p->num_items), static_cast<unsigned>(p->num_kv_heads));
    if (launch_pdl(kern, grid, decode8::THREADS, decode8::SMEM_BYTES, st, p->enable_pdl != 0, tk, tv, a) !=
        cudaSuccess)
      return ATF_ERR_CUDA;
    if (cudaGetLastError() != cudaSuccess) return ATF_ERR_CUDA;
  }
  return merge::launch(merge::decode_merge_args(p), st, /*after_decode=*/p->num_items > 0);
}
