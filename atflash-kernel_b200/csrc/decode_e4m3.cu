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
// exponential costs 4 ex2 per thread and group. P is rounded to f16: 11 bits (where
// the bf16 decode keeps 8) down to 2^-21 of the largest p vs of the warp's keys, and
// an absolute 2^-32 of that per key below (f16's subnormals; M is kept 7 lower than
// the maximum for this). m and M move only when a score exceeds them by
// more than 8, so most stages need no maximum over lanes and no pass over O.
//
// CTA = (unit of atf_decode_plan, kv head): one producer warp with TMA boxes per
// page slice, and 8 consumer warps in two quads that take 64-key stages in turn, 16
// keys per warp; two CTAs per SM. Rows are always read whole: HBM is read in lines of
// 128 bytes here, and boxes of the 32 or 64 bytes that a window needs of a K row took
// as long as whole rows (4 x 128K keys in pages of 64: 170-176 us). A unit holds
// pieces of several requests, cut so that all units cost the same: one wave of CTAs,
// equally long whatever the requests' lengths (37 ragged requests: 73 us with one
// item per CTA, 55 so). The producer runs through the pieces without a stop while
// the consumers write each piece's state (2.8 us of a CTA's time per piece).
//
// Measured: 8 x 128K keys, 24 / 8 heads, window on 326 us in HND pages of 64 (the
// copy bandwidth, rows read whole; off 316), 361 in NHD pages of 16 (boxes of 2 KB; off
// 350); 37 requests up to 20011 keys (28 / 4 heads) 56 us, 80%: the SMs' shares end
// between 44 and 52 us; 3 requests up to 300 keys 8.1 us with the merge.
#include <cuda_fp16.h>
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <vector>

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
using decode::movmatrix_t;

constexpr int STAGE_KEYS = 64;
constexpr int CONSUMERS = 8;                          // two quads of 4 warps, alternate stages
constexpr int THREADS = (CONSUMERS + 1) * 32;
// Even, so that a slot of the ring is always the same quad's: its waits then see
// every phase of the slot's barrier (a parity wait one phase early returns at once).
constexpr int NSTAGE = 4;
static_assert(NSTAGE % 2 == 0, "a slot belongs to one quad");
constexpr uint32_t K_BYTES = STAGE_KEYS * 128;
constexpr uint32_t V_BYTES = STAGE_KEYS * 128;
constexpr uint32_t STAGE_BYTES = K_BYTES + V_BYTES;   // 16 KB
constexpr uint32_t RING_BYTES = NSTAGE * STAGE_BYTES; // 64 KB
constexpr uint32_t MERGE_BYTES = 16384;
constexpr uint32_t Q_PITCH = 272;              // bytes of a staged q row (2-way bank conflicts at most)
constexpr uint32_t Q_BYTES = 2 * 16 * Q_PITCH; // two items' rows
constexpr int MAX_UNIT_PAGES = ATF_DECODE_UNIT_PAGES;
constexpr int MAX_UNIT_ITEMS = ATF_DECODE_UNIT_ITEMS;
constexpr uint32_t OFF_MERGE = RING_BYTES;
constexpr uint32_t OFF_Q = OFF_MERGE + MERGE_BYTES;
constexpr uint32_t OFF_STATS = OFF_Q + Q_BYTES;            // 3 x [CONSUMERS][16] floats
constexpr uint32_t OFF_META = OFF_STATS + 3 * CONSUMERS * 16 * 4;  // Meta[MAX_UNIT_ITEMS]
constexpr uint32_t OFF_LIM = OFF_META + 24 * MAX_UNIT_ITEMS;       // int[MAX_UNIT_ITEMS][8]
constexpr uint32_t OFF_SCALES = OFF_LIM + 32 * MAX_UNIT_ITEMS;     // float2[MAX_UNIT_PAGES]
constexpr uint32_t OFF_PAGES = OFF_SCALES + 8 * MAX_UNIT_PAGES;    // int[MAX_UNIT_PAGES]
constexpr uint32_t OFF_BAR = OFF_PAGES + 4 * MAX_UNIT_PAGES;
constexpr uint32_t OFF_ABORT = OFF_BAR + 8 * 2 * NSTAGE;
constexpr uint32_t SMEM_BYTES = OFF_ABORT + 16 + 1024;
constexpr uint32_t FULLMASK = 0xffffffffu;
constexpr float LAZY = 8.f;      // a maximum moves when a score exceeds it by more
// P's maximum is kept this much lower, so that P <= 2^15 (LAZY + RISE), just below f16's
// largest value, and small weights have the most room above its subnormals
constexpr float RISE = 7.f;
constexpr float LOWEST = -1e30f; // a running maximum before any key
static_assert((OFF_META & 15) == 0 && (OFF_SCALES & 7) == 0 && (OFF_BAR & 7) == 0, "shared memory layout");
static_assert(2 * (SMEM_BYTES + 1024) <= 228 * 1024, "two CTAs per SM");

struct Args {
  const __nv_bfloat16* q;
  long long q_sb, q_sh;
  const int* indptr;
  const int* indices;
  const int* last_page_len;
  const int* items;
  int num_items;
  const int64_t* q_pos;
  const int64_t* kv_pos0;
  const float* ks;
  const float* vs;
  long long ss_page, ss_head;
  long long num_pages;
  int B, Hq, Hkv, G, page_size, page_shift, rows;
  float scale_log2;
  int zhi16[ATF_MAX_LEVELS];
  float* part_o;
  float* part_lse;
  int* err;
};

// an item of the unit, as staged in shared memory
struct Meta {
  int b, k_beg, k_end;
  int page0;     // first of its pages in the unit's list
  int list0;     // where those begin in `indices`
  int first;     // its first page within the request
};
static_assert(sizeof(Meta) == 24, "six ints");

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
__device__ __forceinline__ void consumers_sync() {
  __barrier_sync_count(1, CONSUMERS * 32);
}

// NT: tiles of 8 query heads (the group's size is at most 8 NT). WIN: a window.
template <int NT, bool WIN>
__global__ void __launch_bounds__(THREADS, NT == 1 ? 2 : 1)
    decode_e4m3_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  // the split merge that follows on the stream may be scheduled now; it waits
  // for this grid's completion before reading the partial states
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sb = (raw + 1023u) & ~1023u;
  uint8_t* sp = smem_raw + (sb - raw);
  auto full_bar = [&](int s) { return sb + OFF_BAR + 8u * s; };
  auto empty_bar = [&](int s) { return sb + OFF_BAR + 8u * (NSTAGE + s); };
  volatile int* s_abort = reinterpret_cast<volatile int*>(sp + OFF_ABORT);
  int* s_total = reinterpret_cast<int*>(sp + OFF_ABORT + 4);  // pages of the unit, -1: refused
  Meta* s_meta = reinterpret_cast<Meta*>(sp + OFF_META);
  int* s_lim = reinterpret_cast<int*>(sp + OFF_LIM);  // window: local key that level l is read from on
  int* s_pages = reinterpret_cast<int*>(sp + OFF_PAGES);
  float2* s_scale = reinterpret_cast<float2*>(sp + OFF_SCALES);  // (ks, log2 vs) of the unit's pages

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // Heads run fastest over the grid: a plan with units has rows that name none, and
  // their blocks, which leave at once, come after every block that works.
  const int hk = static_cast<int>(blockIdx.x) % a.Hkv;
  // The unit's items: row x of the plan names its first item (1-based; 0: the
  // row is a unit of its own, negative: no unit).
  const int x = static_cast<int>(blockIdx.x) / a.Hkv;
  const int tag = a.items[4 * x + 3];
  const int next = x + 1 < a.num_items ? a.items[4 * x + 7] : 0;
  if (tag < 0) return;
  const int it0 = tag > 0 ? tag - 1 : x;
  const int n_items = (tag > 0 ? (next > 0 ? next - 1 : a.num_items) : x + 1) - it0;
  // Prologue, part 1: only the plan and the page table, which the kernel just before
  // does not write where programmatic dependent launch is on (this part runs before
  // that kernel's end). An item names a request of the batch, starts on a 64-key
  // boundary and lies inside its request; the unit's pages fit the list. Else it is
  // reported and skipped.
  if (warp == 0) {
    int total = 0;
    bool bad = n_items < 1 || n_items > MAX_UNIT_ITEMS || it0 < 0 || it0 + n_items > a.num_items;
    for (int i0 = 0; !bad && i0 < n_items; i0 += 32) {
      const int i = i0 + lane;
      int n = 0;
      Meta m;
      bool wrong = false;
      if (i < n_items) {
        const int4 row = reinterpret_cast<const int4*>(a.items)[it0 + i];
        m.b = row.x;
        m.k_beg = row.y;
        m.k_end = row.z;
        const bool known = m.b >= 0 && m.b < a.B;
        const int pg0 = known ? a.indptr[m.b] : 0, npages = known ? a.indptr[m.b + 1] - pg0 : 0;
        const long long len =
            npages > 0 ? static_cast<long long>(npages - 1) * a.page_size + a.last_page_len[m.b] : 0;
        wrong = m.k_beg < 0 || m.k_end <= m.k_beg || (m.k_beg & 63) || m.k_end > len;
        m.first = m.k_beg >> a.page_shift;
        m.list0 = pg0 + m.first;
        n = wrong ? 0 : ((m.k_end - 1) >> a.page_shift) - m.first + 1;
      }
      int sum = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(FULLMASK, sum, off);
        if (lane >= off) sum += y;
      }
      m.page0 = total + sum - n;
      if (i < n_items) s_meta[i] = m;
      // (a page list past MAX_UNIT_PAGES cannot wrap: the sum is checked per 32 items)
      total += __shfl_sync(FULLMASK, sum, 31);
      bad = __any_sync(FULLMASK, wrong || n > MAX_UNIT_PAGES) || total > MAX_UNIT_PAGES;
    }
    if (lane == 0) {
      *s_total = bad ? -1 : total;
      *s_abort = stops(a.err) ? 1 : 0;
      if (bad && a.err != nullptr) atomicCAS(a.err, 0, kDevErrIndex);
      for (int s = 0; s < NSTAGE; ++s) {
        mbar_init(full_bar(s), 1);
        mbar_init(empty_bar(s), CONSUMERS / 2);
      }
      fence_mbar_init();
    }
  } else if (warp == CONSUMERS) {
    if (lane == 0) tma_prefetch_desc(&tmK);
    if (lane == 1) tma_prefetch_desc(&tmV);
  }
  __syncthreads();
  const int total_pages = *s_total;
  // read here, where no wait can change it: a warp that left on an error raised later
  // would be missing at the consumers' barriers
  const bool start_ok = *s_abort == 0;
  if (total_pages < 0) return;
  // page j of the unit is page j - page0 of the last item with page0 <= j
  auto item_of_page = [&](int j) {
    int lo = 0, hi = n_items;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_meta[mid].page0 <= j) lo = mid; else hi = mid;
    }
    return lo;
  };
  for (int j = tid; j < total_pages; j += THREADS) {
    const Meta& m = s_meta[item_of_page(j)];
    s_pages[j] = a.indices[m.list0 + j - m.page0];
  }
  // Part 2: what a preceding kernel may have written (positions, query, pages,
  // scales) is read from here on.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (WIN && tid < n_items * ATF_MAX_LEVELS) {
    const int b = s_meta[tid >> 3].b, l = tid & 7;
    const int np = a.indptr[b + 1] - a.indptr[b];  // an item's request is not empty
    const long long len = static_cast<long long>(np - 1) * a.page_size + a.last_page_len[b];
    const long long q_pos = a.q_pos != nullptr ? a.q_pos[b] : len - 1;
    const long long zb = q_pos - (a.kv_pos0 != nullptr ? a.kv_pos0[b] : 0);
    s_lim[tid] = l == 0 ? INT_MIN : key_limit(zb, a.zhi16[l]);
  }
  __syncthreads();
  const AbortCtl ab{s_abort, a.err};
  if (!start_ok) return;

  if (warp == CONSUMERS) {
    // ------------------------------------------------------------ producer
    const int R = a.rows;
    const int slice = lane >> 1, is_v = lane & 1;  // one lane per box
    const int r0 = slice * R;
    int buf = 0, ph = 1, issued = 0;
    bool ok = true;
    for (int i = 0; ok && i < n_items; ++i) {
      const Meta m = s_meta[i];
      for (int k0 = m.k_beg; k0 < m.k_end; k0 += STAGE_KEYS) {
        ok = __all_sync(FULLMASK, mbar_wait(empty_bar(buf), ph, ab, kDevErrTimeout));
        if (!ok) break;
        const bool live = r0 < STAGE_KEYS && k0 + r0 < m.k_end;
        uint32_t bytes = live ? static_cast<uint32_t>(R) * 128u : 0u;
#pragma unroll
        for (int off = 4; off > 0; off >>= 1) bytes += __shfl_xor_sync(FULLMASK, bytes, off);  // lanes 0..7
        if (lane == 0) mbar_arrive_expect_tx(full_bar(buf), bytes);
        __syncwarp();
        if (live) {
          const int n = k0 + r0;
          const int page = s_pages[m.page0 + (n >> a.page_shift) - m.first];
          const int tok = n & (a.page_size - 1);
          const uint32_t st = sb + buf * STAGE_BYTES;
          tma_load_4d(st + (is_v ? K_BYTES : 0u) + static_cast<uint32_t>(r0) * 128u, is_v ? &tmV : &tmK,
                      full_bar(buf), 0, tok, hk, page);
        }
        __syncwarp();
        ++issued;
        if (++buf == NSTAGE) {
          buf = 0;
          ph ^= 1;
        }
      }
    }
    // every copy in flight lands before the CTA ends
    for (int s = issued > NSTAGE ? issued - NSTAGE : 0; s < issued; ++s) {
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(full_bar(s % NSTAGE), (s / NSTAGE) & 1))
        if (globaltimer_ns() - t0 > kWaitLimitNs) break;
    }
    return;
  }

  // -------------------------------------------------------------- consumers
  // An item's q is copied to shared memory while the item before it runs (the first
  // one's before the loads of K and V fill the memory's queues), in two buffers by
  // turns; rows past the group's heads are zero.
  const int G = a.G, hq0 = hk * G;
  auto copy_q = [&](int i) {
    const int b = s_meta[i].b;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = 8 * nt + warp;
      const __nv_bfloat16* src =
          a.q + static_cast<long long>(b) * a.q_sb + static_cast<long long>(hq0 + h) * a.q_sh + 4 * lane;
      const uint32_t dst = sb + OFF_Q + static_cast<uint32_t>((i & 1) * 16 + h) * Q_PITCH + 8u * lane;
      if (h < G)
        asm volatile(
            "cp.async.ca.shared.global [%0], [%1], 4;\n\t"
            "cp.async.ca.shared.global [%0+4], [%1+4], 4;" ::"r"(dst), "l"(src)
            : "memory");
    }
  };
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
    if (8 * nt + warp >= G)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        *reinterpret_cast<uint2*>(sp + OFF_Q + (k * 16 + 8 * nt + warp) * Q_PITCH + 8 * lane) = make_uint2(0, 0);
  copy_q(0);
  // the unit's scales, once, while the first pages are on their way
  for (int j = tid; j < total_pages; j += CONSUMERS * 32) {
    const int page = s_pages[j];
    float2 v = make_float2(0.f, -INFINITY);
    if (page >= 0 && page < a.num_pages) {
      const long long at = page * a.ss_page + hk * a.ss_head;
      v = make_float2(a.ks[at], log2f(a.vs[at]));
    } else if (a.err != nullptr) {
      atomicCAS(a.err, 0, kDevErrIndex);
    }
    s_scale[j] = v;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  consumers_sync();

  const int g = lane >> 2, t4 = lane & 3;
  const int quad = warp >> 2, wq = warp & 3;  // this warp: keys 16 wq .. of every second stage
  const int mi = lane >> 3, mr = lane & 7;
  // ldmatrix rows of the warp's 16 keys, matrices (keys 0-7, chunk c), (keys 8-15, c),
  // (0-7, c + 1), (8-15, c + 1). Rows of 128 bytes: 16-byte chunks XORed with the row.
  const uint32_t row = static_cast<uint32_t>(16 * wq) + ((mi & 1) << 3) + mr;
  uint32_t off[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) off[p] = row * 128u + 16u * ((2u * p + static_cast<uint32_t>(mi >> 1)) ^ (row & 7u));
  int cur = quad, buf = quad, ph = 0;  // this quad's next stage, its slot and parity
  int end = 0;                         // stages of the items so far
  bool ok = true;
  // (after a wait that ran out the items pass without their stages, through the
  // same barriers)
  for (int i = 0; i < n_items; ++i) {
    const Meta m = s_meta[i];
    // levels that the keys up to next_lim - 1 read (keys come in rising order, their
    // distance falls)
    int levels = 0, next_lim = INT_MIN;
    // q as the B operand, heads as columns: in the MMA of level i, k-rows 2 t4,
    // 2 t4 + 1 are dims 16 i + 4 t4 + {0, 1} and k-rows 2 t4 + {8, 9} dims + {2, 3}
    uint32_t qb[NT][8][2];
    float qsl[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t* qrow =
          reinterpret_cast<const uint32_t*>(sp + OFF_Q + ((i & 1) * 16 + 8 * nt + g) * Q_PITCH) + 2 * t4;
      float mx = 0.f;
#pragma unroll
      for (int l = 0; l < 8; ++l)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t w = qrow[8 * l + e];
          qb[nt][l][e] = w;
          mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u))));
        }
      mx = fmaxf(mx, __shfl_xor_sync(FULLMASK, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(FULLMASK, mx, 2));
      // 2^sh with mx * 2^sh in [2^14, 2^15); 1 for a row of zeros or with an infinity
      const int ex = static_cast<int>(__float_as_uint(mx) >> 23);  // biased
      const int sh = (mx > 0.f && ex < 255) ? min(14 + 127 - ex, 126) : 0;
      const float up = __uint_as_float(static_cast<uint32_t>(sh + 127) << 23);
#pragma unroll
      for (int l = 0; l < 8; ++l)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t w = qb[nt][l][e];
          qb[nt][l][e] = pack_f16(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up);
        }
      // log2-domain factor of this lane's column head, then of this thread's heads
      const float f = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - sh) << 23);
      qsl[nt][0] = __shfl_sync(FULLMASK, f, 8 * t4);
      qsl[nt][1] = __shfl_sync(FULLMASK, f, 8 * t4 + 4);
    }
    // this thread's heads: 8 nt + 2 t4 + {0, 1}
    float m_s[NT][2], m_u[NT][2], l_run[NT][2], o[NT][8][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m_s[nt][0] = m_s[nt][1] = m_u[nt][0] = m_u[nt][1] = LOWEST;
      l_run[nt][0] = l_run[nt][1] = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
    }
    if (i + 1 < n_items) copy_q(i + 1);
    const int begin = end;
    end += (m.k_end - m.k_beg + STAGE_KEYS - 1) / STAGE_KEYS;
    while (cur < end) {
      ok = ok && __all_sync(FULLMASK, mbar_wait(full_bar(buf), ph, ab, kDevErrTimeout));
      if (!ok) break;
      const uint32_t kb = sb + buf * STAGE_BYTES;
      const uint32_t vb = kb + K_BYTES;
      const int key0 = m.k_beg + (cur - begin) * STAGE_KEYS + 16 * wq;
      if (key0 < m.k_end) {
        const int last = min(key0 + 15, m.k_end - 1);
        const bool whole = last == key0 + 15;
        const float2 sc = s_scale[m.page0 + (key0 >> a.page_shift) - m.first];
        // this thread's keys: key0 + g (c[0], c[1]) and key0 + g + 8 (c[2], c[3])
        float c[NT][4], c2[NT][4];  // two sums, so that the MMAs wait less for each other
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) c[nt][e] = c2[nt][e] = 0.f;
        // levels that all keys of the group read, and that its newest reads: the same
        // but where a level begins
        int Lmax = ATF_MAX_LEVELS;
        if (WIN) {
          if (last >= next_lim) {
            auto count = [&](int L, int key) {
              while (L < ATF_MAX_LEVELS && key >= s_lim[8 * i + L]) ++L;
              return L;
            };
            levels = count(levels, key0);
            next_lim = levels < ATF_MAX_LEVELS ? s_lim[8 * i + levels] : INT_MAX;
            Lmax = count(levels, last);
          } else {
            Lmax = levels;
          }
        }
        if (!WIN || levels == Lmax) {
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            if (!WIN || 2 * p < Lmax) {
              uint32_t r[4], a0, a1, a2, a3;
              ldsm_x4(kb + off[p], r[0], r[1], r[2], r[3]);
              e4m3x4_to_f16(r[0], a0, a2);
              e4m3x4_to_f16(r[1], a1, a3);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_f16(c[nt], a0, a1, a2, a3, qb[nt][2 * p][0], qb[nt][2 * p][1]);
              if (!WIN || 2 * p + 1 < Lmax) {
                e4m3x4_to_f16(r[2], a0, a2);
                e4m3x4_to_f16(r[3], a1, a3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                  mma_f16(c2[nt], a0, a1, a2, a3, qb[nt][2 * p + 1][0], qb[nt][2 * p + 1][1]);
              }
            }
          }
        } else {
          // level by level: one that only the newer keys read counts from its limit on
#pragma unroll
          for (int l = 0; l < ATF_MAX_LEVELS; ++l) {
            if (l < Lmax) {
              uint32_t r[4], a0, a1, a2, a3;
              ldsm_x4(kb + off[l >> 1], r[0], r[1], r[2], r[3]);
              e4m3x4_to_f16(r[2 * (l & 1)], a0, a2);
              e4m3x4_to_f16(r[2 * (l & 1) + 1], a1, a3);
              const int from = s_lim[8 * i + l];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float t[4] = {0.f, 0.f, 0.f, 0.f};
                mma_f16(t, a0, a1, a2, a3, qb[nt][l][0], qb[nt][l][1]);
                c[nt][0] += key0 + g >= from ? t[0] : 0.f;
                c[nt][1] += key0 + g >= from ? t[1] : 0.f;
                c[nt][2] += key0 + g + 8 >= from ? t[2] : 0.f;
                c[nt][3] += key0 + g + 8 >= from ? t[3] : 0.f;
              }
            }
          }
        }
        bool need = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) c[nt][e] = (c[nt][e] + c2[nt][e]) * (qsl[nt][e & 1] * sc.x);
          if (!whole) {
            if (key0 + g > last) c[nt][0] = c[nt][1] = -INFINITY;
            if (key0 + g + 8 > last) c[nt][2] = c[nt][3] = -INFINITY;
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mx = fmaxf(c[nt][e], c[nt][e + 2]) - LAZY;
            need |= mx > m_s[nt][e] || mx + (sc.y - RISE) > m_u[nt][e];
          }
        }
        if (__any_sync(FULLMASK, need)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mh = fmaxf(c[nt][e], c[nt][e + 2]);  // over the group's 16 keys
#pragma unroll
              for (int of = 4; of < 32; of <<= 1) mh = fmaxf(mh, __shfl_xor_sync(FULLMASK, mh, of));
              const float ns = fmaxf(m_s[nt][e], mh), nu = fmaxf(m_u[nt][e], mh + (sc.y - RISE));
              l_run[nt][e] *= ex2f(m_s[nt][e] - ns);
              const float al = ex2f(m_u[nt][e] - nu);
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
            const float mu = sc.y - m_u[nt][e];
            l_run[nt][e] += ex2f(c[nt][e] - m_s[nt][e]) + ex2f(c[nt][e + 2] - m_s[nt][e]);
            w[e] = ex2f(c[nt][e] + mu);
            w[e + 2] = ex2f(c[nt][e + 2] + mu);
          }
          // P^T (keys x heads) as the B operand: transpose the blocks of 8 keys
          pb[nt][0] = movmatrix_t(pack_f16(w[0], w[1]));
          pb[nt][1] = movmatrix_t(pack_f16(w[2], w[3]));
        }
        // V: bytes (key, dim 2g), (key, dim 2g + 1), (next key, 2g), (next key, 2g + 1)
        // are sorted by dim; MMA rows g and g + 8 are dims 2g and 2g + 1 of the chunk
        auto pv = [&](uint32_t keep0, uint32_t keep1) {
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) {
            uint32_t r[4];
            ldsm_x4_t(vb + off[jj], r[0], r[1], r[2], r[3]);
#pragma unroll
            for (int hl = 0; hl < 2; ++hl) {
              uint32_t a0, a1, a2, a3;
              e4m3x4_to_f16(__byte_perm(r[2 * hl], 0, 0x3120) & keep0, a0, a1);
              e4m3x4_to_f16(__byte_perm(r[2 * hl + 1], 0, 0x3120) & keep1, a2, a3);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma_f16(o[nt][2 * jj + hl], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
            }
          }
        };
        if (whole) {
          pv(FULLMASK, FULLMASK);
        } else {
          // rows past the item's end may hold anything: their P is 0, so that their V
          // must be a number (this thread's V elements are keys 2 t4, 2 t4 + 1 of each 8)
          const int k = key0 + 2 * t4;
          pv((k <= last ? 0x00ff00ffu : 0u) | (k + 1 <= last ? 0xff00ff00u : 0u),
             (k + 8 <= last ? 0x00ff00ffu : 0u) | (k + 9 <= last ? 0xff00ff00u : 0u));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty_bar(buf));
      cur += 2;
      buf += 2;
      if (buf >= NSTAGE) {
        buf -= NSTAGE;
        ph ^= 1;
      }
    }
    // ---------------------------------------------------------- the item's state
    // The 8 warps' states are merged through shared memory of their own, in 2 NT
    // passes over the dims, while the producer goes on with the next item.
    constexpr int ROWS = 8 * NT, PASSES = 2 * NT, DP = 128 / PASSES, JP = 8 / PASSES;
    float* sm_o = reinterpret_cast<float*>(sp + OFF_MERGE);  // [CONSUMERS][ROWS][DP]
    float* sm_s = reinterpret_cast<float*>(sp + OFF_STATS);  // [CONSUMERS][ROWS] each
    float* sm_u = sm_s + CONSUMERS * ROWS;
    float* sm_l = sm_u + CONSUMERS * ROWS;
    static_assert(CONSUMERS * ROWS * DP * 4 <= MERGE_BYTES, "merge buffer");
    float l_sum[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // the sums are per thread (its two keys of each group): add the 8 key rows
        l_sum[nt][e] = l_run[nt][e];
#pragma unroll
        for (int of = 4; of < 32; of <<= 1) l_sum[nt][e] += __shfl_xor_sync(FULLMASK, l_sum[nt][e], of);
      }
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
      if (pass == 0) asm volatile("cp.async.wait_all;" ::: "memory");  // the next item's q
      consumers_sync();  // the buffer has been read
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int rw = warp * ROWS + 8 * nt + 2 * t4 + e;
          float2* dst = reinterpret_cast<float2*>(sm_o + rw * DP);
#pragma unroll
          for (int j = 0; j < JP; ++j)
            dst[8 * j + g] = make_float2(o[nt][JP * pass + j][e], o[nt][JP * pass + j][e + 2]);
          if (pass == 0 && g == 0) {
            sm_s[rw] = m_s[nt][e];
            sm_u[rw] = m_u[nt][e];
            sm_l[rw] = l_sum[nt][e];
          }
        }
      consumers_sync();
      for (int e = tid; e < G * (DP / 4); e += CONSUMERS * 32) {
        const int rw = e / (DP / 4), d = 4 * (e % (DP / 4));
        float ms = LOWEST, mu = LOWEST;
#pragma unroll
        for (int w = 0; w < CONSUMERS; ++w) {
          ms = fmaxf(ms, sm_s[w * ROWS + rw]);
          mu = fmaxf(mu, sm_u[w * ROWS + rw]);
        }
        float L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < CONSUMERS; ++w) {
          L += ex2f(sm_s[w * ROWS + rw] - ms) * sm_l[w * ROWS + rw];
          const float f = ex2f(sm_u[w * ROWS + rw] - mu);
          const float4 v = *reinterpret_cast<const float4*>(sm_o + (w * ROWS + rw) * DP + d);
          acc.x += f * v.x;
          acc.y += f * v.y;
          acc.z += f * v.z;
          acc.w += f * v.w;
        }
        // every V scale 0: mu is still the lowest, and so is f
        const float f = L > 0.f ? ex2f(mu - ms) / L : 0.f;
        const long long at = static_cast<long long>(it0 + i) * a.Hq + hq0 + rw;
        *reinterpret_cast<float4*>(a.part_o + at * 128 + pass * DP + d) =
            make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
        if (pass == 0 && d == 0) a.part_lse[at] = L == 0.f ? -INFINITY : ms + log2f(L);  // NaN stays
      }
    }
  }
}

// The split merge with a warp per (request, head), for many requests of few items,
// where merge_kernel's block of 8 warps a row mostly waits: 256 requests of up to 2000
// keys, 24 heads, 91.5 -> 82.4 us; 64 of 100 keys, 32 heads, 16.5 -> 14.9. With fewer
// rows than its blocks fill at once that kernel is faster (3 requests 8.2 against 9.1).
constexpr int ROW_WARPS = 8;

__global__ void __launch_bounds__(ROW_WARPS * 32) merge_rows_kernel(const merge::Args a) {
  const int lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * ROW_WARPS + (threadIdx.x >> 5);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // the decode kernel is complete and its states are visible past this point
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (row >= static_cast<long long>(a.B) * a.H) return;
  const int b = static_cast<int>(row / a.H), h = static_cast<int>(row % a.H);
  int n;
  long long lb, sl, ob, so;
  merge::ragged_parts(a, b, h, &n, &lb, &sl, &ob, &so);
  float M = -INFINITY;
  for (int i = lane; i < n; i += 32) M = fmaxf(M, a.pl[lb + i * sl]);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(FULLMASK, M, off));
  float L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += 32) {
    // lane k holds the weight of part i0 + k
    const float lp = i0 + lane < n ? a.pl[lb + (i0 + lane) * sl] : -INFINITY;
    const float w = lp == -INFINITY ? 0.f : exp2f(lp - M);
    L += w;
    const float* o = a.po + ob + i0 * so + lane * 4;
    const int m = min(n - i0, 32);
#pragma unroll 4
    for (int k = 0; k < m; ++k) {
      const float wk = __shfl_sync(FULLMASK, w, k);
      const float4 v = *reinterpret_cast<const float4*>(o + k * so);
      acc.x += wk * v.x;
      acc.y += wk * v.y;
      acc.z += wk * v.z;
      acc.w += wk * v.w;
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(FULLMASK, L, off);
  const float inv = L > 0.f ? 1.0f / L : 0.f;
  merge::store_row(a.out, static_cast<long long>(b) * a.o_sb + static_cast<long long>(h) * a.o_sh, a.out_f32, a.lse_out,
                   row, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv),
                   L == 0.f ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f);
}

// keys in whose time an item starts and writes its state (2.8 us measured)
constexpr long long ITEM_COST = 288;

struct Piece {  // an item; opens: the first of its unit
  int b;
  long long k0, k1;
  bool opens;
};

// the cost of the dearest unit, in keys
long long longest_unit(const std::vector<Piece>& pieces) {
  long long most = 0, unit = 0;
  for (const Piece& p : pieces) {
    unit = (p.opens ? 0 : unit) + p.k1 - p.k0 + ITEM_COST;
    most = std::max(most, unit);
  }
  return most;
}

// Keys of the next item of a request with `left` keys, where `want` (a multiple of 64,
// at most room) would do for the balance: an item holds at least min_keys, and leaves as
// many to the next one or none, as far as the request and `room` allow. (At the least
// min_keys, 64, a last item may be shorter.)
long long item_keys(long long left, long long want, long long room, long long min_keys) {
  const long long n = std::min(std::max(want, min_keys), room);
  if (left <= n) return left;
  if (min_keys <= 64 || left - n >= min_keys) return n;
  if (left <= room) return left;
  const long long less = (left - min_keys) / 64 * 64;
  return less >= min_keys ? less : n;
}

// Requests cut into items of about `chunk` keys, each a unit.
std::vector<Piece> cut_evenly(const std::vector<long long>& lens, long long chunk, long long cap, long long min_keys) {
  std::vector<Piece> out;
  for (size_t b = 0; b < lens.size(); ++b)
    for (long long n0 = 0, n; n0 < lens[b]; n0 += n) {
      n = item_keys(lens[b] - n0, chunk, cap, min_keys);
      out.push_back({static_cast<int>(b), n0, n0 + n, true});
    }
  return out;
}

// The requests' keys on one line, each at the same cost (a key's rows are read whole
// whatever the window) and each request with that of its state: unit u is the part up
// to (u + 1) / U of the whole. An item costs a
// start of its own, so a request is not begun for the last keys that a unit wants, nor
// are its own last ones left to the next unit, up to `slack` keys.
std::vector<Piece> cut_in_units(const std::vector<long long>& lens, long long U, long long whole, long long cap,
                                long long min_keys, int ps) {
  const long long slack = std::min(ITEM_COST / 2, whole / (2 * U));
  std::vector<Piece> out;
  long long units = 0, done = 0;  // done: cost of everything cut so far
  long long unit_pages = 0, unit_items = 0;
  for (size_t b = 0; b < lens.size(); ++b) {
    const long long len = lens[b];
    long long n0 = 0;
    while (n0 < len) {
      // the unit in progress is full: by cost, by items or by pages
      bool opens = units == 0 || done * U >= whole * units || unit_items >= MAX_UNIT_ITEMS || unit_pages >= MAX_UNIT_PAGES;
      if (n0 == 0 && whole * units - done * U < slack * U) opens = true;
      if (opens) {
        ++units;
        unit_pages = unit_items = 0;
      }
      // (an item begins at a multiple of 64, so inside a page of 128 or 256)
      long long room = (MAX_UNIT_PAGES - unit_pages) * static_cast<long long>(ps) - n0 % ps;
      room = std::min(room, cap) / 64 * 64;
      const long long left = len - n0, start = n0 == 0 ? ITEM_COST : 0;
      // the first 64-key boundary at which the unit has its share, or the end
      const long long share = (whole * units + U - 1) / U - done - start;  // keys that the unit still wants
      long long n = std::max((share + 63) / 64 * 64, min_keys);
      if (left - n < slack) n = left;
      n = item_keys(left, n, room, min_keys);
      // no room for a block, or for items of min_keys: the next unit takes it
      const bool cramped = min_keys > 64 && unit_items > 0 && (n < std::min(min_keys, left) || (n < left && left - n < min_keys));
      if (room < 64 || cramped) {
        unit_pages = MAX_UNIT_PAGES;
        continue;
      }
      out.push_back({static_cast<int>(b), n0, n0 + n, opens});
      unit_pages += (n0 + n - 1) / ps - n0 / ps + 1;
      ++unit_items;
      done += start + n;
      n0 += n;
    }
  }
  return out;
}

// U fills the slots (two resident CTAs per SM, over the kv heads) in as few waves as
// the units' limits allow, with at least min_chunk_keys (64) keys per item where its
// request has them.
int plan_units(const AtfDecodePlanParams* p, long long slots, int32_t* items_host, int32_t items_capacity,
               int32_t* item_indptr_host, AtfDecodePlan* out) {
  const int B = p->batch_size, ps = p->page_size;
  const long long unit_cap = std::min(MAX_UNIT_PAGES * static_cast<long long>(ps), 16384ll);
  long long cap = unit_cap;  // keys of an item
  if (p->max_chunk_keys > 0 && p->max_chunk_keys < cap) cap = p->max_chunk_keys;
  cap = std::max(cap / 64 * 64, 64ll);
  const long long min_keys = p->min_chunk_keys > 64 ? std::min((p->min_chunk_keys + 63ll) / 64 * 64, cap) : 64;
  std::vector<long long> lens(static_cast<size_t>(B));
  long long whole = 0, keys = 0, pieces = 0;  // pieces: the most that are worth an item
  for (int b = 0; b < B; ++b) {
    const int np = p->indptr_host[b + 1] - p->indptr_host[b];
    const long long len = np > 0 ? static_cast<long long>(np - 1) * ps + p->last_page_len_host[b] : 0;
    lens[static_cast<size_t>(b)] = len;
    if (len > 0) whole += len + ITEM_COST;
    keys += len;
    pieces += (len + min_keys - 1) / min_keys;
  }
  const long long per_wave = std::max(slots / p->num_kv_heads, 1ll);
  const long long waves = std::max((keys + per_wave * unit_cap - 1) / (per_wave * unit_cap), 1ll);
  const long long U = std::max(std::min(per_wave * waves, pieces), 1ll);
  std::vector<Piece> cut = cut_in_units(lens, U, whole, cap, min_keys, ps);
  // Where the requests fit one wave as units of one item: the smallest such items,
  // taken where they end sooner (30 requests of 3 keys 50 -> 9.1 us, 50 of up to 300
  // keys 14.4 -> 11.0, 3 of up to 300 10.5 -> 8.2).
  auto items_of = [&](long long chunk) {
    long long n = 0;
    for (const long long len : lens) n += (len + chunk - 1) / chunk;
    return n;
  };
  if (items_of(cap) <= per_wave) {
    long long lo = min_keys / 64, hi = cap / 64;  // in blocks of 64 keys; hi fits
    while (lo < hi) {
      const long long mid = (lo + hi) / 2;
      if (items_of(mid * 64) <= per_wave) hi = mid; else lo = mid + 1;
    }
    std::vector<Piece> even = cut_evenly(lens, hi * 64, cap, min_keys);
    if (longest_unit(even) < longest_unit(cut)) cut.swap(even);
  }
  const long long n = static_cast<long long>(cut.size());
  if (items_host != nullptr && n > items_capacity) return ATF_ERR_WORKSPACE;
  long long longest = 0, units = 0;
  int b = 0;  // offsets up to here are written
  for (long long i = 0; i < n; ++i) {
    const Piece& c = cut[static_cast<size_t>(i)];
    longest = std::max(longest, c.k1 - c.k0);
    if (item_indptr_host != nullptr)
      for (; b <= c.b; ++b) item_indptr_host[b] = static_cast<int32_t>(i);
    if (items_host == nullptr) continue;
    items_host[4 * i + 0] = c.b;
    items_host[4 * i + 1] = static_cast<int32_t>(c.k0);
    items_host[4 * i + 2] = static_cast<int32_t>(c.k1);
    if (c.opens) items_host[4 * units++ + 3] = static_cast<int32_t>(i + 1);
  }
  if (items_host != nullptr)
    for (; units < n; ++units) items_host[4 * units + 3] = -1;
  if (item_indptr_host != nullptr)
    for (; b <= B; ++b) item_indptr_host[b] = static_cast<int32_t>(n);
  out->num_items = static_cast<int32_t>(n);
  out->chunk_keys = static_cast<int32_t>(longest);
  out->partial_o_floats = static_cast<int64_t>(n) * p->num_qo_heads * ATF_HEAD_DIM;
  out->partial_lse_floats = static_cast<int64_t>(n) * p->num_qo_heads;
  return ATF_OK;
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
    a.num_items = p->num_items;
    a.q_pos = p->q_pos;
    a.kv_pos0 = p->kv_pos0;
    a.ks = sc->k_scale;
    a.vs = sc->v_scale;
    a.ss_page = sc->stride_page;
    a.ss_head = sc->stride_head;
    a.num_pages = p->num_pages;
    a.B = p->batch_size;
    a.Hq = p->num_qo_heads;
    a.Hkv = p->num_kv_heads;
    a.G = G;
    a.page_size = ps;
    a.page_shift = 0;
    while ((1 << a.page_shift) < ps) ++a.page_shift;
    a.rows = ps < 64 ? ps : 64;
    a.scale_log2 = p->sm_scale * 1.4426950408889634f;
    const bool win = p->window == ATF_WINDOW_SNAP16;
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
    const uint64_t vdims[4] = {128, static_cast<uint64_t>(ps), hkv, npg};
    const uint64_t vstr[3] = {s_tok, s_head, s_page};
    const uint32_t vbox[4] = {128, rows, 1, 1};
    CUtensorMap tk, tv;
    if ((rc = encode_tiled_u8(&tk, p->k_cache, 4, vdims, vstr, vbox, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_128B)) != ATF_OK)
      return rc;
    if ((rc = encode_tiled_u8(&tv, p->v_cache, 4, vdims, vstr, vbox, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_128B)) != ATF_OK)
      return rc;
    auto kern = G > 8 ? (win ? decode8::decode_e4m3_kernel<2, true> : decode8::decode_e4m3_kernel<2, false>)
                      : (win ? decode8::decode_e4m3_kernel<1, true> : decode8::decode_e4m3_kernel<1, false>);
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, decode8::SMEM_BYTES) != cudaSuccess)
      return ATF_ERR_CUDA;
    const long long blocks = static_cast<long long>(p->num_items) * p->num_kv_heads;
    if (blocks > INT_MAX) return ATF_ERR_UNSUPPORTED;
    const dim3 grid(static_cast<unsigned>(blocks));
    if (launch_pdl(kern, grid, decode8::THREADS, decode8::SMEM_BYTES, st, p->enable_pdl != 0, tk, tv, a) !=
        cudaSuccess)
      return ATF_ERR_CUDA;
    if (cudaGetLastError() != cudaSuccess) return ATF_ERR_CUDA;
  }
  const long long rows = static_cast<long long>(p->batch_size) * p->num_qo_heads;
  // more rows than blocks of merge_kernel run at once, with few items each (an item's
  // parts are read one after another here): a warp per row
  if (p->num_items > 0 && p->num_items <= 4ll * p->batch_size && rows > 8 * 148 && rows <= INT_MAX) {
    const dim3 grid(static_cast<unsigned>((rows + decode8::ROW_WARPS - 1) / decode8::ROW_WARPS));
    return launch_pdl(decode8::merge_rows_kernel, grid, decode8::ROW_WARPS * 32, 0, st, true,
                      merge::decode_merge_args(p)) == cudaSuccess ? ATF_OK : ATF_ERR_CUDA;
  }
  return merge::launch(merge::decode_merge_args(p), st, /*after_decode=*/p->num_items > 0);
}
