// RMS norms of the query and key heads with the position rotation in the same pass.
//
// Per row x of 128 bf16: y = x w / sqrt(mean(x^2) + eps), then the rotation of
// rope_math.cuh on y's pairs (i, 64 + i), rounded once to bf16 and written in either
// pair order. Sums, norm and rotation are fp32.
//
// 8 lanes hold a row: 8 pairs each, two 16-byte loads, so that the sum of squares is 16
// products and three shuffles, both elements of a pair are in one lane, and each lane's
// 8 angles are those of its column. They are loaded once for all heads of the token that
// the warp covers: a warp takes 4 U heads of a token, 4 at a time, or U heads of four tokens,
// with the loads of all of them issued before the first is used. A row is read whole before any of it is
// written (the shuffles wait for all 8 lanes), so the outputs may be the inputs.
//
// What bounds it: HBM for prompts, 512 bytes in and out per row; the launch and one
// chain of loads (position -> angles -> row) for a step's tokens, where U = 1 spreads
// them over more SMs. The loads in flight are what counts for prompts: 65521 tokens x 32
// heads take 183 to 191 us on the device (replayed from a graph; 88 to 92% of HBM) with 16 heads
// a warp and four CTAs an SM (64 registers), and beside the 191 196 with three, 202 with 32 heads
// and two, 216 with 8 heads and four; indexes in 64 bits cost 12 us, and streaming hints on loads
// or stores change nothing.
#include "atf_internal.h"
#include "norm_math.cuh"

namespace atf {
namespace qknorm {

constexpr int WARPS = 8;

struct Part {  // the query heads, or the key heads
  const __nv_bfloat16* x;
  __nv_bfloat16* out;
  long long x_b, x_s, x_h, o_b, o_s, o_h;
  const void* w;
};
struct Args {
  Part p[2];
  int Hq, H;  // query heads, all heads
  unsigned S, tokens;
  unsigned units;  // of 4 U heads per token, or of U heads per four tokens
  int w32, pos64, sorted;
  float eps;
  const float* cs;
  const float* sn;
  long long cs_stride, n_pos;
  const void* positions;
  long long pos_b, pos_s, pos_offset;
};

template <int U, bool TOKENS>
__global__ void __launch_bounds__(WARPS * 32, 4) qk_norm_kernel(const Args a) {
  __shared__ __align__(16) float s_w[2][128];
  const int tid = threadIdx.x, lane = tid & 31, c = lane & 7;
  {
    const void* w = a.p[tid >> 7].w;
    s_w[tid >> 7][tid & 127] = w != nullptr ? normmath::weight_at(w, a.w32, tid & 127) : 0.f;
  }
  __syncthreads();
  const unsigned unit = blockIdx.x * WARPS + (tid >> 5);  // all units and a CTA more fit 32 bits
  const unsigned first = unit / a.units;  // token, or four of them
  if ((TOKENS ? 4 * first : first) >= a.tokens) return;
  const int hu = static_cast<int>(unit - first * a.units);
  const int h0 = TOKENS ? hu * U : hu * (4 * U) + (lane >> 3);
  constexpr int STEP = TOKENS ? 1 : 4;
  const bool in = !TOKENS || 4 * first + (lane >> 3) < a.tokens;
  const unsigned t = TOKENS ? min(4 * first + (lane >> 3), a.tokens - 1) : first;
  const long long b = t / a.S, s = t - static_cast<unsigned>(b) * a.S;
  long long pos = a.pos_offset + s;
  if (a.positions != nullptr) {
    const long long at = b * a.pos_b + s * a.pos_s;
    pos = a.pos64 ? static_cast<const int64_t*>(a.positions)[at] : static_cast<const int32_t*>(a.positions)[at];
  }
  pos = pos < 0 ? 0 : (pos >= a.n_pos ? a.n_pos - 1 : pos);
  uint4 lo[U], hi[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = min(h0 + STEP * u, a.H - 1);  // (rows past the last head are not written)
    const Part& p = a.p[h < a.Hq ? 0 : 1];
    const __nv_bfloat16* row = p.x + b * p.x_b + s * p.x_s + (h < a.Hq ? h : h - a.Hq) * p.x_h;
    lo[u] = *reinterpret_cast<const uint4*>(row + 8 * c);
    hi[u] = *reinterpret_cast<const uint4*>(row + 64 + 8 * c);
  }
  float cv[8], sv[8];
  normmath::load8(a.cs + pos * a.cs_stride + 8 * c, cv);
  normmath::load8(a.sn + pos * a.cs_stride + 8 * c, sv);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + STEP * u;
    const bool q = h < a.Hq;
    float x1[8], x2[8], w1[8], w2[8];
    normmath::unpack(lo[u], x1);
    normmath::unpack(hi[u], x2);
    normmath::load8(&s_w[q ? 0 : 1][8 * c], w1);
    normmath::load8(&s_w[q ? 0 : 1][64 + 8 * c], w2);
    normmath::normalise(x1, x2, w1, w2, a.eps, 0xffffffffu);
    uint32_t o[8];
    normmath::rotate(x1, x2, cv, sv, a.sorted != 0, o);
    if (in && h < a.H) {
      const Part& p = a.p[q ? 0 : 1];
      __nv_bfloat16* row = p.out + b * p.o_b + s * p.o_s + (q ? h : h - a.Hq) * p.o_h;
      normmath::store_pairs(row, c, a.sorted != 0, 16, o);
    }
  }
}

}  // namespace qknorm
}  // namespace atf

using namespace atf;

extern "C" int atf_qk_norm_rope(const AtfQkNormParams* p, atf_stream_t stream) {
  if (p == nullptr || p->cos == nullptr || p->sin == nullptr) return ATF_ERR_INVALID_ARG;
  if (p->head_dim != ATF_HEAD_DIM) return ATF_ERR_UNSUPPORTED;
  if (p->batch < 0 || p->seqlen < 0 || p->num_heads_q < 0 || p->num_heads_k < 0 || p->n_pos < 1 ||
      p->cs_stride_pos < 64 || !(p->eps > 0.f && p->eps <= FLT_MAX))
    return ATF_ERR_INVALID_ARG;
  if ((p->num_heads_q > 0 && (p->q == nullptr || p->q_out == nullptr || p->q_weight == nullptr)) ||
      (p->num_heads_k > 0 && (p->k == nullptr || p->k_out == nullptr || p->k_weight == nullptr)))
    return ATF_ERR_INVALID_ARG;
  if ((p->weight_dtype != ATF_DTYPE_BF16 && p->weight_dtype != ATF_DTYPE_F32) ||
      (p->out_layout != ATF_LAYOUT_SORTED_PAIR && p->out_layout != ATF_LAYOUT_ROTATE_HALF))
    return ATF_ERR_INVALID_ARG;
  if (p->num_heads_q > (1 << 20) || p->num_heads_k > (1 << 20)) return ATF_ERR_UNSUPPORTED;
  const int64_t strides[12] = {p->q_stride_b,     p->q_stride_s,     p->q_stride_h,     p->k_stride_b,
                               p->k_stride_s,     p->k_stride_h,     p->q_out_stride_b, p->q_out_stride_s,
                               p->q_out_stride_h, p->k_out_stride_b, p->k_out_stride_s, p->k_out_stride_h};
  for (int i = 0; i < 12; ++i)
    if ((strides[i] & 7) != 0) return ATF_ERR_ALIGNMENT;
  if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->q_out) || !aligned16(p->k_out) || !aligned16(p->cos) ||
      !aligned16(p->sin) || (p->cs_stride_pos & 3) != 0)
    return ATF_ERR_ALIGNMENT;
  // an output over its own input has the same strides, or rows would be read after they
  // were written
  if ((p->q == p->q_out && p->num_heads_q > 0 &&
       (p->q_stride_b != p->q_out_stride_b || p->q_stride_s != p->q_out_stride_s ||
        p->q_stride_h != p->q_out_stride_h)) ||
      (p->k == p->k_out && p->num_heads_k > 0 &&
       (p->k_stride_b != p->k_out_stride_b || p->k_stride_s != p->k_out_stride_s ||
        p->k_stride_h != p->k_out_stride_h)))
    return ATF_ERR_INVALID_ARG;
  qknorm::Args a = {};
  a.Hq = static_cast<int>(p->num_heads_q);
  a.H = static_cast<int>(p->num_heads_q + p->num_heads_k);
  if (p->batch == 0 || p->seqlen == 0 || a.H == 0) return ATF_OK;
  const long long narrow = (a.H + 3) / 4;  // units of 4 heads a token
  if (p->batch > (1ll << 30) || p->seqlen > (1ll << 30) || p->batch * p->seqlen > (1ll << 30) / narrow)
    return ATF_ERR_UNSUPPORTED;
  a.S = static_cast<unsigned>(p->seqlen);
  a.tokens = static_cast<unsigned>(p->batch * p->seqlen);
  int dev = 0;
  int rc = check_device(&dev);
  if (rc != ATF_OK) return rc;
  a.p[0] = {static_cast<const __nv_bfloat16*>(p->q), static_cast<__nv_bfloat16*>(p->q_out), p->q_stride_b,
            p->q_stride_s, p->q_stride_h, p->q_out_stride_b, p->q_out_stride_s, p->q_out_stride_h,
            a.Hq > 0 ? p->q_weight : nullptr};
  a.p[1] = {static_cast<const __nv_bfloat16*>(p->k), static_cast<__nv_bfloat16*>(p->k_out), p->k_stride_b,
            p->k_stride_s, p->k_stride_h, p->k_out_stride_b, p->k_out_stride_s, p->k_out_stride_h,
            p->num_heads_k > 0 ? p->k_weight : nullptr};
  a.w32 = p->weight_dtype == ATF_DTYPE_F32 ? 1 : 0;
  a.pos64 = p->positions_64 ? 1 : 0;
  a.sorted = p->out_layout == ATF_LAYOUT_SORTED_PAIR ? 1 : 0;
  a.eps = p->eps;
  a.cs = p->cos;
  a.sn = p->sin;
  a.cs_stride = p->cs_stride_pos;
  a.n_pos = p->n_pos;
  a.positions = p->positions;
  a.pos_b = p->pos_stride_b;
  a.pos_s = p->pos_stride_s;
  a.pos_offset = p->pos_offset;
  // 16 rows per warp once that gives every SM two CTAs, else 4: 16 heads of a token, or 4 of
  // four tokens where that leaves fewer lanes idle (65521 tokens x 5 heads 84 and 54 us, x 8
  // 88 and 62, x 20 170 and 133, x 40 263 and 250; but x 16 104 and 109, x 32 194 and 203)
  const long long wide = (a.H + 15) / 16;
  const bool many = a.tokens * wide >= 2ll * 148 * qknorm::WARPS;
  const bool tokens = many && narrow < 4 * wide;
  a.units = static_cast<unsigned>(many && !tokens ? wide : narrow);
  const long long items = tokens ? (a.tokens + 3ll) / 4 : a.tokens;
  const unsigned blocks = static_cast<unsigned>((items * a.units + qknorm::WARPS - 1) / qknorm::WARPS);
  constexpr int threads = qknorm::WARPS * 32;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (tokens)
    qknorm::qk_norm_kernel<4, true><<<blocks, threads, 0, st>>>(a);
  else if (many)
    qknorm::qk_norm_kernel<4, false><<<blocks, threads, 0, st>>>(a);
  else
    qknorm::qk_norm_kernel<1, false><<<blocks, threads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? ATF_OK : ATF_ERR_CUDA;
}
