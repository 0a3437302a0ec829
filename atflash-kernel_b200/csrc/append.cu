// Paged-KV append: writes appended K/V tokens into their pages, optionally
// rotating K (HF rotate_half RoPE, rope_math.cuh) and packing it into the
// cache's pair order on the way. This is the write side that feeds the decode
// from a prefill (FlashInfer's append_paged_kv_cache, which the reference's
// decode path relies on: kernels/flashinfer_port, e2e_pipeline/atflash_e2e_fafi.py:219-223).
//
// Thread = one (token, kv head, chunk c in 0..7): 2 x 16 B of K and of V.
// Token i of request b = batch_indices[i] at position pos = positions[i] goes
// to page kv_indices[kv_indptr[b] + pos / page], slot pos % page. A token
// whose page index lies outside the request's pages or the cache is skipped
// and reported through the error flag (kDevErrIndex).
//
// append_norm_kernel norms K before it rotates it.
#include "atf_internal.h"
#include "norm_math.cuh"
#include "rope_math.cuh"

namespace atf {
namespace append {

struct Args {
  const __nv_bfloat16* ak;
  const __nv_bfloat16* av;
  long long nnz, as_n, as_h;
  const int32_t* batch_indices;
  const int32_t* positions;
  __nv_bfloat16* kc;
  __nv_bfloat16* vc;
  long long num_pages, s_page, s_tok, s_head;
  int H, page_size, B;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  const float* cs;
  const float* sn;
  long long cs_stride, n_pos;
  const int64_t* rope_pos;
  int rope, sorted;
  int* err;
  int k_lm;                              // level-major K pages
  long long k_s_page, k_s_head, k_s_level;
  const void* norm_w;
  int norm_f32;
  float eps;
  unsigned units;  // of heads, per token or per four tokens
};

__global__ void append_kernel(const Args a) {
  const long long gid = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (gid >= a.nnz * a.H * 8) return;
  const int c = static_cast<int>(gid & 7);
  const long long th = gid >> 3;
  const int h = static_cast<int>(th % a.H);
  const long long i = th / a.H;
  const int b = a.batch_indices[i];
  const int pos = a.positions[i];
  bool bad = b < 0 || b >= a.B || pos < 0;
  long long page = -1;
  if (!bad) {
    const int pidx = a.kv_indptr[b] + pos / a.page_size;
    bad = pidx >= a.kv_indptr[b + 1];
    if (!bad) {
      page = a.kv_indices[pidx];
      bad = page < 0 || page >= a.num_pages;
    }
  }
  if (bad) {
    if (a.err != nullptr && c == 0) atomicCAS(a.err, 0, kDevErrIndex);
    return;
  }
  const long long slot = pos % a.page_size;
  const long long dst = page * a.s_page + slot * a.s_tok + static_cast<long long>(h) * a.s_head;
  const long long src = i * a.as_n + static_cast<long long>(h) * a.as_h;
  // V: plain copy of dims [8c, 8c+8) and [64+8c, 64+8c+8)
  *reinterpret_cast<uint4*>(a.vc + dst + 8 * c) = *reinterpret_cast<const uint4*>(a.av + src + 8 * c);
  *reinterpret_cast<uint4*>(a.vc + dst + 64 + 8 * c) = *reinterpret_cast<const uint4*>(a.av + src + 64 + 8 * c);
  // K row base and level stride: a plain row has its 16-dim levels 16 apart;
  // level-major pages keep each level of the page as its own run of 16-dim rows
  const long long kdst = a.k_lm ? page * a.k_s_page + static_cast<long long>(h) * a.k_s_head + slot * 16 : dst;
  const long long lstride = a.k_lm ? a.k_s_level : 16;
  if (!a.rope) {
    // dims [8c, 8c+8) are half (c & 1) of level c/2, dims [64+8c, ..) of level 4 + c/2
    *reinterpret_cast<uint4*>(a.kc + kdst + (c >> 1) * lstride + 8 * (c & 1)) =
        *reinterpret_cast<const uint4*>(a.ak + src + 8 * c);
    *reinterpret_cast<uint4*>(a.kc + kdst + (4 + (c >> 1)) * lstride + 8 * (c & 1)) =
        *reinterpret_cast<const uint4*>(a.ak + src + 64 + 8 * c);
    return;
  }
  long long rp = a.rope_pos != nullptr ? a.rope_pos[i] : pos;
  if (rp < 0) rp = 0;
  if (rp >= a.n_pos) rp = a.n_pos - 1;
  ropemath::rotate_chunk(a.ak + src, a.cs + rp * a.cs_stride, a.sn + rp * a.cs_stride, a.kc + kdst, c,
                         a.sorted != 0, lstride);
}

// With a norm of K in front of the rotation (norm_math.cuh). 8 lanes hold a row, as above,
// and a warp 8 rows, whose loads are on the way while the pages are looked up: two heads
// of four tokens, so that no lane is idle for few heads and the pieces that level-major K
// leaves in (32 bytes a row and level) make up whole lines. A step's tokens (too few for two
// CTAs an SM) go by 4 heads of one token.
//
// HBM-bound for prompts, from cold memory: 64K tokens x 8 heads take 96 us into pages of 16 (90%
// of HBM), 102 into level-major ones; x 4 heads 55 and 57, x 1 head 27 and 29. (Replayed from a
// graph 91 and 96, 49 and 53, 20 and 21: a part comes from L2.) With 8 heads of a token per warp,
// cold, 96 and 107, 73 and 77, 64 and 65. A thread per (row, 8 pairs) as above took 129 / 120
// us (115 / 104 with the loads in front of the lookup), 4 heads a warp 119 / 107, 8 heads with
// more registers and fewer CTAs 123 / 111.
template <bool MANY>
__global__ void __launch_bounds__(256, MANY ? 3 : 4) append_norm_kernel(const Args a) {
  constexpr int U = MANY ? 2 : 1, HSTEP = MANY ? 1 : 4;
  __shared__ __align__(16) float s_w[128];
  const int lane = threadIdx.x & 31, c = lane & 7;
  if (threadIdx.x < 128) s_w[threadIdx.x] = normmath::weight_at(a.norm_w, a.norm_f32 != 0, threadIdx.x);
  __syncthreads();
  const unsigned unit = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);  // (the host keeps them within 32 bits)
  const unsigned first = unit / a.units;  // token, or four of them
  if (first * (MANY ? 4u : 1u) >= a.nnz) return;
  const int hu = static_cast<int>(unit - first * a.units);
  const int h0 = MANY ? hu * U : hu * 4 + (lane >> 3);
  // (lanes behind the last token repeat it and write nothing)
  const bool in = !MANY || first * 4u + (lane >> 3) < a.nnz;
  const unsigned i = MANY ? min(first * 4u + (lane >> 3), static_cast<unsigned>(a.nnz - 1)) : first;
  const int b = a.batch_indices[i];
  const int pos = a.positions[i];
  uint4 k0[U], k1[U], v0[U], v1[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long src = i * a.as_n + static_cast<long long>(min(h0 + HSTEP * u, a.H - 1)) * a.as_h;
    k0[u] = *reinterpret_cast<const uint4*>(a.ak + src + 8 * c);
    k1[u] = *reinterpret_cast<const uint4*>(a.ak + src + 64 + 8 * c);
    v0[u] = *reinterpret_cast<const uint4*>(a.av + src + 8 * c);
    v1[u] = *reinterpret_cast<const uint4*>(a.av + src + 64 + 8 * c);
  }
  long long rp = a.rope_pos != nullptr ? a.rope_pos[i] : pos;
  rp = rp < 0 ? 0 : (rp >= a.n_pos ? a.n_pos - 1 : rp);
  float cv[8], sv[8];
  normmath::load8(a.cs + rp * a.cs_stride + 8 * c, cv);
  normmath::load8(a.sn + rp * a.cs_stride + 8 * c, sv);
  bool bad = b < 0 || b >= a.B || pos < 0;
  long long page = -1;
  if (!bad) {
    const int pidx = a.kv_indptr[b] + pos / a.page_size;
    bad = pidx >= a.kv_indptr[b + 1];
    if (!bad) {
      page = a.kv_indices[pidx];
      bad = page < 0 || page >= a.num_pages;
    }
  }
  if (bad) {
    if (a.err != nullptr && c == 0) atomicCAS(a.err, 0, kDevErrIndex);
    if (!MANY) return;  // (the shuffles below need all lanes of a warp with several tokens)
  }
  const int slot = pos % a.page_size;
  const long long lstride = a.k_lm ? a.k_s_level : 16;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + HSTEP * u;
    const bool on = in && !bad && h < a.H;
    const long long dst = page * a.s_page + slot * a.s_tok + h * a.s_head;
    if (on) {
      *reinterpret_cast<uint4*>(a.vc + dst + 8 * c) = v0[u];
      *reinterpret_cast<uint4*>(a.vc + dst + 64 + 8 * c) = v1[u];
    }
    float x1[8], x2[8], w1[8], w2[8];
    normmath::unpack(k0[u], x1);
    normmath::unpack(k1[u], x2);
    normmath::load8(&s_w[8 * c], w1);
    normmath::load8(&s_w[64 + 8 * c], w2);
    normmath::normalise(x1, x2, w1, w2, a.eps, 0xffffffffu);
    uint32_t o[8];
    normmath::rotate(x1, x2, cv, sv, a.sorted != 0, o);
    if (on)
      normmath::store_pairs(a.kc + (a.k_lm ? page * a.k_s_page + h * a.k_s_head + slot * 16 : dst), c, a.sorted != 0,
                            lstride, o);
  }
}

}  // namespace append
}  // namespace atf

using namespace atf;

extern "C" int atf_paged_kv_append(const AtfAppendParams* p, atf_stream_t stream) {
  return append_bf16(p, nullptr, stream);
}

extern "C" int atf_paged_kv_append_norm(const AtfAppendParams* p, const AtfKvScales* s, const AtfKNorm* n,
                                        atf_stream_t stream) {
  if (n == nullptr) return ATF_ERR_INVALID_ARG;
  return s != nullptr ? append_e4m3(p, s, n, stream) : append_bf16(p, n, stream);
}

int atf::append_bf16(const AtfAppendParams* p, const AtfKNorm* norm, atf_stream_t stream) {
  if (p == nullptr || p->append_k == nullptr || p->append_v == nullptr || p->batch_indices == nullptr ||
      p->positions == nullptr || p->k_cache == nullptr || p->v_cache == nullptr ||
      p->kv_indptr == nullptr || p->kv_indices == nullptr)
    return ATF_ERR_INVALID_ARG;
  if (p->head_dim != ATF_HEAD_DIM) return ATF_ERR_UNSUPPORTED;
  if (p->nnz < 0 || p->num_kv_heads < 1 || p->page_size < 1 || p->batch_size < 1 || p->num_pages < 1)
    return ATF_ERR_INVALID_ARG;
  const bool rope = p->cos != nullptr;
  if (rope != (p->sin != nullptr)) return ATF_ERR_INVALID_ARG;
  if (rope && (p->n_pos < 1 || p->cs_stride_pos < 64)) return ATF_ERR_INVALID_ARG;
  if (p->out_layout != ATF_LAYOUT_SORTED_PAIR && p->out_layout != ATF_LAYOUT_ROTATE_HALF)
    return ATF_ERR_INVALID_ARG;
  if (p->k_level_major) {
    if (rope && p->out_layout != ATF_LAYOUT_SORTED_PAIR) return ATF_ERR_UNSUPPORTED;
    if ((p->k_stride_page & 7) || (p->k_stride_head & 7) || (p->k_stride_level & 7) ||
        p->k_stride_level < 16 * static_cast<int64_t>(p->page_size))
      return ATF_ERR_ALIGNMENT;
  }
  if (!aligned16(p->append_k) || !aligned16(p->append_v) || !aligned16(p->k_cache) ||
      !aligned16(p->v_cache) || (p->a_stride_n & 7) || (p->a_stride_h & 7) || (p->kv_stride_page & 7) ||
      (p->kv_stride_token & 7) || (p->kv_stride_head & 7))
    return ATF_ERR_ALIGNMENT;
  int rc = norm_args_ok(p, norm);
  if (rc != ATF_OK) return rc;
  const long long total = p->nnz * p->num_kv_heads * 8;
  if (total == 0) return ATF_OK;
  int dev = 0;
  rc = check_device(&dev);
  if (rc != ATF_OK) return rc;
  append::Args a;
  a.ak = static_cast<const __nv_bfloat16*>(p->append_k);
  a.av = static_cast<const __nv_bfloat16*>(p->append_v);
  a.nnz = p->nnz;
  a.as_n = p->a_stride_n;
  a.as_h = p->a_stride_h;
  a.batch_indices = p->batch_indices;
  a.positions = p->positions;
  a.kc = static_cast<__nv_bfloat16*>(p->k_cache);
  a.vc = static_cast<__nv_bfloat16*>(p->v_cache);
  a.num_pages = p->num_pages;
  a.s_page = p->kv_stride_page;
  a.s_tok = p->kv_stride_token;
  a.s_head = p->kv_stride_head;
  a.H = p->num_kv_heads;
  a.page_size = p->page_size;
  a.B = p->batch_size;
  a.kv_indptr = p->kv_indptr;
  a.kv_indices = p->kv_indices;
  a.cs = p->cos;
  a.sn = p->sin;
  a.cs_stride = p->cs_stride_pos;
  a.n_pos = p->n_pos;
  a.rope_pos = p->rope_positions;
  a.rope = rope ? 1 : 0;
  a.sorted = p->out_layout == ATF_LAYOUT_SORTED_PAIR ? 1 : 0;
  a.err = p->error_flag;
  a.k_lm = p->k_level_major ? 1 : 0;
  a.k_s_page = p->k_stride_page;
  a.k_s_head = p->k_stride_head;
  a.k_s_level = p->k_stride_level;
  const int threads = 256;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (norm != nullptr) {
    a.norm_w = norm->weight;
    a.norm_f32 = norm->weight_dtype == ATF_DTYPE_F32 ? 1 : 0;
    a.eps = norm->eps;
    const long long narrow = (a.H + 3) / 4;  // units of 4 heads a token
    if (a.nnz > (1ll << 30) / narrow) return ATF_ERR_UNSUPPORTED;
    // 8 rows per warp once that gives every SM two CTAs
    const bool many = a.nnz * ((a.H + 7) / 8) >= 2ll * 148 * 8;
    a.units = static_cast<unsigned>(many ? (a.H + 1) / 2 : narrow);
    const long long items = many ? (a.nnz + 3) / 4 : a.nnz;
    const unsigned blocks = static_cast<unsigned>((items * a.units + 7) / 8);
    if (many)
      append::append_norm_kernel<true><<<blocks, threads, 0, st>>>(a);
    else
      append::append_norm_kernel<false><<<blocks, threads, 0, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? ATF_OK : ATF_ERR_CUDA;
  }
  const long long blocks = (total + threads - 1) / threads;
  if (blocks > 0x7fffffffLL) return ATF_ERR_UNSUPPORTED;
  append::append_kernel<<<static_cast<unsigned>(blocks), threads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? ATF_OK : ATF_ERR_CUDA;
}
