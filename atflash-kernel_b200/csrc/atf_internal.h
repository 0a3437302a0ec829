// Host-side helpers shared by the C-ABI translation units.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "../../include/atflash_b200.h"

namespace atf {

// Error code a bounded device wait writes to the caller's error flag.
constexpr int kDevErrTimeout = 1;
// Error code for indices out of range: lengths, pages, rows or items of a call that its
// kernel reports and leaves out.
constexpr int kDevErrIndex = 2;

// Encodes a tiled TMA descriptor through the driver entry point (loaded once).
// dims / strides are innermost first; strides are in bytes for dims 1..rank-1.
int encode_tiled_bf16(CUtensorMap* map, const void* base, int rank, const uint64_t* dims,
                      const uint64_t* strides_bytes, const uint32_t* box,
                      CUtensorMapSwizzle swizzle,
                      CUtensorMapL2promotion promotion = CU_TENSOR_MAP_L2_PROMOTION_L2_256B);

// The same over bytes (e4m3 caches).
int encode_tiled_u8(CUtensorMap* map, const void* base, int rank, const uint64_t* dims,
                    const uint64_t* strides_bytes, const uint32_t* box,
                    CUtensorMapSwizzle swizzle, CUtensorMapL2promotion promotion);

// True when the current device is an sm_100 part.
int check_device(int* device_out);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// The K norm of an append (optional): it stands before a rotation, and its weights are
// read 16 bytes at a time.
inline int norm_args_ok(const AtfAppendParams* p, const AtfKNorm* n) {
  if (n == nullptr) return ATF_OK;
  if (n->weight == nullptr || p->cos == nullptr || !(n->eps > 0.f && n->eps <= FLT_MAX) ||
      (n->weight_dtype != ATF_DTYPE_BF16 && n->weight_dtype != ATF_DTYPE_F32))
    return ATF_ERR_INVALID_ARG;
  if (!aligned16(n->weight) || !aligned16(p->cos) || !aligned16(p->sin) || (p->cs_stride_pos & 3) != 0)
    return ATF_ERR_ALIGNMENT;
  return ATF_OK;
}

// The appends, with an optional norm of K (append.cu, append_e4m3.cu)
int append_bf16(const AtfAppendParams* p, const AtfKNorm* norm, atf_stream_t stream);
int append_e4m3(const AtfAppendParams* p, const AtfKvScales* s, const AtfKNorm* norm, atf_stream_t stream);

// atf_decode_run's checks and its split-KV kernel launch, without the merge
// (decode.cu); atf_decode_run and atf_decode_run_exchange add their merges.
int decode_launch_split(const AtfDecodeParams* p, cudaStream_t st);

namespace decode8 {
// atf_decode_plan's cut into units, on checked parameters (decode_e4m3.cu).
int plan_units(const AtfDecodePlanParams* p, long long slots, int32_t* items_host, int32_t items_capacity,
               int32_t* item_indptr_host, AtfDecodePlan* out);
}  // namespace decode8

}  // namespace atf
