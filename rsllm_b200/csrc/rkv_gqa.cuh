// rkv_gqa.cuh -- layout of the grouped-head (GQA) paged cache and what its
// kernels share: element types, page addressing, host checks.
//
// The cache is [n_layers][n_pages][2 (K, V)][n_kv_heads][64 rows][head_dim]:
// the 64 rows of one kv head in a page are contiguous (8 or 16 KB), which is
// the unit every kernel moves -- one tensor-map box per 64 lanes of it.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "rkv_common.cuh"
#include "rkv_host.h"

namespace rkv {
namespace gqa {

constexpr int kPage = RKV_PAGE_TOKENS;

// Row index (in rows of head_dim elements) of row 0 of (layer, page, K or V, head).
__host__ __device__ __forceinline__ int64_t row_base(const rkv_gqa_view& c, int layer, int64_t page, int which,
                                                     int head) {
  return ((((int64_t)layer * c.n_pages + page) * 2 + which) * c.n_kv_heads + head) * kPage;
}

// The two element types: conversions to and from f32.
struct Bf16 {
  static constexpr int kCode = RKV_GQA_BF16;
  static constexpr uint32_t kExpMask = 0x7f80u;  // all ones: infinity or NaN
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};
struct F16 {
  static constexpr int kCode = RKV_GQA_F16;
  static constexpr uint32_t kExpMask = 0x7c00u;
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};

// Whether a word of two elements holds an infinity or a NaN.
template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  return (w & T::kExpMask) == T::kExpMask || ((w >> 16) & T::kExpMask) == T::kExpMask;
}

// ---- host checks (rkv_gqa.cu) -------------------------------------------------
// Validates a view and a layer index.
rkv_status check_cache(const rkv_gqa_view* c, int32_t layer, const char* what);
// Validates a strided [tokens][heads][head_dim] operand.
rkv_status check_rows(const void* p, int64_t token_stride, int64_t head_stride, const char* name, const char* what);
// Validates the head counts: a group of 1 to RKV_GQA_MAX_GROUP q heads per kv head.
rkv_status check_heads(const rkv_gqa_view* c, int32_t n_q_heads, const char* what);

}  // namespace gqa
}  // namespace rkv
