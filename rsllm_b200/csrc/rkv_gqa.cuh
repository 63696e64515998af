// rkv_gqa.cuh -- layout of the grouped-head (GQA) paged cache and what its
// kernels share: element types, page addressing, host checks.
//
// The cache is [n_layers][n_pages][2 (K, V)][n_kv_heads][64 rows][head_dim]:
// the 64 rows of one kv head in a page are contiguous (8 or 16 KB), which is
// the unit every kernel moves -- one tensor-map box per 64 lanes of it.
#pragma once
#include <cuda.h>
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

// ---- device helpers of the two attention kernels ---------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
constexpr uint64_t kWaitNs = 1000000000ull;
// Bounded wait (1 s) for the phase of the given parity; false on a timeout, or
// as soon as another thread of the CTA gave up.
__device__ __forceinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  const uint64_t t0 = now_ns();
  while (!mbar_test(bar, parity)) {
    if (*abort_flag) return false;
    if (now_ns() - t0 > kWaitNs) return false;
  }
  return true;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_test(bar, parity)) return true;
  return mbar_wait_slow(bar, parity, abort_flag);
}
// The same for copies in flight: it ignores the abort flag, so that a CTA
// never ends while one still writes into its shared memory.
__device__ __forceinline__ bool mbar_wait_copy(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = now_ns();
  while (!mbar_test(bar, parity))
    if (now_ns() - t0 > kWaitNs) return false;
  return true;
}
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// One box of a 2-d tensor map into shared memory (no multicast).
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;"); }

// The exponent reference m of a running softmax only moves when a maximum
// exceeds it by kLazyLog2, so that sums and outputs are seldom rescaled; weights
// then reach 2^kLazyLog2 above 1.  For f16 weights the reference is put kBias
// below the maximum as well: their largest is 2^15, and a weight keeps its 11
// bits down to 2^-21 of the maximum instead of 2^-14.
constexpr float kLazyLog2 = 8.0f;
template <typename T>
struct SoftmaxBias {
  static constexpr float kBias = T::kCode == RKV_GQA_F16 ? 7.0f : 0.0f;
};

// ---- host helpers (rkv_gqa.cu) ------------------------------------------------------
// The whole cache as a 2-d tensor map, [rows of 64 of every (layer, page, K or
// V, head)][head_dim], box 64 lanes x 64 rows (8 KB), 128-byte swizzle.
rkv_status cache_map(const rkv_gqa_view& c, CUtensorMap* out, const char* what);
// A q operand as a 3-d map [tokens][heads][head_dim], box 64 lanes x `heads` x `tokens`.
rkv_status q_map(const rkv_gqa_view& c, const void* q, int64_t token_stride, int64_t head_stride, int64_t n_tokens,
                 int32_t n_heads, int box_tokens, int box_heads, CUtensorMap* out, const char* what);

// What an attention launch gets, checked.
struct AttendArgs {
  rkv_gqa_view cache;
  int32_t layer;
  const void* q;
  int64_t q_ts, q_hs;
  int64_t n_tokens;
  int32_t n_q_heads;
  const int32_t* page_table;
  int64_t pt_stride;
  const int32_t* kv_lens;
  int32_t window;
  const float* sinks;
  float scale;
  void* out;
  uint32_t* status;
};
// Validates what both attentions take (n_tokens > 0).
rkv_status check_attend(const AttendArgs& a, const char* what);

// ---- host checks (rkv_gqa.cu) -------------------------------------------------
// Validates a view and a layer index.
rkv_status check_cache(const rkv_gqa_view* c, int32_t layer, const char* what);
// Validates a strided [tokens][heads][head_dim] operand.
rkv_status check_rows(const void* p, int64_t token_stride, int64_t head_stride, const char* name, const char* what);
// Validates the head counts: a group of 1 to RKV_GQA_MAX_GROUP q heads per kv head.
rkv_status check_heads(const rkv_gqa_view* c, int32_t n_q_heads, const char* what);

}  // namespace gqa
}  // namespace rkv
