// rkv_gqa_prefill.cu -- causal attention of packed new tokens over the
// grouped-head paged cache.
//
//   x_j = softmax_scale * q . k_j over the rows j that the token sees,
//   out = sum_j exp(x_j - m) v_j / (sum_j exp(x_j - m) + exp(sink - m)).
//
// One warp per (token, q head), one pass over the rows with the running
// maximum and sum; a lane holds head_dim / 32 lanes of q, k and v.
#include "rkv_gqa.cuh"

namespace rkv {
namespace gqa {

struct AttendParams {
  rkv_gqa_view cache;
  int layer;
  const uint16_t* q;
  int64_t q_ts, q_hs;
  int64_t n_tokens;
  int n_q_heads;
  const int32_t* cu_q;
  int n_seq;
  const int32_t* page_table;
  int64_t pt_stride;
  const int32_t* kv_lens;
  int window;
  const float* sinks;
  float scale_log2;
  uint16_t* out;
  uint32_t* status;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) attend_kernel(const AttendParams p) {
  constexpr int kWords = D / 64;  // words of two lanes each
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int64_t t = item / p.n_q_heads;
  const int h = (int)(item % p.n_q_heads);
  if (t >= p.n_tokens) return;
  int seq = 0, hi = p.n_seq;  // the last sequence that starts at or before t
  while (hi - seq > 1) {
    const int mid = (seq + hi) / 2;
    if (p.cu_q[mid] <= t) seq = mid;
    else hi = mid;
  }
  if (t < p.cu_q[seq] || t >= p.cu_q[seq + 1]) {
    if (lane == 0) set_status(p.status, RKV_ERR_INDEX_OUT_OF_RANGE);
    return;
  }
  const int q_len = p.cu_q[seq + 1] - p.cu_q[seq];
  const int i = (int)(t - p.cu_q[seq]);
  int64_t len = p.kv_lens[seq];
  if (len < 0 || len > p.pt_stride * kPage) {
    if (lane == 0) set_status(p.status, RKV_ERR_INDEX_OUT_OF_RANGE);
    len = len < 0 ? 0 : p.pt_stride * kPage;
  }
  const int64_t at = len - q_len + i;
  const int64_t first = p.window > 0 && at >= p.window ? at - p.window + 1 : 0;
  const int hkv = h / (p.n_q_heads / p.cache.n_kv_heads);
  const uint16_t* qp = p.q + t * p.q_ts + h * p.q_hs + lane * 2 * kWords;
  float2 q[kWords], acc[kWords];
#pragma unroll
  for (int w = 0; w < kWords; ++w) {
    q[w] = T::unpack(reinterpret_cast<const uint32_t*>(qp)[w]);
    acc[w] = make_float2(0.f, 0.f);
  }
  float m = p.sinks ? p.sinks[h] * 1.4426950408889634f : -INFINITY, l = p.sinks ? 1.0f : 0.0f;
  for (int64_t j = first; j <= at; ++j) {
    const int32_t page = p.page_table[seq * p.pt_stride + j / kPage];
    uint32_t k[kWords], v[kWords];
    if (page >= 0 && page < p.cache.n_pages) {
      const uint16_t* base = static_cast<const uint16_t*>(p.cache.base) + lane * 2 * kWords;
      const uint32_t* kp = reinterpret_cast<const uint32_t*>(base + (row_base(p.cache, p.layer, page, 0, hkv) + j % kPage) * D);
      const uint32_t* vp = reinterpret_cast<const uint32_t*>(base + (row_base(p.cache, p.layer, page, 1, hkv) + j % kPage) * D);
#pragma unroll
      for (int w = 0; w < kWords; ++w) k[w] = kp[w], v[w] = vp[w];
    } else {
      if (lane == 0) set_status(p.status, RKV_ERR_INDEX_OUT_OF_RANGE);
#pragma unroll
      for (int w = 0; w < kWords; ++w) k[w] = v[w] = 0u;
    }
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      const float2 f = T::unpack(k[w]);
      x += q[w].x * f.x + q[w].y * f.y;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    x *= p.scale_log2;
    const float top = fmaxf(m, x);
    const float old = m == -INFINITY ? 0.f : ex2(m - top), e = ex2(x - top);
    m = top;
    l = l * old + e;
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      const float2 f = T::unpack(v[w]);
      acc[w] = make_float2(acc[w].x * old + e * f.x, acc[w].y * old + e * f.y);
    }
  }
  const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
  uint32_t* op = reinterpret_cast<uint32_t*>(p.out + (t * p.n_q_heads + h) * D + lane * 2 * kWords);
#pragma unroll
  for (int w = 0; w < kWords; ++w) op[w] = T::pack(acc[w].x * inv, acc[w].y * inv);
}

static rkv_status attend(const AttendParams& p, const char* what, cudaStream_t s) {
  const int64_t blocks = (p.n_tokens * p.n_q_heads + 3) / 4;
  if (blocks > INT32_MAX) return fail(RKV_ERR_SHAPE_MISMATCH, "%s: too many tokens", what);
  if (p.cache.dtype == RKV_GQA_BF16) {
    if (p.cache.head_dim == 64) attend_kernel<Bf16, 64><<<(unsigned)blocks, 128, 0, s>>>(p);
    else attend_kernel<Bf16, 128><<<(unsigned)blocks, 128, 0, s>>>(p);
  } else {
    if (p.cache.head_dim == 64) attend_kernel<F16, 64><<<(unsigned)blocks, 128, 0, s>>>(p);
    else attend_kernel<F16, 128><<<(unsigned)blocks, 128, 0, s>>>(p);
  }
  return check_launch(what);
}

}  // namespace gqa
}  // namespace rkv

extern "C" int32_t rkv_gqa_prefill_splits(const rkv_gqa_view* cache, int64_t n_tokens, int32_t n_q_heads,
                                          int32_t n_seq, int64_t pt_stride) {
  if (!cache || n_tokens < 0 || n_q_heads < 1 || n_seq < 0 || pt_stride < 1) return -1;
  return 1;
}

extern "C" int64_t rkv_gqa_prefill_workspace_bytes(const rkv_gqa_view* cache, int64_t n_tokens, int32_t n_q_heads,
                                                   int32_t n_splits) {
  if (!cache || n_tokens < 0 || n_q_heads < 1 || n_splits < 1) return -1;
  return 0;
}

extern "C" rkv_status rkv_gqa_prefill(const rkv_gqa_view* cache, int32_t layer, const void* q, int64_t q_token_stride,
                                      int64_t q_head_stride, int64_t n_tokens, int32_t n_q_heads, const int32_t* cu_q,
                                      int32_t n_seq, const int32_t* page_table, int64_t pt_stride,
                                      const int32_t* kv_lens, int32_t window, const float* sinks, float softmax_scale,
                                      int32_t n_splits, void* workspace, void* out, uint32_t* d_status,
                                      rkv_stream_t stream) {
  using namespace rkv;
  using namespace rkv::gqa;
  static const char* what = "rkv_gqa_prefill";
  rkv_status st = check_cache(cache, layer, what);
  if (st != RKV_OK) return st;
  if ((st = check_heads(cache, n_q_heads, what)) != RKV_OK) return st;
  if (n_tokens < 0 || n_tokens > INT32_MAX) return fail_shape("n_tokens", 0, n_tokens, "%s: bad n_tokens", what);
  if (n_seq < 0) return fail_shape("n_seq", 0, n_seq, "%s: n_seq < 0", what);
  if (n_splits < 1 || n_splits > 64) return fail_shape("n_splits", 1, n_splits, "%s: 1 <= n_splits <= 64", what);
  if (n_tokens == 0 || n_seq == 0) {
    if (n_tokens > 0) return fail_shape("n_tokens", 0, n_tokens, "%s: tokens without a sequence", what);
    clear_error();
    return RKV_OK;
  }
  const AttendArgs args = {*cache,     layer,   q,      q_token_stride, q_head_stride, n_tokens, n_q_heads, page_table,
                           pt_stride,  kv_lens, window, sinks,          softmax_scale, out,      d_status};
  st = check_attend(args, what);
  if (st != RKV_OK) return st;
  if (!cu_q) return fail(RKV_ERR_INVALID_ARGUMENT, "%s: cu_q is required", what);
  const AttendParams p = {*cache,    layer,      static_cast<const uint16_t*>(q),
                          q_token_stride, q_head_stride, n_tokens,
                          n_q_heads, cu_q,       n_seq,
                          page_table, pt_stride, kv_lens,
                          window,    sinks,      (float)((double)softmax_scale * 1.4426950408889634),
                          static_cast<uint16_t*>(out), d_status};
  return attend(p, what, (cudaStream_t)stream);
}
