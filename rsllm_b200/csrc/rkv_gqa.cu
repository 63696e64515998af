// rkv_gqa.cu -- the grouped-head cache's host checks and its two data
// movers: rotary append (k, v into their pages, q rotated beside them) and
// whole-page copies.
#include "rkv_gqa.cuh"

#include <cmath>

namespace rkv {
namespace gqa {

rkv_status check_cache(const rkv_gqa_view* c, int32_t layer, const char* what) {
  if (!c) return fail(RKV_ERR_INVALID_ARGUMENT, "%s: cache view is NULL", what);
  if (!c->base || !aligned(c->base, 256))
    return fail(RKV_ERR_INVALID_ARGUMENT, "%s: cache base must be a non-null 256-byte aligned device pointer", what);
  if (c->n_pages <= 0 || c->n_layers <= 0 || c->n_kv_heads <= 0)
    return fail(RKV_ERR_INVALID_ARGUMENT, "%s: cache needs n_pages > 0, n_layers > 0, n_kv_heads > 0", what);
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail_shape("head_dim", 128, c->head_dim, "%s: head_dim must be 64 or 128, got %d", what, c->head_dim);
  if (c->dtype != RKV_GQA_BF16 && c->dtype != RKV_GQA_F16)
    return fail(RKV_ERR_INVALID_ARGUMENT, "%s: dtype must be RKV_GQA_BF16 or RKV_GQA_F16", what);
  // slots are int32, and so are the row coordinates of the tensor maps
  if (c->n_pages > (int64_t)(INT32_MAX / kPage) ||
      c->n_pages > INT32_MAX / ((int64_t)2 * kPage * c->n_kv_heads) / c->n_layers)
    return fail(RKV_ERR_INVALID_ARGUMENT, "%s: n_layers * n_pages * 2 * n_kv_heads * 64 must fit in int32", what);
  if (layer < 0 || layer >= c->n_layers)
    return fail_layer(layer, c->n_layers, "%s: layer %d outside cache of %d layers", what, layer, c->n_layers);
  return RKV_OK;
}

rkv_status check_rows(const void* p, int64_t token_stride, int64_t head_stride, const char* name, const char* what) {
  if (!p || !aligned(p, 16))
    return fail(RKV_ERR_INVALID_ARGUMENT, "%s: %s must be a non-null 16-byte aligned device pointer", what, name);
  if (token_stride < 0 || head_stride < 0 || token_stride % 8 != 0 || head_stride % 8 != 0)
    return fail(RKV_ERR_SHAPE_MISMATCH, "%s: strides of %s must be non-negative multiples of 8 elements", what, name);
  return RKV_OK;
}

rkv_status check_heads(const rkv_gqa_view* c, int32_t n_q_heads, const char* what) {
  if (n_q_heads <= 0 || n_q_heads % c->n_kv_heads != 0 || n_q_heads / c->n_kv_heads > RKV_GQA_MAX_GROUP)
    return fail_shape("n_q_heads", c->n_kv_heads, n_q_heads,
                      "%s: n_q_heads must be a multiple of the %d kv heads, at most %d times as many; got %d", what,
                      c->n_kv_heads, RKV_GQA_MAX_GROUP, n_q_heads);
  return RKV_OK;
}

rkv_status check_attend(const AttendArgs& a, const char* what) {
  rkv_status st = check_rows(a.q, a.q_ts, a.q_hs, "q", what);
  if (st != RKV_OK) return st;
  if (a.pt_stride < 1 || a.pt_stride > INT32_MAX / kPage)
    return fail_shape("pt_stride", 1, a.pt_stride, "%s: pt_stride must be at least 1 and pt_stride * 64 fit in int32", what);
  if (a.window < 0) return fail_shape("window", 0, a.window, "%s: window must not be negative", what);
  if (!(a.scale > 0.f) || !std::isfinite(a.scale))
    return fail(RKV_ERR_INVALID_ARGUMENT, "%s: softmax_scale must be finite and positive", what);
  if (!a.page_table || !a.kv_lens || !a.out || !aligned(a.out, 16))
    return fail(RKV_ERR_INVALID_ARGUMENT, "%s: page_table, kv_lens and a 16-byte aligned out are required", what);
  return RKV_OK;
}

// ---- tensor maps ---------------------------------------------------------------------
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder, looked up once (the library does not link the driver).
static EncodeTiled encoder() {
  static EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

static rkv_status encode(const rkv_gqa_view& c, const void* base, int rank, const cuuint64_t* dims,
                         const cuuint64_t* strides, const cuuint32_t* box, CUtensorMap* out, const char* what) {
  const EncodeTiled fn = encoder();
  if (!fn) return fail(RKV_ERR_CUDA, "%s: the driver has no cuTensorMapEncodeTiled", what);
  const cuuint32_t step[3] = {1, 1, 1};
  const CUresult r = fn(out, c.dtype == RKV_GQA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                        rank, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(RKV_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
  return RKV_OK;
}

rkv_status cache_map(const rkv_gqa_view& c, CUtensorMap* out, const char* what) {
  const cuuint64_t dims[2] = {(cuuint64_t)c.head_dim, (cuuint64_t)row_base(c, c.n_layers, 0, 0, 0)};
  const cuuint64_t strides[1] = {(cuuint64_t)c.head_dim * 2};
  const cuuint32_t box[2] = {64, kPage};
  return encode(c, c.base, 2, dims, strides, box, out, what);
}

rkv_status q_map(const rkv_gqa_view& c, const void* q, int64_t token_stride, int64_t head_stride, int64_t n_tokens,
                 int32_t n_heads, int box_tokens, int box_heads, CUtensorMap* out, const char* what) {
  const cuuint64_t dims[3] = {(cuuint64_t)c.head_dim, (cuuint64_t)n_heads, (cuuint64_t)n_tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)token_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
  return encode(c, q, 3, dims, strides, box, out, what);
}

// ---- rotary append ---------------------------------------------------------------
struct AppendParams {
  rkv_gqa_view cache;
  int layer;
  const uint16_t *k, *v, *q;
  int64_t k_ts, k_hs, v_ts, v_hs, q_ts, q_hs;
  int64_t n_tokens;
  const int32_t* slots;
  const int32_t* pos;
  const float* table;
  int64_t table_rows;
  int rot;          // 0: no rotation
  int edge[3];      // first pair of axes 1, 2, 3
  int n_q_heads;
  uint16_t* q_out;
  uint32_t* status;
};

// One CTA per token.  A work item is 16 lanes of one head's row: with
// rotation, the 8 + 8 lanes that eight pairs need (two 16-byte chunks half a
// rotary width apart, or 16 lanes in a row when interleaved), else 16 lanes in
// a row.  Items of q come first, then k, then v.
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(128) append_kernel(const AppendParams p) {
  const int64_t t = blockIdx.x;
  const int d = p.cache.head_dim, per_row = d / 16, hkv = p.cache.n_kv_heads;
  const int slot = p.slots[t];
  bool store = slot >= 0, bad_pos = false;
  if (store && slot >= p.cache.n_pages * kPage) {
    store = false;
    if (threadIdx.x == 0) set_status(p.status, RKV_ERR_INDEX_OUT_OF_RANGE);
  }
  int32_t pos[4] = {0, 0, 0, 0};
  if (p.rot) {
    const int axes = 1 + (p.edge[0] < p.rot / 2) + (p.edge[1] < p.rot / 2) + (p.edge[2] < p.rot / 2);
#pragma unroll
    for (int a = 0; a < 4; ++a)
      if (a < axes) {
        pos[a] = p.pos[(int64_t)a * p.n_tokens + t];
        bad_pos |= pos[a] < 0 || pos[a] >= p.table_rows;
      }
    if (bad_pos) {
      store = false;
      if (threadIdx.x == 0) set_status(p.status, RKV_ERR_INDEX_OUT_OF_RANGE);
    }
  }
  const int64_t page = store ? slot / kPage : 0;
  const int row = store ? slot % kPage : 0;
  const int heads = p.n_q_heads + 2 * hkv;
  // the items of a row are 4 or 8 consecutive lanes of one warp
  for (int item = threadIdx.x; item < (heads * per_row + 31) / 32 * 32; item += blockDim.x) {
    const int h = item / per_row, c = item % per_row;
    const bool live = h < heads;
    const bool is_q = h < p.n_q_heads, is_v = h >= p.n_q_heads + hkv;
    const int head = is_q ? h : is_v ? h - p.n_q_heads - hkv : h - p.n_q_heads;
    const uint16_t* src = is_q ? p.q + t * p.q_ts + head * p.q_hs
                          : is_v ? p.v + t * p.v_ts + head * p.v_hs
                                 : p.k + t * p.k_ts + head * p.k_hs;
    // first lanes of the two chunks
    const bool turn = p.rot > 0 && !is_v && 16 * c < p.rot;
    const int a = turn && !kInterleaved ? 8 * c : 16 * c;
    const int b = turn && !kInterleaved ? a + p.rot / 2 : a + 8;
    uint32_t x[4] = {0, 0, 0, 0}, y[4] = {0, 0, 0, 0};
    const bool read = live && (is_q || store);
    if (read) {
      *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(src + a);
      *reinterpret_cast<uint4*>(y) = *reinterpret_cast<const uint4*>(src + b);
    }
    if (read && turn && !bad_pos) {
      float2 u[4], w[4];  // the pairs' first and second members, two pairs an entry
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (kInterleaved) {  // word i of x is pair i, word i of y pair 4 + i
          const float2 e = T::unpack(x[i]), f = T::unpack(y[i]);
          u[i] = make_float2(e.x, f.x);
          w[i] = make_float2(e.y, f.y);
        } else {
          u[i] = T::unpack(x[i]);
          w[i] = T::unpack(y[i]);
        }
      }
      float2 ru[4], rw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p0 = 8 * c + (kInterleaved ? i : 2 * i), p1 = 8 * c + (kInterleaved ? 4 + i : 2 * i + 1);
        auto cs = [&](int pair) {
          const int axis = (pair >= p.edge[0]) + (pair >= p.edge[1]) + (pair >= p.edge[2]);
          const int32_t at = axis == 0 ? pos[0] : axis == 1 ? pos[1] : axis == 2 ? pos[2] : pos[3];
          return __ldg(reinterpret_cast<const float2*>(p.table) + (int64_t)at * (p.rot / 2) + pair);
        };
        const float2 c0 = cs(p0), c1 = cs(p1);
        ru[i] = make_float2(u[i].x * c0.x - w[i].x * c0.y, u[i].y * c1.x - w[i].y * c1.y);
        rw[i] = make_float2(w[i].x * c0.x + u[i].x * c0.y, w[i].y * c1.x + u[i].y * c1.y);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = kInterleaved ? T::pack(ru[i].x, rw[i].x) : T::pack(ru[i].x, ru[i].y);
        y[i] = kInterleaved ? T::pack(ru[i].y, rw[i].y) : T::pack(rw[i].x, rw[i].y);
      }
    }
    // a K or V row is refused as a whole: its lanes vote
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= not_finite<T>(x[i]) || not_finite<T>(y[i]);
    const unsigned votes = __ballot_sync(0xffffffffu, bad && read && !is_q);
    const int first = (threadIdx.x & 31) / per_row * per_row;
    const bool refused = ((votes >> first) & ((1u << per_row) - 1u)) != 0u;
    uint16_t* dst;
    bool write = live;
    if (is_q) {
      dst = p.q_out + (t * p.n_q_heads + head) * d;
      if (bad_pos)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = y[i] = 0u;
    } else {
      dst = static_cast<uint16_t*>(p.cache.base) + (row_base(p.cache, p.layer, page, is_v, live ? head : 0) + row) * d;
      write = live && store && !refused;
      if (refused && live) set_status(p.status, RKV_ERR_NON_FINITE_INPUT);
    }
    if (write) {
      *reinterpret_cast<uint4*>(dst + a) = make_uint4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<uint4*>(dst + b) = make_uint4(y[0], y[1], y[2], y[3]);
    }
  }
}

// ---- page copies ---------------------------------------------------------------------
constexpr int kCopyThreads = 256;
constexpr int kCopyChunk = kCopyThreads * 4 * 16;  // 16 KB: four 16-byte vectors a thread, loads before stores

// One CTA per (pair, layer, 16 KB of the page); pages are multiples of 16 KB.
__global__ void __launch_bounds__(kCopyThreads)
copy_kernel(rkv_gqa_view c, int64_t page_bytes, int chunks, const int32_t* __restrict__ src,
            const int32_t* __restrict__ dst, uint32_t* __restrict__ status) {
  const int64_t i = blockIdx.x / chunks;
  const int chunk = blockIdx.x % chunks;
  const int32_t s = __ldg(src + i), d = __ldg(dst + i);
  if (s < 0 || s >= c.n_pages || d < 0 || d >= c.n_pages) {
    if (threadIdx.x == 0 && blockIdx.y == 0) set_status(status, RKV_ERR_INDEX_OUT_OF_RANGE);
    return;
  }
  uint8_t* base = static_cast<uint8_t*>(c.base) + (int64_t)blockIdx.y * c.n_pages * page_bytes +
                  (int64_t)chunk * kCopyChunk;
  const uint4* sp = reinterpret_cast<const uint4*>(base + s * page_bytes) + threadIdx.x;
  uint4* dp = reinterpret_cast<uint4*>(base + d * page_bytes) + threadIdx.x;
  uint4 v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = ld_stream16(sp + j * kCopyThreads);
#pragma unroll
  for (int j = 0; j < 4; ++j) st_stream16(dp + j * kCopyThreads, v[j]);
}

}  // namespace gqa
}  // namespace rkv

extern "C" int64_t rkv_gqa_page_bytes(int32_t n_kv_heads, int32_t head_dim) {
  if (n_kv_heads <= 0 || (head_dim != 64 && head_dim != 128)) return -1;
  return (int64_t)2 * n_kv_heads * RKV_PAGE_TOKENS * head_dim * 2;
}

extern "C" int64_t rkv_gqa_bytes(const rkv_gqa_view* c) {
  if (!c || c->n_pages < 0 || c->n_layers < 0) return -1;
  const int64_t page = rkv_gqa_page_bytes(c->n_kv_heads, c->head_dim);
  return page < 0 ? -1 : c->n_pages * c->n_layers * page;
}

extern "C" rkv_status rkv_gqa_append(const rkv_gqa_view* cache, int32_t layer, const void* k, int64_t k_token_stride,
                                     int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                     int64_t v_head_stride, int64_t n_tokens, const int32_t* slot_mapping,
                                     const rkv_gqa_rotary* rotary, const int32_t* pos, const void* q,
                                     int64_t q_token_stride, int64_t q_head_stride, int32_t n_q_heads, void* q_out,
                                     uint32_t* d_status, rkv_stream_t stream) {
  using namespace rkv;
  using namespace rkv::gqa;
  static const char* what = "rkv_gqa_append";
  rkv_status st = check_cache(cache, layer, what);
  if (st != RKV_OK) return st;
  if (n_tokens < 0 || n_tokens > INT32_MAX) return fail_shape("n_tokens", 0, n_tokens, "%s: bad n_tokens", what);
  AppendParams p = {};
  if (rotary) {
    if (rotary->rot_dim <= 0 || rotary->rot_dim % 16 != 0 || rotary->rot_dim > cache->head_dim)
      return fail_shape("rot_dim", cache->head_dim, rotary->rot_dim,
                        "%s: rot_dim must be a positive multiple of 16, at most head_dim", what);
    if (rotary->n_axes < 1 || rotary->n_axes > 4)
      return fail_shape("n_axes", 4, rotary->n_axes, "%s: 1 to 4 position axes", what);
    if (rotary->interleaved != 0 && rotary->interleaved != 1)
      return fail(RKV_ERR_INVALID_ARGUMENT, "%s: interleaved must be 0 or 1", what);
    int64_t sum = 0;
    for (int a = 0; a < rotary->n_axes; ++a) {
      // an axis without pairs would leave its positions unread
      if (rotary->section[a] <= 0) return fail(RKV_ERR_SHAPE_MISMATCH, "%s: sections must be positive", what);
      sum += rotary->section[a];
      if (a < 3) p.edge[a] = (int)sum;
    }
    for (int a = rotary->n_axes - 1; a < 3; ++a) p.edge[a] = rotary->rot_dim / 2;
    if (sum != rotary->rot_dim / 2)
      return fail_shape("section", rotary->rot_dim / 2, sum, "%s: sections must add up to rot_dim / 2", what);
    if (!rotary->table || !aligned(rotary->table, 16) || rotary->table_rows < 1)
      return fail(RKV_ERR_INVALID_ARGUMENT, "%s: a 16-byte aligned rotary table of at least one row is required", what);
    p.table = rotary->table;
    p.table_rows = rotary->table_rows;
    p.rot = rotary->rot_dim;
  } else if (q) {
    return fail(RKV_ERR_INVALID_ARGUMENT, "%s: q is only taken with a rotary table", what);
  }
  if (q && (st = check_heads(cache, n_q_heads, what)) != RKV_OK) return st;
  if (n_tokens == 0) {
    clear_error();
    return RKV_OK;
  }
  if ((st = check_rows(k, k_token_stride, k_head_stride, "k", what)) != RKV_OK) return st;
  if ((st = check_rows(v, v_token_stride, v_head_stride, "v", what)) != RKV_OK) return st;
  if (q && (st = check_rows(q, q_token_stride, q_head_stride, "q", what)) != RKV_OK) return st;
  if (!slot_mapping || (rotary && !pos) || (q && (!q_out || !aligned(q_out, 16))))
    return fail(RKV_ERR_INVALID_ARGUMENT, "%s: slot_mapping, with rotary pos, and with q a 16-byte aligned q_out are "
                "required", what);
  p.cache = *cache;
  p.layer = layer;
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.q = static_cast<const uint16_t*>(q);
  p.k_ts = k_token_stride, p.k_hs = k_head_stride;
  p.v_ts = v_token_stride, p.v_hs = v_head_stride;
  p.q_ts = q_token_stride, p.q_hs = q_head_stride;
  p.n_tokens = n_tokens;
  p.slots = slot_mapping;
  p.pos = pos;
  p.n_q_heads = q ? n_q_heads : 0;
  p.q_out = static_cast<uint16_t*>(q_out);
  p.status = d_status;
  cudaStream_t s = (cudaStream_t)stream;
  const unsigned grid = (unsigned)n_tokens;
  const bool inter = rotary && rotary->interleaved;
  if (cache->dtype == RKV_GQA_BF16) {
    if (inter) append_kernel<Bf16, true><<<grid, 128, 0, s>>>(p);
    else append_kernel<Bf16, false><<<grid, 128, 0, s>>>(p);
  } else {
    if (inter) append_kernel<F16, true><<<grid, 128, 0, s>>>(p);
    else append_kernel<F16, false><<<grid, 128, 0, s>>>(p);
  }
  return check_launch(what);
}

extern "C" rkv_status rkv_gqa_copy_pages(const rkv_gqa_view* cache, const int32_t* src, const int32_t* dst, int64_t n,
                                         uint32_t* d_status, rkv_stream_t stream) {
  using namespace rkv;
  using namespace rkv::gqa;
  static const char* what = "rkv_gqa_copy_pages";
  rkv_status st = check_cache(cache, 0, what);
  if (st != RKV_OK) return st;
  if (n < 0) return fail_shape("n", 0, n, "%s: n < 0", what);
  if (n == 0) {
    clear_error();
    return RKV_OK;
  }
  if (!src || !dst) return fail(RKV_ERR_INVALID_ARGUMENT, "%s: src and dst are required", what);
  const int64_t page = rkv_gqa_page_bytes(cache->n_kv_heads, cache->head_dim);
  const int64_t chunks = page / kCopyChunk;
  if (cache->n_layers > 65535 || n > INT32_MAX / chunks)
    return fail(RKV_ERR_SHAPE_MISMATCH, "%s: too many pages", what);
  copy_kernel<<<dim3((unsigned)(n * chunks), (unsigned)cache->n_layers), kCopyThreads, 0, (cudaStream_t)stream>>>(
      *cache, page, (int)chunks, src, dst, d_status);
  return check_launch(what);
}
