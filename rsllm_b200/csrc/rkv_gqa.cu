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

// A CTA takes one token after another, and of each kHeads heads (blockIdx.y says
// which; those of q come first, then k, then v).  A thread has the 16 lanes of chunk
// c of kAhead heads: with rotation, the 8 + 8 lanes that eight pairs need (two
// 16-byte chunks half a rotary width apart, or 16 lanes in a row when
// interleaved), else 16 lanes in a row; so it loads its eight cosines and sines once
// for all of them, and what depends on its heads it works out once for all tokens.
//
// Bytes bound it -- every row once in and once out -- if the instructions are few
// and the bytes on their way many: a token's slot and positions are loaded while
// the one before is worked on, so that its rows and its cosines and sines are
// one trip to memory together.  20011 tokens of 28 + 4 + 4 heads of 128, three
// axes, f16: 76 us, 4.95 TB/s (101 to 133 us where every thread worked out its heads
// and the axes of its pairs for every token: 67 instead of 41 million instructions).
// Heads a thread x CTAs an SM: 3 x 4 and 3 x 5 76 us, 3 x 6 82 (spills), 2 x 8 99,
// 4 x 4 80, 1 x 12 118.  Where a token's heads fill fewer of a CTA's chunks, less is
// on its way: 20000 tokens of 32 + 8 + 8 heads of 128 reach 5.9 TB/s, of 28 + 4 + 4
// heads of 64 3.4, of 14 + 2 + 2 of 64 2.2.
constexpr int kAppendThreads = 128, kAhead = 3, kAppendCtas = 4;
template <int D>
struct AppendShape {
  static constexpr int kPerRow = D / 16;                    // threads of a row: lanes of one warp
  static constexpr int kStep = kAppendThreads / kPerRow;    // heads at a time
  static constexpr int kHeads = kAhead * kStep;             // heads of a CTA: 48 (head_dim 128) or 96
};
template <typename T, int D, bool kInterleaved>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas) append_kernel(const AppendParams p) {
  using A = AppendShape<D>;
  const int c = threadIdx.x % A::kPerRow, hkv = p.cache.n_kv_heads, heads = p.n_q_heads + 2 * hkv;
  const int half = p.rot / 2;
  // ---- per thread: where its chunk lies, and its heads
  const bool turned = 16 * c < p.rot;  // rotated in q and k
  const int a1 = turned && !kInterleaved ? 8 * c : 16 * c, b1 = turned && !kInterleaved ? a1 + half : a1 + 8;
  const int axes = p.rot ? 1 + (p.edge[0] < half) + (p.edge[1] < half) + (p.edge[2] < half) : 0;
  auto axis_of = [&](int pair) { return (pair >= p.edge[0]) + (pair >= p.edge[1]) + (pair >= p.edge[2]); };
  const int axis0 = axis_of(8 * c), axis7 = axis_of(8 * c + 7);  // mostly the same
  const float2* const table = reinterpret_cast<const float2*>(p.table) + 8 * c;
  enum { kQ, kK, kV, kNone };
  int kind[kAhead];
  const uint16_t* src[kAhead];  // of token 0
  int64_t src_ts[kAhead];
  int64_t dst_at[kAhead];       // elements from the token's row in q_out, or from its page and row in the cache
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const int h = blockIdx.y * A::kHeads + k * A::kStep + threadIdx.x / A::kPerRow;
    kind[k] = h < p.n_q_heads ? kQ : h < p.n_q_heads + hkv ? kK : h < heads ? kV : kNone;
    const int head = kind[k] == kQ ? h : kind[k] == kK ? h - p.n_q_heads : h - p.n_q_heads - hkv;
    src[k] = kind[k] == kQ ? p.q + head * p.q_hs : kind[k] == kK ? p.k + head * p.k_hs : p.v + head * p.v_hs;
    src_ts[k] = kind[k] == kQ ? p.q_ts : kind[k] == kK ? p.k_ts : p.v_ts;
    dst_at[k] = kind[k] == kQ ? (int64_t)head * D : (int64_t)((kind[k] == kV ? hkv : 0) + head) * kPage * D;
  }
  const int64_t page_elems = (int64_t)2 * hkv * kPage * D;
  uint16_t* const layer_base = static_cast<uint16_t*>(p.cache.base) + p.layer * p.cache.n_pages * page_elems;

  int slot = 0, pos[4] = {0, 0, 0, 0};
  auto look = [&](int64_t t) {
    if (t >= p.n_tokens) return;
    slot = p.slots[t];
#pragma unroll
    for (int a = 0; a < 4; ++a)
      if (a < axes) pos[a] = p.pos[(int64_t)a * p.n_tokens + t];
  };
  look(blockIdx.x);
  for (int64_t t = blockIdx.x; t < p.n_tokens; t += gridDim.x) {
    bool store = slot >= 0, bad_pos = false;
    if (store && slot >= p.cache.n_pages * kPage) {
      store = false;
      if (threadIdx.x == 0) set_status(p.status, RKV_ERR_INDEX_OUT_OF_RANGE);
    }
#pragma unroll
    for (int a = 0; a < 4; ++a) bad_pos |= a < axes && (pos[a] < 0 || pos[a] >= p.table_rows);
    if (bad_pos) {
      store = false;
      if (threadIdx.x == 0) set_status(p.status, RKV_ERR_INDEX_OUT_OF_RANGE);
    }
    uint16_t* const row = layer_base + (slot / kPage) * page_elems + slot % kPage * D;  // used if stored
    uint16_t* const q_row = p.q_out + t * p.n_q_heads * D;
    uint4 u[kAhead], w[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      u[k] = w[k] = make_uint4(0, 0, 0, 0);
      if (kind[k] == kNone || !(kind[k] == kQ || store)) continue;
      const uint16_t* at = src[k] + t * src_ts[k];
      u[k] = *reinterpret_cast<const uint4*>(at + (kind[k] == kV ? 16 * c : a1));
      w[k] = *reinterpret_cast<const uint4*>(at + (kind[k] == kV ? 16 * c + 8 : b1));
    }
    float2 cs[8];  // cosine and sine of pairs 8 c ..
    if (turned && !bad_pos) {
      auto pos_of = [&](int axis) { return axis == 0 ? pos[0] : axis == 1 ? pos[1] : axis == 2 ? pos[2] : pos[3]; };
      if (axis0 == axis7) {
        const float4* from = reinterpret_cast<const float4*>(table + (int64_t)pos_of(axis0) * half);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 f = __ldg(from + i);
          cs[2 * i] = make_float2(f.x, f.y);
          cs[2 * i + 1] = make_float2(f.z, f.w);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) cs[i] = __ldg(table + (int64_t)pos_of(axis_of(8 * c + i)) * half + i);
      }
    }
    look(t + gridDim.x);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      uint32_t x[4] = {u[k].x, u[k].y, u[k].z, u[k].w}, y[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
      if (turned && !bad_pos && kind[k] < kV) {
        // interleaved: word i of x is pair i, word i of y pair 4 + i; else x holds the pairs' first members, y the second
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 e = T::unpack(x[i]), f = T::unpack(y[i]);
          const float2 c0 = cs[kInterleaved ? i : 2 * i], c1 = cs[kInterleaved ? 4 + i : 2 * i + 1];
          const float u0 = e.x, w0 = kInterleaved ? e.y : f.x, u1 = kInterleaved ? f.x : e.y, w1 = f.y;
          const float r0 = u0 * c0.x - w0 * c0.y, s0 = w0 * c0.x + u0 * c0.y;
          const float r1 = u1 * c1.x - w1 * c1.y, s1 = w1 * c1.x + u1 * c1.y;
          x[i] = kInterleaved ? T::pack(r0, s0) : T::pack(r0, r1);
          y[i] = kInterleaved ? T::pack(r1, s1) : T::pack(s0, s1);
        }
      }
      // a K or V row is refused as a whole: its threads vote
      const bool cached = kind[k] == kK || kind[k] == kV;
      bool bad = false;
      if (cached) {
        uint32_t top = 0;  // largest magnitude bits
#pragma unroll
        for (int i = 0; i < 4; ++i) top = __vmaxu2(top, __vmaxu2(x[i] & 0x7fff7fffu, y[i] & 0x7fff7fffu));
        bad = store && max(top & 0xffffu, top >> 16) >= T::kExpMask;
      }
      const unsigned votes = __ballot_sync(0xffffffffu, bad);
      const bool refused = ((votes >> ((threadIdx.x & 31) / A::kPerRow * A::kPerRow)) & ((1u << A::kPerRow) - 1u)) != 0u;
      if (kind[k] == kNone) continue;
      if (cached) {
        if (refused) set_status(p.status, RKV_ERR_NON_FINITE_INPUT);
        if (!store || refused) continue;
      } else if (bad_pos) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = y[i] = 0u;
      }
      uint16_t* dst = (cached ? row : q_row) + dst_at[k];
      *reinterpret_cast<uint4*>(dst + (kind[k] == kV ? 16 * c : a1)) = make_uint4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<uint4*>(dst + (kind[k] == kV ? 16 * c + 8 : b1)) = make_uint4(y[0], y[1], y[2], y[3]);
    }
  }
}

template <typename T>
static void launch_append(const AppendParams& p, bool interleaved, cudaStream_t s) {
  const int64_t heads = p.n_q_heads + 2 * (int64_t)p.cache.n_kv_heads;
  const int per = p.cache.head_dim == 64 ? AppendShape<64>::kHeads : AppendShape<128>::kHeads;
  const int64_t most = 148 * kAppendCtas;
  const dim3 grid((unsigned)(p.n_tokens < most ? p.n_tokens : most), (unsigned)((heads + per - 1) / per));
  if (p.cache.head_dim == 64) {
    if (interleaved) append_kernel<T, 64, true><<<grid, kAppendThreads, 0, s>>>(p);
    else append_kernel<T, 64, false><<<grid, kAppendThreads, 0, s>>>(p);
  } else {
    if (interleaved) append_kernel<T, 128, true><<<grid, kAppendThreads, 0, s>>>(p);
    else append_kernel<T, 128, false><<<grid, kAppendThreads, 0, s>>>(p);
  }
}

// ---- page copies ---------------------------------------------------------------------
constexpr int kCopyThreads = 256;
constexpr int kCopyChunk = kCopyThreads * 4 * 16;  // 16 KB: four 16-byte vectors a thread, loads before stores

// One CTA per (pair, layer, 16 KB of the page); pages are multiples of 16 KB.
// Bytes bound it: 2500 pages of 256 KB take 203 us, 6.45 TB/s, the rate of a copy.
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
  const bool inter = rotary && rotary->interleaved;
  if (cache->dtype == RKV_GQA_BF16) launch_append<Bf16>(p, inter, s);
  else launch_append<F16>(p, inter, s);
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
