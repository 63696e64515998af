// rkv_gqa_decode.cu -- attention of one new token per sequence over the
// grouped-head paged cache.
//
//   x_j = softmax_scale * q . k_j over the sequence's rows j (the last `window`
//   of them), out = sum_j exp(x_j - m) v_j / (sum_j exp(x_j - m) + exp(sink - m)).
//
// Every K and V row is read once, and 4 head_dim flops per (q head, row) are
// little beside 4 head_dim bytes per (kv head, row): HBM bounds it.  So the
// design is about bytes in flight and about every SM moving the same share of
// them:
//
//   * A unit of work is one page (64 rows) of one kv head: its K and its V are
//     8 or 16 KB of contiguous memory each.  The units of all sequences in
//     (sequence, kv head, page) order are cut into equal runs, one per CTA, so
//     ragged lengths, which only the device knows, leave no CTA idle.  Beginning
//     and ending a (sequence, kv head) costs some 3 us, and counts as so many
//     pages.  A run may begin and end inside one; such ends are written as
//     partial softmaxes (m, l, O) and joined by a second small kernel, in the
//     order of the rows.
//   * A producer warp keeps a ring of pages in shared memory full (tensor-map
//     copies, 128-byte swizzle); four consumer warps take 16 rows of each page,
//     keep their own running softmax, and meet only at the end of a (sequence,
//     kv head).
//   * The products are mma.sync m16n8k16 with the group's q heads (16 at a
//     time) as rows: S = Q K^T from ldmatrix, P stays in registers as the A
//     operand of O += P V (ldmatrix.trans).  Rows past the group are zero: the
//     tensor cores have time for them.  They have time for the weights twice,
//     too: rounded to the cache's type, and then what that rounding left of them,
//     so that the result is as good as with weights of 32 bits (without the
//     second product its error against 64 bits was 1.1 to 1.45 times as large;
//     it costs 1% of the 64-sequence time below, and the ragged one nothing).
//
// Groups of more than 16 q heads are taken 16 at a time, each reading the
// pages again, and from HBM: the runs that do are far apart (64 sequences of
// 32768 rows, one kv head of 128: 328 us with 32 q heads and 637 with 64, 3.3 and
// 1.7 TB/s of the cache).
//
// Measured: 64 sequences of 32768 rows, 32 q and 8 kv heads of 128, bf16: 1.28 ms,
// 6.7 TB/s (a copy, which also writes, reaches 6.47).  One sequence of 131072
// rows and 2 kv heads: 31.0 us, of which 5 pass before the first page is there
// and 5 in the join; 256 ragged ones of up to 4096 rows, 4 kv heads of 64, f16: 133
// to 138 us, 5.8 to 6 TB/s.
#include "rkv_gqa.cuh"
#include "rkv_gqa_plan.h"

#include <atomic>

namespace rkv {
namespace gqa {
namespace dec {

constexpr int kRows = 16;      // q heads of a work item
constexpr int kConsumers = 4;  // warps, 16 rows of a page each
constexpr int kThreads = 32 * (kConsumers + 1);
constexpr int kCtasPerSm = 2;
constexpr int kGrid = 148 * kCtasPerSm;
// Up to so many pages are not shared out: with page tables no wider than that, no
// join is launched.  (13 pages of 8 kv heads: 24.4 us to the result when shared
// out and joined, 28.6 us when whole, a page after another.)
constexpr int kWhole = 8;
constexpr int kRing = 3 * 32768;  // bytes of the ring of a CTA: two CTAs' rings and buffers fit an SM

struct Params {
  rkv_gqa_view cache;
  int layer;
  const uint16_t* q;
  int64_t q_ts, q_hs;
  int n_seq, n_q_heads, group, chunks;  // chunks of 16 q heads in a group
  const int32_t* page_table;
  int64_t pt_stride;
  const int32_t* kv_lens;
  int window;
  const float* sinks;
  float scale_log2;
  float* part_o;   // [2 * kGrid][rows][head_dim], rows = min(group, 16)
  float* part_ml;  // [2 * kGrid][rows][2]
  int by_item;     // joins has an entry for each item (fewer than the runs), else for each run, whose last item it is
  int runs;        // CTAs of the launch
  int4* joins;     // [kGrid]: first slot of a shared item (-1: none), last run, sequence, and kv head and chunk
  uint16_t* out;
  uint32_t* status;
};

// The rows [lo, hi) that a sequence's token sees.
struct Seen {
  int lo, hi;
  __device__ int first_page() const { return lo / kPage; }
  __device__ int pages() const { return hi > lo ? (hi + kPage - 1) / kPage - lo / kPage : 0; }
  // an item's units: its pages behind what beginning and ending it costs (256 ragged sequences: runs of 13 items ended
  // at 134 us and runs of 3 at 104 when only pages counted)
  template <int D>
  __device__ int units() const {
    return hi > lo ? pages() + item_units<D>() : 0;
  }
  template <int D>
  static __device__ constexpr int item_units() {
    return D == 64 ? 4 : 2;
  }
  // the page where a cut at unit x goes; items of up to kWhole pages stay whole
  template <int D>
  __device__ int cut(int x) const {
    const int n = pages();
    return n <= kWhole ? (2 * x >= units<D>() ? n : 0) : max(0, x - item_units<D>());
  }
};
__device__ __forceinline__ Seen seen_rows(const Params& p, int s) {
  const int most = (int)p.pt_stride * kPage;
  const int len = min(max(__ldg(p.kv_lens + s), 0), most);
  return {p.window > 0 && len > p.window ? len - p.window : 0, len};
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (T::kCode == RKV_GQA_BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
// The same, and whether all of them say yes: they go on or give up together.
__device__ __forceinline__ bool consumers_agree(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)ok)
      : "memory");
  return r != 0;
}

// Byte of 16-byte chunk c (8 lanes) of row r in a page operand: 64-lane column
// blocks of 8 KB, 128-byte rows, the swizzle of the tensor map.
__device__ __forceinline__ uint32_t sw_off(int r, int c) {
  return (uint32_t)((c >> 3) * 8192 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// Weight of one value-less key with the logit of a head's sink, log2 units.
__device__ __forceinline__ float sink_log2(const float* sinks, int h) {
  return sinks ? sinks[h] * 1.4426950408889634f : -INFINITY;
}

template <int D>
struct Layout {
  static constexpr int kOperand = kPage * D * 2;  // K or V of a page
  static constexpr int kStage = 2 * kOperand;
  static constexpr int kStages = kRing / kStage;  // 3 (head_dim 128) or 6 (64)
  static constexpr int kMerge = kRing;            // two [16][D / 2] f32 buffers, then m and l of every warp
  static constexpr int kMl = kMerge + kRows * D * 4;
  static constexpr int kBars = kMl + kConsumers * kRows * 2 * 4;
  static constexpr int kScan = kBars + 16 * kStages + 16;
  static constexpr int kTotal = kScan + 64 + 1024;  // slack for the 1024-byte alignment
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) decode_kernel(const Params p, const __grid_constant__ CUtensorMap map) {
  using L = Layout<D>;
  constexpr int kStages = L::kStages, kK = D / 16;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  const uint32_t base = smem_u32(smem), bars = base + L::kBars;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kBars + 16 * kStages);
  long long* scan = reinterpret_cast<long long*>(smem + L::kScan);
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(bars + 8 * i, 1);
      mbar_init(bars + 8 * (kStages + i), kConsumers);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
  }
  grid_dependency_wait();
  grid_launch_dependents();

  // ---- this CTA's run of units: pages of all sequences, counted by all threads
  const int per = (p.n_seq + kThreads - 1) / kThreads;
  const int s_begin = min(tid * per, p.n_seq), s_end = min(s_begin + per, p.n_seq);
  long long mine = 0;
  for (int s = s_begin; s < s_end; ++s) mine += seen_rows(p, s).template units<D>();
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) scan[warp] = upto;
  __syncthreads();
  long long total = 0;
  for (int w = 0; w <= kConsumers; ++w) {
    if (w < warp) upto += scan[w];
    total += scan[w];
  }
  const int hg = p.cache.n_kv_heads * p.chunks;  // items of a sequence
  total *= hg;
  const long long ctas = max(1ll, min((long long)gridDim.x, total));
  const long long u0 = blockIdx.x < ctas ? blockIdx.x * total / ctas : total;
  const long long u1 = blockIdx.x < ctas ? (blockIdx.x + 1) * total / ctas : total;
  long long* found = scan + 5;
  const long long before = upto - mine;
  if (u0 < u1 && u0 >= before * hg && u0 < upto * hg) {
    long long at = before;
    int s = s_begin;
    for (; s < s_end; ++s) {
      const int n = seen_rows(p, s).template units<D>();
      if (u0 < (at + n) * hg) break;
      at += n;
    }
    found[0] = s;
    found[1] = u0 - at * hg;
  }
  // sequences that see nothing: zeros; lengths the tables cannot hold: reported
  for (int s = blockIdx.x; s < p.n_seq; s += gridDim.x) {
    const int len = __ldg(p.kv_lens + s);
    if (tid == 0 && (len < 0 || len > p.pt_stride * kPage)) set_status(p.status, RKV_ERR_INDEX_OUT_OF_RANGE);
    if (seen_rows(p, s).pages() == 0) {
      for (int i = tid; i < p.n_q_heads * D / 2; i += kThreads)
        reinterpret_cast<uint32_t*>(p.out)[(int64_t)s * p.n_q_heads * D / 2 + i] = 0u;
      if (p.by_item)
        for (int i = tid; i < hg; i += kThreads) p.joins[s * hg + i] = make_int4(-1, 0, 0, 0);
    }
  }
  if (tid == 0 && !p.by_item) p.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);  // unless its last item goes on
  __syncthreads();
  if (u0 >= u1) return;
  int s = (int)found[0];
  long long rest = found[1];  // units of sequence s before this run
  long long left = u1 - u0;

  if (warp == kConsumers) {
    // ---------------------------------------------------------------- producer
    // The whole warp walks the pages, 32 page ids a load; one lane copies.
    const int rows_total = (int)row_base(p.cache, p.cache.n_layers, 0, 0, 0);  // out of range: zero rows
    int n = 0;
    bool ok = true;
    for (; left > 0 && ok && s < p.n_seq; ++s) {
      const Seen see = seen_rows(p, s);
      const int pages = see.pages();
      if (pages == 0) continue;
      const int units = see.units<D>();
      for (int item = (int)(rest / units), x = (int)(rest % units); item < hg && left > 0 && ok; ++item, x = 0) {
        const int head = item / p.chunks;
        const int32_t* ids = p.page_table + s * p.pt_stride + see.first_page();
        const int stop = (int)min((long long)units, x + left);
        const int pg = see.cut<D>(x), end = see.cut<D>(stop);
        left -= stop - x;
        for (int at = pg; at < end && ok; at += 32) {
          const int id = at + lane < end ? __ldg(ids + at + lane) : 0;
          const bool good = id >= 0 && id < p.cache.n_pages;
          if (!good) set_status(p.status, RKV_ERR_INDEX_OUT_OF_RANGE);
          const int row = good ? (int)row_base(p.cache, p.layer, id, 0, head) : rows_total;
          const int count = min(32, end - at);
          for (int i = 0; i < count; ++i, ++n) {
            const int y = __shfl_sync(0xffffffffu, row, i);
            const int st = n % kStages;
            if (n >= kStages && !__all_sync(0xffffffffu, mbar_wait(bars + 8 * (kStages + st), (n / kStages - 1) & 1, abort_flag))) {
              ok = false;
              break;
            }
            if (lane == 0) {
              const uint32_t full = bars + 8 * st, dst = base + st * L::kStage;
              const int yv = y == rows_total ? y : y + p.cache.n_kv_heads * kPage;
              mbar_expect_tx(full, L::kStage);
#pragma unroll
              for (int c = 0; c < D / 64; ++c) tma_load_2d(dst + c * 8192, &map, 64 * c, y, full);
#pragma unroll
              for (int c = 0; c < D / 64; ++c) tma_load_2d(dst + L::kOperand + c * 8192, &map, 64 * c, yv, full);
            }
          }
        }
      }
      rest = 0;
    }
    if (!ok) {
      *abort_flag = 1;
      set_status(p.status, RKV_ERR_CUDA);
    }
    // every copy has landed before the CTA ends
    for (int i = max(0, n - kStages); i < n; ++i) mbar_wait_copy(bars + 8 * (i % kStages), (i / kStages) & 1);
    return;
  }

  // ------------------------------------------------------------------ consumers
  // Warp w has rows 16 w .. 16 w + 15 of every page.  Of the accumulators a
  // thread holds q heads r0 = lane / 4 and r0 + 8.
  const int r0 = lane >> 2, t4 = lane & 3;
  const int krow = 16 * warp + ((lane >> 4) << 3) + (lane & 7), kchunk = (lane >> 3) & 1;  // ldmatrix addresses, K
  const int vrow = 16 * warp + (lane & 15), vchunk = lane >> 4;                             // and V
  float* merge = reinterpret_cast<float*>(smem + L::kMerge);
  float* ml = reinterpret_cast<float*>(smem + L::kMl);
  const int rows = min(p.group, kRows);
  int n = 0, segment = 0;
  bool ok = true;
  for (; left > 0 && ok && s < p.n_seq; ++s) {
    const Seen see = seen_rows(p, s);
    const int pages = see.pages();
    if (pages == 0) continue;
    const int units = see.units<D>();
    for (int item = (int)(rest / units), x = (int)(rest % units); item < hg && left > 0 && ok; ++item, x = 0) {
      const int stop = (int)min((long long)units, x + left);
      const int pg = see.cut<D>(x), end = see.cut<D>(stop);
      const long long begin = u1 - left - x;  // the item's first unit
      left -= stop - x;
      if (end <= pg) continue;
      const int head0 = (item / p.chunks) * p.group + (item % p.chunks) * kRows;  // first q head
      const int live = min(kRows, p.group - (item % p.chunks) * kRows);
      uint32_t qf[kK][4];
      const uint16_t* q0 = p.q + (int64_t)s * p.q_ts + (head0 + r0) * p.q_hs + 2 * t4;
      const uint16_t* q1 = q0 + 8 * p.q_hs;
#pragma unroll
      for (int i = 0; i < kK; ++i) {
        qf[i][0] = r0 < live ? *reinterpret_cast<const uint32_t*>(q0 + 16 * i) : 0u;
        qf[i][1] = r0 + 8 < live ? *reinterpret_cast<const uint32_t*>(q1 + 16 * i) : 0u;
        qf[i][2] = r0 < live ? *reinterpret_cast<const uint32_t*>(q0 + 16 * i + 8) : 0u;
        qf[i][3] = r0 + 8 < live ? *reinterpret_cast<const uint32_t*>(q1 + 16 * i + 8) : 0u;
      }
      float o[D / 8][4];
#pragma unroll
      for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;  // exponent references; l: this thread's columns
      for (int at = pg; at < end; ++at, ++n) {
        const int st = n % kStages;
        if (!__all_sync(0xffffffffu, mbar_wait(bars + 8 * st, (n / kStages) & 1, abort_flag))) {
          ok = false;
          *abort_flag = 1;
          break;
        }
        const uint32_t ks = base + st * L::kStage, vs = ks + L::kOperand;
        float x[2][4] = {};
#pragma unroll
        for (int i = 0; i < kK; ++i) {
          uint32_t b[4];
          ldsm4(ks + sw_off(krow, 2 * i + kchunk), b);
          mma<T>(x[0], qf[i], b[0], b[1]);
          mma<T>(x[1], qf[i], b[2], b[3]);
        }
        // rows of this page that the token sees: [from, to)
        const int page0 = (see.first_page() + at) * kPage;
        const int from = see.lo - page0, to = see.hi - page0;
        if (from > 0 || to < kPage) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = 16 * warp + 8 * j + 2 * t4 + (e & 1);
              x[j][e] = key >= from && key < to ? x[j][e] * p.scale_log2 : -INFINITY;
            }
          // their V rows may hold anything: a weight of zero must meet zeros
          for (int c = lane; c < 16 * (D / 8); c += 32) {
            const int r = 16 * warp + c / (D / 8);
            if (r < from || r >= to)
              *reinterpret_cast<uint4*>(smem + st * L::kStage + L::kOperand + sw_off(r, c % (D / 8))) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
          __syncwarp();
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[j][e] *= p.scale_log2;
        }
        float t0 = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[1][0], x[1][1]));
        float t1 = fmaxf(fmaxf(x[0][2], x[0][3]), fmaxf(x[1][2], x[1][3]));
#pragma unroll
        for (int d = 1; d <= 2; d <<= 1) {
          t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, d));
          t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, d));
        }
        t0 -= SoftmaxBias<T>::kBias;
        t1 -= SoftmaxBias<T>::kBias;
        const bool up0 = t0 > m0 + kLazyLog2 || (m0 == -INFINITY && t0 > -INFINITY);
        const bool up1 = t1 > m1 + kLazyLog2 || (m1 == -INFINITY && t1 > -INFINITY);
        if (__any_sync(0xffffffffu, up0 || up1)) {
          const float a0 = up0 ? ex2(m0 - t0) : 1.f, a1 = up1 ? ex2(m1 - t1) : 1.f;  // 0 from -inf
          m0 = up0 ? t0 : m0;
          m1 = up1 ? t1 : m1;
          l0 *= a0;
          l1 *= a1;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            o[i][0] *= a0;
            o[i][1] *= a0;
            o[i][2] *= a1;
            o[i][3] *= a1;
          }
        }
        const float s0 = m0 == -INFINITY ? 0.f : m0, s1 = m1 == -INFINITY ? 0.f : m1;  // nothing seen yet: weights 0
        uint32_t pf[4], pr[4];  // the weights in the type, and what that rounding left of them
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float e0 = ex2(x[j][0] - s0), e1 = ex2(x[j][1] - s0), e2 = ex2(x[j][2] - s1), e3 = ex2(x[j][3] - s1);
          l0 += e0 + e1;
          l1 += e2 + e3;
          pf[2 * j] = T::pack(e0, e1);
          pf[2 * j + 1] = T::pack(e2, e3);
          const float2 h0 = T::unpack(pf[2 * j]), h1 = T::unpack(pf[2 * j + 1]);
          pr[2 * j] = T::pack(e0 - h0.x, e1 - h0.y);
          pr[2 * j + 1] = T::pack(e2 - h1.x, e3 - h1.y);
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t b[4];
          ldsm4t(vs + sw_off(vrow, 2 * i + vchunk), b);
          mma<T>(o[2 * i], pf, b[0], b[1]);
          mma<T>(o[2 * i + 1], pf, b[2], b[3]);
          mma<T>(o[2 * i], pr, b[0], b[1]);
          mma<T>(o[2 * i + 1], pr, b[2], b[3]);
        }
        // This warp's reads of the stage come before the copy that overwrites it.  The barrier alone orders them among loads
        // and stores, not with the copies of the other proxy: without the fence a copy that came at once (pages in L2,
        // launches close behind one another) overtook the last reads of V, once in some hundred to thousand launches.
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + 8 * (kStages + st));
      }
      // ---- the four warps' softmaxes joined, the result by warp 0
      l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
      l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
      if (t4 == 0) {
        ml[2 * (warp * kRows + r0)] = m0;
        ml[2 * (warp * kRows + r0) + 1] = l0;
        ml[2 * (warp * kRows + r0 + 8)] = m1;
        ml[2 * (warp * kRows + r0 + 8) + 1] = l1;
      }
      ok = consumers_agree(ok);
      if (!ok) break;
      float M0 = -INFINITY, M1 = -INFINITY;
      for (int w = 0; w < kConsumers; ++w) {
        M0 = fmaxf(M0, ml[2 * (w * kRows + r0)]);
        M1 = fmaxf(M1, ml[2 * (w * kRows + r0 + 8)]);
      }
      const float z0 = M0 == -INFINITY ? 0.f : M0, z1 = M1 == -INFINITY ? 0.f : M1;
      float L0 = 0.f, L1 = 0.f;
      for (int w = 0; w < kConsumers; ++w) {
        L0 += ml[2 * (w * kRows + r0) + 1] * ex2(ml[2 * (w * kRows + r0)] - z0);
        L1 += ml[2 * (w * kRows + r0 + 8) + 1] * ex2(ml[2 * (w * kRows + r0 + 8)] - z1);
      }
      const float f0 = ex2(m0 - z0), f1 = ex2(m1 - z1);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][0] *= f0;
        o[i][1] *= f0;
        o[i][2] *= f1;
        o[i][3] *= f1;
      }
      // warps 2 and 3 onto 0 and 1, then 1 onto 0, half of the lanes at a time; a thread's values keep their place
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int half = 2; half >= 1; half >>= 1) {
          if (warp >= half && warp < 2 * half) {
            float4* dst = reinterpret_cast<float4*>(merge + (warp - half) * kRows * D / 2);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              const float(&v)[4] = o[h * (D / 16) + i];
              dst[i * 32 + lane] = make_float4(v[0], v[1], v[2], v[3]);
            }
          }
          consumers_sync();
          if (warp < half) {
            const float4* src = reinterpret_cast<const float4*>(merge + warp * kRows * D / 2);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              const float4 v = src[i * 32 + lane];
              float(&d)[4] = o[h * (D / 16) + i];
              d[0] += v.x;
              d[1] += v.y;
              d[2] += v.z;
              d[3] += v.w;
            }
          }
          consumers_sync();
        }
      }
      if (warp == 0) {
        if (pg == 0 && end == pages) {
          auto norm = [&](int r, float M, float l) {
            const float sink = sink_log2(p.sinks, head0 + r);
            const float top = fmaxf(M, sink);
            const float w = ex2(M - top);
            return M == -INFINITY && l == 0.f ? 0.f : w / (l * w + ex2(sink - top));
          };
          const float n0 = r0 < live ? norm(r0, M0, L0) : 0.f, n1 = r0 + 8 < live ? norm(r0 + 8, M1, L1) : 0.f;
          uint16_t* d0 = p.out + ((int64_t)s * p.n_q_heads + head0 + r0) * D + 2 * t4;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            if (r0 < live) *reinterpret_cast<uint32_t*>(d0 + 8 * i) = T::pack(o[i][0] * n0, o[i][1] * n0);
            if (r0 + 8 < live) *reinterpret_cast<uint32_t*>(d0 + 8 * D + 8 * i) = T::pack(o[i][2] * n1, o[i][3] * n1);
          }
          if (lane == 0 && p.by_item) p.joins[s * hg + item] = make_int4(-1, 0, 0, 0);
        } else {
          const int64_t slot = 2 * blockIdx.x + (segment > 0);
          float* d0 = p.part_o + (slot * rows + r0) * D + 2 * t4;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            if (r0 < live) *reinterpret_cast<float2*>(d0 + 8 * i) = make_float2(o[i][0], o[i][1]);
            if (r0 + 8 < live) *reinterpret_cast<float2*>(d0 + 8 * D + 8 * i) = make_float2(o[i][2], o[i][3]);
          }
          if (t4 == 0) {
            if (r0 < live) *reinterpret_cast<float2*>(p.part_ml + 2 * (slot * rows + r0)) = make_float2(M0, L0);
            if (r0 + 8 < live) *reinterpret_cast<float2*>(p.part_ml + 2 * (slot * rows + r0 + 8)) = make_float2(M1, L1);
          }
          // the run that holds the item's first unit says which runs the join reads (thread 0, as above)
          if (lane == 0 && pg == 0) {
            const long long last = ((begin + units) * ctas - 1) / total;  // its last unit is a page
            p.joins[p.by_item ? s * hg + item : blockIdx.x] = make_int4(2 * blockIdx.x + (segment > 0), (int)last, s, item);
          }
        }
      }
      ++segment;
    }
    rest = 0;
  }
  if (!ok) set_status(p.status, RKV_ERR_CUDA);
}

// Joins the partial softmaxes of the q heads of a shared item: first slot as
// recorded, then slot 2 c' of every later run c'.  kWarps warps
// take the parts of a head in turn, several at a time with their loads out
// together, lanes the head's lanes; the warps' sums are added in order.  Sixteen
// warps where an item has many parts (one sequence of 131072 rows and 2 kv heads:
// 148; 14 us with eight warps and one load after another, 5.8 with sixteen and four
// loads, a microsecond less with ten: one trip for all), one where it has a few (256
// ragged sequences: 13.5 us with sixteen, whose threads mostly start for nothing).
constexpr int kJoinThreads = 128;  // with one warp a head: four heads
template <typename T, int D, int kWarps>
__global__ void __launch_bounds__(kWarps == 1 ? kJoinThreads : 32 * kWarps) join_kernel(const Params p) {
  __shared__ float acc[kWarps == 1 ? 1 : kWarps][D];
  __shared__ float2 ends[kWarps];
  grid_dependency_wait();
  const int4 join = p.joins[blockIdx.x];
  const int warp = kWarps == 1 ? 0 : threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t s = join.z;
  const int item = join.w, r = kWarps == 1 ? blockIdx.y * (kJoinThreads / 32) + (threadIdx.x >> 5) : blockIdx.y;
  if (!join_holds(join.x, join.y, join.z, join.w, p.runs, p.n_seq, p.cache.n_kv_heads * p.chunks) ||
      r >= min(kRows, p.group - (item % p.chunks) * kRows))
    return;
  const int rows = min(p.group, kRows);
  const int head = (item / p.chunks) * p.group + (item % p.chunks) * kRows + r;
  const int count = join.y - join.x / 2 + 1;
  auto slot = [&](int i) { return (int64_t)(i == 0 ? join.x : 2 * (join.x / 2 + i)); };
  constexpr int kAhead = kWarps == 1 ? 4 : 10;
  float o[D / 32] = {};
  float m = -INFINITY, l = 0.f;
  for (int i0 = warp; i0 < count; i0 += kAhead * kWarps) {
    float2 e[kAhead];
    float v[kAhead][D / 32];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * kWarps;
      e[k] = make_float2(-INFINITY, 0.f);
      if (i >= count) continue;
      const int64_t at = slot(i) * rows + r;
      e[k] = *reinterpret_cast<const float2*>(p.part_ml + 2 * at);
      if constexpr (D == 128) {
        const float4 f = *reinterpret_cast<const float4*>(p.part_o + at * D + 4 * lane);
        v[k][0] = f.x, v[k][1] = f.y, v[k][2] = f.z, v[k][3] = f.w;
      } else {
        const float2 f = *reinterpret_cast<const float2*>(p.part_o + at * D + 2 * lane);
        v[k][0] = f.x, v[k][1] = f.y;
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (e[k].x == -INFINITY && e[k].y == 0.f) continue;  // nothing there (a sum of NaN is something)
      const float top = fmaxf(m, e[k].x);
      const float a = ex2(m - top), w = ex2(e[k].x - top);  // 0 from -inf
      l = l * a + w * e[k].y;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) o[j] = o[j] * a + w * v[k][j];
      m = top;
    }
  }
  const float sink = sink_log2(p.sinks, head);
  uint32_t* const out = reinterpret_cast<uint32_t*>(p.out + (s * p.n_q_heads + head) * D);
  if constexpr (kWarps == 1) {
    float top = fmaxf(m, sink);
    if (top == -INFINITY) top = 0.f;
    const float f = ex2(m - top), total = l * f + ex2(sink - top), inv = total == 0.f ? 0.f : f / total;
#pragma unroll
    for (int j = 0; j < D / 64; ++j) out[D / 64 * lane + j] = T::pack(o[2 * j] * inv, o[2 * j + 1] * inv);
  } else {
#pragma unroll
    for (int j = 0; j < D / 32; ++j) acc[warp][D / 32 * lane + j] = o[j];
    if (lane == 0) ends[warp] = make_float2(m, l);
    __syncthreads();
    if (threadIdx.x < D / 2) {
      float top = sink;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ends[w].x);
      if (top == -INFINITY) top = 0.f;
      float a = 0.f, b = 0.f, total = ex2(sink - top);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(ends[w].x - top);
        a += f * acc[w][2 * threadIdx.x];
        b += f * acc[w][2 * threadIdx.x + 1];
        total += f * ends[w].y;
      }
      const float inv = total == 0.f ? 0.f : 1.f / total;
      out[threadIdx.x] = T::pack(a * inv, b * inv);
    }
  }
}

template <typename T, int D>
static rkv_status launch(Params p, const CUtensorMap& map, cudaStream_t s, const char* what) {
  static std::atomic<bool> ready[kMaxDevicesCached];  // the shared-memory opt-in is per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevicesCached || !ready[dev].load(std::memory_order_acquire)) {
    const cudaError_t e =
        cudaFuncSetAttribute(decode_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::kTotal);
    if (e != cudaSuccess) return fail(RKV_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    if (dev >= 0 && dev < kMaxDevicesCached) ready[dev].store(true, std::memory_order_release);
  }
  // both kernels may start while the one before drains; they wait before they read
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  // no more CTAs than there can be units
  const int64_t units = (int64_t)p.n_seq * p.cache.n_kv_heads * p.chunks * p.pt_stride;
  const unsigned grid = (unsigned)(units < kGrid ? units : kGrid);
  const int64_t items = (int64_t)p.n_seq * p.cache.n_kv_heads * p.chunks;
  p.runs = (int)grid;
  p.by_item = grid > 8 * items;  // more than eight parts an item, were they alike
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Layout<D>::kTotal;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, decode_kernel<T, D>, p, map);
  if (e == cudaSuccess && p.pt_stride > kWhole) {
    const unsigned rows = (unsigned)(p.group < kRows ? p.group : kRows);
    cfg.dynamicSmemBytes = 0;
    if (p.by_item) {
      cfg.gridDim = dim3((unsigned)items, rows);
      cfg.blockDim = dim3(32 * 16);
      e = cudaLaunchKernelEx(&cfg, join_kernel<T, D, 16>, p);
    } else {
      cfg.gridDim = dim3(grid, (rows + kJoinThreads / 32 - 1) / (kJoinThreads / 32));
      cfg.blockDim = dim3(kJoinThreads);
      e = cudaLaunchKernelEx(&cfg, join_kernel<T, D, 1>, p);
    }
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(RKV_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
  }
  return check_launch(what);
}

}  // namespace dec
}  // namespace gqa
}  // namespace rkv

extern "C" int64_t rkv_gqa_decode_workspace_bytes(const rkv_gqa_view* cache, int32_t n_seq, int32_t n_q_heads) {
  using namespace rkv::gqa::dec;
  if (!cache || n_seq < 0 || n_q_heads < 1 || cache->n_kv_heads < 1 || n_q_heads % cache->n_kv_heads != 0) return -1;
  const int64_t group = n_q_heads / cache->n_kv_heads, rows = group < kRows ? group : kRows;
  return 2 * kGrid * rows * (cache->head_dim + 2) * 4 + kGrid * 16;
}

extern "C" rkv_status rkv_gqa_decode(const rkv_gqa_view* cache, int32_t layer, const void* q, int64_t q_token_stride,
                                     int64_t q_head_stride, int32_t n_seq, int32_t n_q_heads, const int32_t* page_table,
                                     int64_t pt_stride, const int32_t* kv_lens, int32_t window, const float* sinks,
                                     float softmax_scale, void* workspace, void* out, uint32_t* d_status,
                                     rkv_stream_t stream) {
  using namespace rkv;
  using namespace rkv::gqa;
  using namespace rkv::gqa::dec;
  static const char* what = "rkv_gqa_decode";
  rkv_status st = check_cache(cache, layer, what);
  if (st != RKV_OK) return st;
  if ((st = check_heads(cache, n_q_heads, what)) != RKV_OK) return st;
  if (n_seq < 0) return fail_shape("n_seq", 0, n_seq, "%s: n_seq < 0", what);
  if (n_seq == 0) {
    clear_error();
    return RKV_OK;
  }
  const AttendArgs a = {*cache,    layer,   q,      q_token_stride, q_head_stride, n_seq, n_q_heads, page_table,
                        pt_stride, kv_lens, window, sinks,          softmax_scale, out,   d_status};
  if ((st = check_attend(a, what)) != RKV_OK) return st;
  if (!workspace || !aligned(workspace, 16))
    return fail(RKV_ERR_INVALID_ARGUMENT, "%s: a 16-byte aligned workspace is required", what);
  Params p;
  p.cache = *cache;
  p.layer = layer;
  p.q = static_cast<const uint16_t*>(q);
  p.q_ts = q_token_stride;
  p.q_hs = q_head_stride;
  p.n_seq = n_seq;
  p.n_q_heads = n_q_heads;
  p.group = n_q_heads / cache->n_kv_heads;
  p.chunks = (p.group + kRows - 1) / kRows;
  p.page_table = page_table;
  p.pt_stride = pt_stride;
  p.kv_lens = kv_lens;
  p.window = window_of(window, pt_stride);
  p.sinks = sinks;
  p.scale_log2 = (float)((double)softmax_scale * 1.4426950408889634);
  const int64_t rows = p.group < kRows ? p.group : kRows;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + 2 * kGrid * rows * cache->head_dim;
  p.joins = reinterpret_cast<int4*>(p.part_ml + 2 * kGrid * rows * 2);
  p.out = static_cast<uint16_t*>(out);
  p.status = d_status;
  CUtensorMap map;
  if ((st = cache_map(*cache, &map, what)) != RKV_OK) return st;
  cudaStream_t s = (cudaStream_t)stream;
  if (cache->dtype == RKV_GQA_BF16)
    return cache->head_dim == 64 ? launch<Bf16, 64>(p, map, s, what) : launch<Bf16, 128>(p, map, s, what);
  return cache->head_dim == 64 ? launch<F16, 64>(p, map, s, what) : launch<F16, 128>(p, map, s, what);
}
