// rkv_gqa_prefill.cu -- causal attention of packed new tokens over the
// grouped-head paged cache.
//
//   x_j = softmax_scale * q . k_j over the rows j that a token sees,
//   out = sum_j exp(x_j - m) v_j / (sum_j exp(x_j - m) + exp(sink - m)).
//
// 4 head_dim flops per (q head, token, visible row): the 5th-generation tensor
// cores bound it, and close behind them the 16 exponentials a clock that an SM
// evaluates (a 128 x 128 tile: 1024 clocks of each at head_dim 128).
//
// One CTA takes two tiles of 128 q rows of one kv head, against a page (64 key
// rows) at a time.  A tile's rows are the group's q heads of 128 / group
// consecutive tokens, token by token, so that every K and V row fetched serves
// the whole group and a tile of a long prompt has a short diagonal.
//
//   warps 0-15      softmax, one row a thread: S from tensor memory, running
//                   maximum and sum, P (in the cache's type) back over S; the
//                   epilogue.  Four warps have the even steps of tile 0, four
//                   its odd steps, and so for tile 1
//   warps 16, 17    issue S = Q K^T (Q, K in shared memory) and O += P V (P in
//                   tensor memory, V in shared memory) of tile 0 and of tile 1
//   warp 18         copies Q, K and V by tensor maps into a ring of stages
//
// Tensor memory: two S buffers of 64 columns for each tile (P over the first 32
// of its own), O0, O1 (head_dim columns each).  S of step j + 2 is issued behind
// O += P V of step j, so a tile's next logits are there before its warps are
// done with the last ones, and neither they nor the tensor cores wait for the
// other's latency.  (With one S buffer of 128 columns a tile the chain softmax
// -> P -> O -> next S was 3400-4000 clocks a step beside 2400 of MMAs.)  An
// issuing thread is held up until the tensor cores are nearly done with what it
// issued, so each tile has a warp of its own for it: one warp for both left
// them idle for the 200-700 clocks of its waits between two batches.
//
// The exponentials of a step take four warps (one a scheduler) 512 clocks at the
// least; the loads, maxima, conversions and waits around them as long again.  So
// two sets of warps take a tile's steps in turn, one's latencies behind the
// other's exponentials.  They share the rows' exponent reference: a step's
// warps publish it (shared memory, one barrier a warp) as soon as they have
// their maxima, and the next step's take it from there.
#include <atomic>

#include "rkv_gqa.cuh"

namespace rkv {
namespace gqa {
namespace pre {

constexpr int kM = 128;        // q rows of a tile
constexpr int kN = kPage;      // key rows of a step
constexpr int kThreads = 640;  // warp 19 only completes the last warpgroup
constexpr int kMmaWarp = 16, kLoadWarp = 18;
constexpr uint32_t kTmemCols = 512;
// The launch has 96 registers a thread; the four softmax warpgroups take what the
// fifth does without.  (Calls that are not inlined do not go with it: ptxas
// does not end.)
constexpr int kSoftmaxRegs = 104, kOtherRegs = 64;
static_assert(4 * kSoftmaxRegs + kOtherRegs <= 5 * 96, "more registers than the launch has");

struct Params {
  rkv_gqa_view cache;
  int layer;
  int n_tokens, n_q_heads, group, tile_tokens;  // tokens of a tile: 128 / group
  const int32_t* cu_q;
  int n_seq;
  const int32_t* page_table;
  int64_t pt_stride;
  const int32_t* kv_lens;
  int window;
  const float* sinks;
  float scale_log2;
  int n_splits;
  float* part_o;   // [n_splits][n_tokens][n_q_heads][head_dim]
  float* part_ml;  // [n_splits][n_tokens][n_q_heads][2]
  uint16_t* out;
  uint32_t* status;
};

template <int D>
struct Layout {
  static constexpr int kQ = kM * D * 2;      // bytes of a Q tile
  static constexpr int kStage = kN * D * 2;  // K or V of a page
  static constexpr int kStages = D == 128 ? 10 : 16;
  static constexpr int kQCol = kM * 128;     // a 64-lane column block of a Q tile
  static constexpr int kCol = kN * 128;      // and of a page
  static constexpr int kRing = 2 * kQ;
  static constexpr int kBars = kRing + kStages * kStage;
  // full[kStages], empty[kStages], S full [2][2], P full [2][2], PV done [2], Q full, drain [2], reference [2][4], O complete [2]
  static constexpr int kBarEmpty = 8 * kStages, kBarS = 16 * kStages, kBarP = kBarS + 32, kBarPv = kBarP + 32,
                       kBarQ = kBarPv + 16, kBarDrain = kBarQ + 8;
  static constexpr int kBarRef = kBarDrain + 16;
  static constexpr int kBarO = kBarRef + 64;
  static constexpr int kMisc = kBars + kBarO + 16;  // TMEM address, abort flag, found, scan
  static constexpr int kRef = kMisc + 128;           // exponent references [2][128]
  static constexpr int kTotal = kRef + 1024 + 1024;  // slack for the 1024-byte alignment
};

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ bool elect_one() {
  uint32_t pred = 0;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(pred));
  return pred != 0;
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// D = A B (+ D): A in shared memory, or (ta) in tensor memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// 128-byte-swizzle matrix descriptor.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3fffu) | ((uint64_t)((lbo >> 4) & 0x3fffu) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3fffu) << 32) | (1ull << 46) | (2ull << 61);
}
// A warp's 32 lanes x 32 columns: thread t holds lane t.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// max(a, b, c) in one instruction (sm_100); NaN handling as fmaxf.
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ unsigned long long pk2(uint32_t lo, uint32_t hi) {
  return ((unsigned long long)hi << 32) | lo;
}
__device__ __forceinline__ unsigned long long dup2(float x) { return pk2(__float_as_uint(x), __float_as_uint(x)); }

// The weights 2^(x scale - m) of a row's 64 logits, stored over S as P in the
// cache's type; returns their sum.  (A cubic on the FMA pipe in place of a
// quarter to a half of the exponentials made the 8192-token prompt 2 to 12%
// slower: its 7 instructions a pair cost more than the exponential unit has
// to spare.)
template <typename T>
__device__ __forceinline__ float weights(const uint32_t (&x)[kN], uint32_t ts, unsigned long long c2, unsigned long long n2) {
  unsigned long long sum0 = 0ull, sum1 = 0ull;
#pragma unroll
  for (int i = 0; i < kN; i += 32) {
    uint32_t pw[16];
#pragma unroll
    for (int k = 0; k < 32; k += 2) {
      const unsigned long long a = fma_f32x2(pk2(x[i + k], x[i + k + 1]), c2, n2);
      const float e0 = ex2(__uint_as_float((uint32_t)a)), e1 = ex2(__uint_as_float((uint32_t)(a >> 32)));
      if (k & 2) sum1 = add_f32x2(sum1, pk2(__float_as_uint(e0), __float_as_uint(e1)));
      else sum0 = add_f32x2(sum0, pk2(__float_as_uint(e0), __float_as_uint(e1)));
      pw[k / 2] = T::pack(e0, e1);
    }
    tmem_st16(ts + i / 2, pw);
  }
  const unsigned long long sum = add_f32x2(sum0, sum1);
  return __uint_as_float((uint32_t)sum) + __uint_as_float((uint32_t)(sum >> 32));
}

// Place of step j's K and V in the ring's order K0 K1 V0 K2 V1 K3 ...
__device__ __forceinline__ int k_place(int j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ int v_place(int j) { return 2 * j + 2; }

// The new tokens of sequence s in q: [begin, end), cut to what q holds.
__device__ __forceinline__ int2 new_tokens(const Params& p, int s) {
  const int a = min(max(__ldg(p.cu_q + s), 0), p.n_tokens);
  return make_int2(a, min(max(__ldg(p.cu_q + s + 1), a), p.n_tokens));
}

// What a CTA works on, the same for all of its threads.
struct Work {
  int head;         // kv head
  int seq;
  int token;        // first token (row of q)
  int tokens;       // tokens of both tiles
  int pos;          // position of the first token, may be negative
  int len;          // rows of the sequence
  int step0, steps; // pages of this CTA's split
  int steps0;       // of which tile 0 needs the first ones only
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
prefill_kernel(const Params p, const __grid_constant__ CUtensorMap map, const __grid_constant__ CUtensorMap qmap) {
  using L = Layout<D>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  const uint32_t base = smem_u32(smem), bars = base + L::kBars;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);
  int* found = reinterpret_cast<int*>(smem + L::kMisc + 8);  // sequence, block within it
  int* scan = reinterpret_cast<int*>(smem + L::kMisc + 16);  // [20] per warp

  if (tid == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(bars + 8 * i, 1);
      mbar_init(bars + L::kBarEmpty + 8 * i, 2);  // both tiles
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(bars + L::kBarS + 8 * i, 1);
      mbar_init(bars + L::kBarP + 8 * i, 128);
    }
    mbar_init(bars + L::kBarPv, 1);
    mbar_init(bars + L::kBarPv + 8, 1);
    mbar_init(bars + L::kBarQ, 1);
    mbar_init(bars + L::kBarDrain, 1);
    mbar_init(bars + L::kBarDrain + 8, 1);
    for (int i = 0; i < 8; ++i) mbar_init(bars + L::kBarRef + 8 * i, 1);
    mbar_init(bars + L::kBarO, 1);
    mbar_init(bars + L::kBarO + 8, 1);
    *abort_flag = 0;
    found[0] = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&qmap) : "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // q rows that no token has (groups that do not divide 128): zeros
  const int used = p.tile_tokens * p.group;
  for (int i = tid; i < 2 * (kM - used) * (D / 8); i += kThreads) {
    const int chunk = i % (D / 8), r = used + (i / (D / 8)) % (kM - used), t = i / ((D / 8) * (kM - used));
    *reinterpret_cast<uint4*>(smem + t * L::kQ + (chunk >> 3) * L::kQCol + r * 128 + (((chunk & 7) ^ (r & 7)) << 4)) =
        make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async();
  grid_dependency_wait();
  grid_launch_dependents();

  // ---- which sequence and tokens: blocks of two tiles, the last tokens first
  const int span = 2 * p.tile_tokens;
  const int rank = blockIdx.x / p.cache.n_kv_heads;
  {
    const int per = (p.n_seq + kThreads - 1) / kThreads;
    const int s_begin = min(tid * per, p.n_seq), s_end = min(s_begin + per, p.n_seq);
    int mine = 0;
    for (int s = s_begin; s < s_end; ++s) {
      const int2 t = new_tokens(p, s);
      mine += (t.y - t.x + span - 1) / span;
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) scan[warp] = upto;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    for (int w = 0; w < warp; ++w) upto += scan[w];
    int at = upto - mine;
    if (rank >= at && rank < upto) {
      for (int s = s_begin; s < s_end; ++s) {
        const int2 t = new_tokens(p, s);
        const int n = (t.y - t.x + span - 1) / span;
        if (rank < at + n) {
          found[0] = s;
          found[1] = n - 1 - (rank - at);
          break;
        }
        at += n;
      }
    }
    __syncthreads();
  }
  const uint32_t tmem = *tmem_slot;
  Work w;
  w.seq = found[0];
  w.steps = w.steps0 = 0;
  if (w.seq >= 0) {
    const int2 t = new_tokens(p, w.seq);
    w.head = blockIdx.x % p.cache.n_kv_heads;
    const int first = found[1] * span;
    w.token = t.x + first;
    w.tokens = min(span, t.y - t.x - first);
    const int given = __ldg(p.kv_lens + w.seq), most = (int)p.pt_stride * kPage;
    w.len = min(max(given, 0), most);
    w.pos = w.len - (t.y - t.x) + first;
    const int end = w.pos + w.tokens;  // rows [.., end) are seen
    const int begin = p.window > 0 ? max(0, w.pos - p.window + 1) : 0;
    const int s0 = begin / kN, s1 = end > 0 ? (end + kN - 1) / kN : 0;
    const int per = (max(0, s1 - s0) + p.n_splits - 1) / p.n_splits;
    w.step0 = s0 + blockIdx.y * per;
    w.steps = max(0, min(per, s1 - w.step0));
    const int end0 = w.pos + min(w.tokens, p.tile_tokens);
    w.steps0 = max(0, min(w.steps, (end0 > 0 ? (end0 + kN - 1) / kN : 0) - w.step0));
    if (tid == 0 && (given != w.len || __ldg(p.cu_q) != 0 || __ldg(p.cu_q + p.n_seq) != p.n_tokens ||
                     t.x != __ldg(p.cu_q + w.seq) || t.y != __ldg(p.cu_q + w.seq + 1)))
      set_status(p.status, RKV_ERR_INDEX_OUT_OF_RANGE);
  }
  const int tiles = w.tokens > p.tile_tokens ? 2 : 1;

  if (warp >= kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp < kMmaWarp + 2 && w.steps > 0) {
      // ----------------------------------------------------------- MMA issuers
      // The whole warp waits, so that it stays converged; one lane issues.
      constexpr uint32_t kType = T::kCode == RKV_GQA_BF16 ? (1u << 7) | (1u << 10) : 0u;
      constexpr uint32_t kIdescS = (1u << 4) | kType | ((kN >> 3) << 17) | ((kM >> 4) << 24);
      constexpr uint32_t kIdescO = (1u << 4) | kType | (1u << 16) | ((D >> 3) << 17) | ((kM >> 4) << 24);
      const int t = warp - kMmaWarp;
      const int steps = t == tiles - 1 ? w.steps : t < tiles ? w.steps0 : 0;
      const uint64_t qd = sw128_desc(base + t * L::kQ, 16, 1024);
      const uint64_t kd0 = sw128_desc(base + L::kRing, 16, 1024), vd0 = sw128_desc(base + L::kRing, L::kCol, 1024);
      const uint32_t ts = tmem + t * 128, to = tmem + 256 + t * D;
      struct Place {  // in the ring: stage and parity of its phase
        int st;
        uint32_t ph;
        __device__ __forceinline__ void skip(int n) {
          st += n;
          if (st >= L::kStages) {
            st -= L::kStages;
            ph ^= 1u;
          }
        }
      };
      auto full = [&](const Place& at) {
        return (bool)__all_sync(0xffffffffu, mbar_wait(bars + 8 * at.st, at.ph, abort_flag));
      };
      // S of step j (one lane)
      auto qk = [&](const Place& at, int j) {
        const uint64_t kd = kd0 + (uint64_t)((at.st * L::kStage) >> 4);
        const uint32_t d = ts + (j & 1) * 64;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_ss(d, qd + (uint64_t)(((k >> 2) * L::kQCol + (k & 3) * 32) >> 4),
                 kd + (uint64_t)(((k >> 2) * L::kCol + (k & 3) * 32) >> 4), kIdescS, k > 0);
        mma_commit(bars + L::kBarS + 16 * t + 8 * (j & 1));
        mma_commit(bars + L::kBarEmpty + 8 * at.st);
      };
      bool ok = __all_sync(0xffffffffu, mbar_wait(bars + L::kBarQ, 0, abort_flag));
      Place kp = {0, 0u}, vp = {2, 0u};
      for (int j = 0; ok && j < 2 && j < w.steps; ++j, kp.skip(j)) {  // places 0, 1, 3
        ok = full(kp);
        if (!ok) break;
        if (elect_one()) {
          if (j < steps) qk(kp, j);
          else mbar_arrive(bars + L::kBarEmpty + 8 * kp.st);
        }
        __syncwarp();
      }
      for (int j = 0; ok && j < w.steps; ++j, vp.skip(2), kp.skip(2)) {
        ok = full(vp) && (j + 2 >= w.steps || full(kp));
        if (!ok) break;
        const int past = w.len - (w.step0 + j) * kN;  // first row past the sequence's end: zeros there (both warps do it)
        if (past < kN) {
          for (int i = lane; i < (kN - past) * (D / 8); i += 32) {
            const int r = past + i / (D / 8), c = i % (D / 8);
            *reinterpret_cast<uint4*>(smem + L::kRing + vp.st * L::kStage + (c >> 3) * L::kCol + r * 128 +
                                      (((c & 7) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
          __syncwarp();
        }
        if (j >= steps) {  // the other tile's steps
          if (elect_one()) {
            mbar_arrive(bars + L::kBarEmpty + 8 * vp.st);
            if (j + 2 < w.steps) mbar_arrive(bars + L::kBarEmpty + 8 * kp.st);
          }
          __syncwarp();
          continue;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(bars + L::kBarP + 16 * t + 8 * (j & 1), (j >> 1) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vd = vd0 + (uint64_t)((vp.st * L::kStage) >> 4);
          const uint32_t pa = ts + (j & 1) * 64;
#pragma unroll
          for (int k = 0; k < kN / 16; ++k)
            mma_ts(to, pa + 8 * k, vd + (uint64_t)((k * 2048) >> 4), kIdescO, (j > 0 || k > 0) ? 1u : 0u);
          mma_commit(bars + L::kBarPv + 8 * t);
          if (j == steps - 1) mma_commit(bars + L::kBarO + 8 * t);
          mma_commit(bars + L::kBarEmpty + 8 * vp.st);
          if (j + 2 < steps) qk(kp, j + 2);
          else if (j + 2 < w.steps) mbar_arrive(bars + L::kBarEmpty + 8 * kp.st);
        }
        __syncwarp();
      }
      if (!ok) {
        *abort_flag = 1;
        set_status(p.status, RKV_ERR_CUDA);
      }
      // every MMA is done before the tensor memory is freed
      if (elect_one()) mma_commit(bars + L::kBarDrain + 8 * t);
      __syncwarp();
      mbar_wait_copy(bars + L::kBarDrain + 8 * t, 0);
    } else if (warp == kLoadWarp && w.steps > 0) {
      // ---------------------------------------------------------------- loader
      const int rows_total = (int)row_base(p.cache, p.cache.n_layers, 0, 0, 0);  // out of range: zero rows
      const int v_off = p.cache.n_kv_heads * kPage;
      if (lane == 0) {
        mbar_expect_tx(bars + L::kBarQ, tiles * (D / 64) * used * 128);
        for (int t = 0; t < tiles; ++t)
          for (int c = 0; c < D / 64; ++c)
            asm volatile(
                "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
                "%4}], [%5];" ::"r"(base + t * L::kQ + c * L::kQCol),
                "l"(&qmap), "r"(64 * c), "r"(w.head * p.group), "r"(w.token + t * p.tile_tokens), "r"(bars + L::kBarQ)
                : "memory");
      }
      const int32_t* ids = p.page_table + w.seq * p.pt_stride + w.step0;
      // cache rows of the pages of 32 steps, one a lane
      auto rows_of = [&](int at) {
        int row = rows_total;
        if (at + lane < w.steps) {
          const int id = __ldg(ids + at + lane);
          if (id >= 0 && id < p.cache.n_pages) row = (int)row_base(p.cache, p.layer, id, 0, w.head);
          else set_status(p.status, RKV_ERR_INDEX_OUT_OF_RANGE);
        }
        return row;
      };
      bool ok = true;
      int filled = 0;  // places of the ring's order that were filled or skipped
      auto fill = [&](int n, int y) {
        const int st = n % L::kStages;
        if (n >= L::kStages)
          ok = __all_sync(0xffffffffu, mbar_wait(bars + L::kBarEmpty + 8 * st, (n / L::kStages - 1) & 1, abort_flag));
        if (!ok) return;
        filled = n + 1;
        if (lane == 0) {
          const uint32_t full = bars + 8 * st, dst = base + L::kRing + st * L::kStage;
          mbar_expect_tx(full, L::kStage);
#pragma unroll
          for (int c = 0; c < D / 64; ++c) tma_load_2d(dst + c * L::kCol, &map, 64 * c, y, full);
        }
      };
      int v_rows = rows_of(0), k_rows = v_rows;  // of the 32 steps that V and K are at
      fill(0, __shfl_sync(0xffffffffu, k_rows, 0));
      if (w.steps > 1) fill(1, __shfl_sync(0xffffffffu, k_rows, 1));
      for (int j = 0; ok && j < w.steps; ++j) {
        if (j > 0 && j % 32 == 0) v_rows = k_rows;
        const int y = __shfl_sync(0xffffffffu, v_rows, j % 32);
        fill(v_place(j), y == rows_total ? y : y + v_off);
        if (!ok || j + 2 >= w.steps) continue;
        if ((j + 2) % 32 == 0) k_rows = rows_of(j + 2);
        fill(k_place(j + 2), __shfl_sync(0xffffffffu, k_rows, (j + 2) % 32));
      }
      if (!ok) {
        *abort_flag = 1;
        set_status(p.status, RKV_ERR_CUDA);
      }
      // every copy has landed before the CTA ends
      mbar_wait_copy(bars + L::kBarQ, 0);
      const int skipped = 2 * w.steps - 1;  // the place of the K after the last; with one step, of K1
      for (int i = max(0, filled - L::kStages); i < filled; ++i)
        if (i != skipped) mbar_wait_copy(bars + 8 * (i % L::kStages), (i / L::kStages) & 1);
    }
  } else {
    // --------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int t = warp >> 3, b = (warp >> 2) & 1;      // tile, and which of its steps (and S buffers)
    const int r = 32 * (warp & 3) + lane;              // row of the tile
    const int token = t * p.tile_tokens + r / p.group; // of the CTA's tokens
    const bool live = w.seq >= 0 && r < used && token < w.tokens;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + lanes + t * 128 + 64 * b;
    const uint32_t to = tmem + lanes + 256 + t * D;
    const int steps = t < tiles - 1 ? w.steps0 : t < tiles ? w.steps : 0;  // a row past them sees nothing there
    const int pos = w.pos + token;                  // this row's position
    const int pos_min = w.pos + t * p.tile_tokens;  // the tile's first and last
    const int pos_max = pos_min + p.tile_tokens - 1;
    const uint32_t ref_bar = bars + L::kBarRef + 32 * t + 8 * (warp & 3);
    volatile float* ref = reinterpret_cast<volatile float*>(smem + L::kRef) + 128 * t + r;
    float m = -INFINITY;  // exponent reference of l
    float l = 0.f;        // sum of the weights of this set's steps
    bool ok = true;
    const unsigned long long c2 = dup2(p.scale_log2);
    for (int j = b; j < steps; j += 2) {
      if (!__all_sync(0xffffffffu, mbar_wait(bars + L::kBarS + 16 * t + 8 * b, (j >> 1) & 1, abort_flag))) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t x[kN];
#pragma unroll
      for (int i = 0; i < kN; i += 32) tmem_ld32(ts + i, x + i);
      tmem_wait_ld();
      const int key0 = (w.step0 + j) * kN;
      const bool masked = key0 + kN - 1 > pos_min || (p.window > 0 && key0 <= pos_max - p.window);
      if (masked) {
        const int last = pos - key0, first = p.window > 0 ? last - p.window : -1;
#pragma unroll
        for (int i = 0; i < kN; ++i)
          if (i > last || i <= first) x[i] = 0xff800000u;  // -inf
      }
      float t0 = __uint_as_float(x[0]), t1 = __uint_as_float(x[1]), t2 = __uint_as_float(x[2]),
            t3 = __uint_as_float(x[3]);
#pragma unroll
      for (int i = 4; i < kN - 4; i += 8) {
        t0 = fmax3(t0, __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
        t1 = fmax3(t1, __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
        t2 = fmax3(t2, __uint_as_float(x[i + 4]), __uint_as_float(x[i + 5]));
        t3 = fmax3(t3, __uint_as_float(x[i + 6]), __uint_as_float(x[i + 7]));
      }
      t0 = fmax3(t0, __uint_as_float(x[kN - 4]), __uint_as_float(x[kN - 3]));
      t1 = fmax3(t1, __uint_as_float(x[kN - 2]), __uint_as_float(x[kN - 1]));
      const float top = fmaxf(fmax3(t0, t1, t2), t3) * p.scale_log2 - SoftmaxBias<T>::kBias;
      // the reference that the step before left, and this step's
      float was = m;
      if (j > 0) {
        if (!__all_sync(0xffffffffu, mbar_wait(ref_bar, (j - 1) & 1, abort_flag))) {
          ok = false;
          break;
        }
        was = *ref;
      }
      const bool up = top > was + kLazyLog2 || (was == -INFINITY && top > -INFINITY);
      const float now = up ? top : was;
      *ref = now;
      __syncwarp();
      if (lane == 0) mbar_arrive(ref_bar);
      if (__any_sync(0xffffffffu, now != m)) {  // it moved in this step or in the one before
        l *= now == m ? 1.f : ex2(m - now);     // 0 from -inf
        m = now;
        if (j > 0 && __any_sync(0xffffffffu, up)) {
          const float a = up ? ex2(was - now) : 1.f;
          // O holds the steps up to j - 1 once their MMAs are done: S of this step was issued behind step j - 2's, and
          // step j's wait for this warp, so the barrier is in phase j - 1 or just past it
          if (!__all_sync(0xffffffffu, mbar_wait(bars + L::kBarPv + 8 * t, (j - 1) & 1, abort_flag))) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16(to + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
            tmem_st16(to + c, o);
          }
        }
      }
      const unsigned long long n2 = dup2(m == -INFINITY ? 0.f : -m);  // nothing seen yet: weights 0
      l += weights<T>(x, ts, c2, n2);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(bars + L::kBarP + 16 * t + 8 * b);
    }
    if (ok && steps > 0) ok = __all_sync(0xffffffffu, mbar_wait(bars + L::kBarO + 8 * t, 0, abort_flag));
    if (!ok) {
      *abort_flag = 1;
      set_status(p.status, RKV_ERR_CUDA);
    }
    tc_fence_after();
    // ---- epilogue: both sets' sums together, then one row a thread, half of its lanes a set
    if (w.seq >= 0 && t < tiles) {
      if (steps > 0) {  // through the tile's Q, which no MMA needs any more
        float2* ends = reinterpret_cast<float2*>(smem + t * L::kQ) + r;
        ends[kM * b] = make_float2(m, l);
        if (t == 0) asm volatile("bar.sync 1, 256;" ::: "memory");
        else asm volatile("bar.sync 2, 256;" ::: "memory");
        const float2 other = ends[kM * (1 - b)];
        const float mm = fmaxf(m, other.x);
        if (mm != -INFINITY) l = l * ex2(m - mm) + other.y * ex2(other.x - mm);
        m = mm;
      }
      const int head = w.head * p.group + r % p.group;
      const int64_t row = (int64_t)(w.token + token) * p.n_q_heads + head;
      const bool have = ok && steps > 0;
      float f = 1.f;
      float* part = nullptr;
      if (p.n_splits > 1) {
        const int64_t at = (int64_t)blockIdx.y * p.n_tokens * p.n_q_heads + row;
        part = p.part_o + at * D;
        if (live && b == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(have ? m : -INFINITY, l);
      } else if (live) {
        const float sink = p.sinks ? p.sinks[head] * 1.4426950408889634f : -INFINITY;
        const float top = fmaxf(m, sink);
        const float e = ex2(m - top);
        f = m == -INFINITY ? 0.f : e / (l * e + ex2(sink - top));
      }
      const bool seen = have && m != -INFINITY;  // a row that saw nothing: zeros, whatever O holds
#pragma unroll 1
      for (int c = b * (D / 2); c < (b + 1) * (D / 2); c += 32) {
        uint32_t o[32];
        if (have) {
          tmem_ld32(to + c, o);
          tmem_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = seen ? __float_as_uint(__uint_as_float(o[i]) * f) : 0u;
        if (!live) continue;
        if (part) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint4*>(part + c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 v;
            v.x = T::pack(__uint_as_float(o[i]), __uint_as_float(o[i + 1]));
            v.y = T::pack(__uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
            v.z = T::pack(__uint_as_float(o[i + 4]), __uint_as_float(o[i + 5]));
            v.w = T::pack(__uint_as_float(o[i + 6]), __uint_as_float(o[i + 7]));
            *reinterpret_cast<uint4*>(p.out + row * D + c + i) = v;
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// Joins the splits of one (token, q head) a warp, in their order.
template <typename T, int D>
__global__ void __launch_bounds__(128) join_kernel(const Params p) {
  grid_dependency_wait();
  const int64_t rows = (int64_t)p.n_tokens * p.n_q_heads;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  const int head = (int)(row % p.n_q_heads);
  const float sink = p.sinks ? p.sinks[head] * 1.4426950408889634f : -INFINITY;
  float top = sink;
  for (int i = 0; i < p.n_splits; ++i) top = fmaxf(top, p.part_ml[2 * (i * rows + row)]);
  if (top == -INFINITY) top = 0.f;
  float o[D / 32] = {};
  float l = ex2(sink - top);
  for (int i = 0; i < p.n_splits; ++i) {
    const int64_t at = i * rows + row;
    const float2 e = *reinterpret_cast<const float2*>(p.part_ml + 2 * at);
    if (e.x == -INFINITY) continue;
    const float w = ex2(e.x - top);
    l += w * e.y;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) o[j] += w * p.part_o[at * D + D / 32 * lane + j];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int j = 0; j < D / 32; j += 2)
    *reinterpret_cast<uint32_t*>(p.out + row * D + D / 32 * lane + j) = T::pack(o[j] * inv, o[j + 1] * inv);
}

template <typename T, int D>
static rkv_status launch(const Params& p, const CUtensorMap& map, const CUtensorMap& qmap, cudaStream_t s,
                         const char* what) {
  static std::atomic<bool> ready[kMaxDevicesCached];  // the shared-memory opt-in is per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevicesCached || !ready[dev].load(std::memory_order_acquire)) {
    const cudaError_t e =
        cudaFuncSetAttribute(prefill_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::kTotal);
    if (e != cudaSuccess) return fail(RKV_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    if (dev >= 0 && dev < kMaxDevicesCached) ready[dev].store(true, std::memory_order_release);
  }
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  // every sequence rounds its tokens up to whole blocks: at most one more each
  const int64_t blocks = ((int64_t)p.n_tokens / (2 * p.tile_tokens) + p.n_seq) * p.cache.n_kv_heads;
  if (blocks > INT32_MAX) return fail(RKV_ERR_SHAPE_MISMATCH, "%s: too many tokens", what);
  cfg.gridDim = dim3((unsigned)blocks, (unsigned)p.n_splits);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Layout<D>::kTotal;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, prefill_kernel<T, D>, p, map, qmap);
  if (e == cudaSuccess && p.n_splits > 1) {
    cfg.gridDim = dim3((unsigned)(((int64_t)p.n_tokens * p.n_q_heads + 3) / 4));
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, join_kernel<T, D>, p);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(RKV_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
  }
  return check_launch(what);
}

}  // namespace pre
}  // namespace gqa
}  // namespace rkv

extern "C" int32_t rkv_gqa_prefill_splits(const rkv_gqa_view* cache, int64_t n_tokens, int32_t n_q_heads,
                                          int32_t n_seq, int64_t pt_stride) {
  if (!cache || n_tokens < 0 || n_q_heads < 1 || n_seq < 0 || pt_stride < 1 || cache->n_kv_heads < 1 ||
      n_q_heads % cache->n_kv_heads != 0 || n_q_heads / cache->n_kv_heads > RKV_GQA_MAX_GROUP)
    return -1;
  // CTAs of the tokens alone; with fewer than half the SMs busy, cut the rows so that the SMs are covered, but
  // not below 16 pages
  const int64_t span = 2 * (128 / (n_q_heads / cache->n_kv_heads));
  int64_t blocks = (n_tokens + span - 1) / span;
  if (blocks < n_seq) blocks = n_seq;
  blocks *= cache->n_kv_heads;
  if (blocks == 0 || 2 * blocks > 148) return 1;
  int64_t splits = 148 / blocks;
  const int64_t most = pt_stride / 16;
  if (splits > most) splits = most;
  return splits < 1 ? 1 : splits > 64 ? 64 : (int32_t)splits;
}

extern "C" int64_t rkv_gqa_prefill_workspace_bytes(const rkv_gqa_view* cache, int64_t n_tokens, int32_t n_q_heads,
                                                   int32_t n_splits) {
  if (!cache || n_tokens < 0 || n_q_heads < 1 || n_splits < 1) return -1;
  return n_splits == 1 ? 0 : n_splits * n_tokens * n_q_heads * (cache->head_dim + 2) * 4;
}

extern "C" rkv_status rkv_gqa_prefill(const rkv_gqa_view* cache, int32_t layer, const void* q, int64_t q_token_stride,
                                      int64_t q_head_stride, int64_t n_tokens, int32_t n_q_heads, const int32_t* cu_q,
                                      int32_t n_seq, const int32_t* page_table, int64_t pt_stride,
                                      const int32_t* kv_lens, int32_t window, const float* sinks, float softmax_scale,
                                      int32_t n_splits, void* workspace, void* out, uint32_t* d_status,
                                      rkv_stream_t stream) {
  using namespace rkv;
  using namespace rkv::gqa;
  using namespace rkv::gqa::pre;
  static const char* what = "rkv_gqa_prefill";
  rkv_status st = check_cache(cache, layer, what);
  if (st != RKV_OK) return st;
  if ((st = check_heads(cache, n_q_heads, what)) != RKV_OK) return st;
  if (n_tokens < 0 || n_tokens > INT32_MAX / 2) return fail_shape("n_tokens", 0, n_tokens, "%s: bad n_tokens", what);
  if (n_seq < 0) return fail_shape("n_seq", 0, n_seq, "%s: n_seq < 0", what);
  if (n_splits < 1 || n_splits > 64) return fail_shape("n_splits", 1, n_splits, "%s: 1 <= n_splits <= 64", what);
  if (n_tokens == 0 || n_seq == 0) {
    if (n_tokens > 0) return fail_shape("n_tokens", 0, n_tokens, "%s: tokens without a sequence", what);
    clear_error();
    return RKV_OK;
  }
  const AttendArgs args = {*cache,     layer,   q,      q_token_stride, q_head_stride, n_tokens, n_q_heads, page_table,
                           pt_stride,  kv_lens, window, sinks,          softmax_scale, out,      d_status};
  if ((st = check_attend(args, what)) != RKV_OK) return st;
  if (!cu_q) return fail(RKV_ERR_INVALID_ARGUMENT, "%s: cu_q is required", what);
  if (n_splits > 1 && (!workspace || !aligned(workspace, 16)))
    return fail(RKV_ERR_INVALID_ARGUMENT, "%s: a 16-byte aligned workspace is required", what);
  Params p;
  p.cache = *cache;
  p.layer = layer;
  p.n_tokens = (int)n_tokens;
  p.n_q_heads = n_q_heads;
  p.group = n_q_heads / cache->n_kv_heads;
  p.tile_tokens = kM / p.group;
  p.cu_q = cu_q;
  p.n_seq = n_seq;
  p.page_table = page_table;
  p.pt_stride = pt_stride;
  p.kv_lens = kv_lens;
  p.window = window;
  p.sinks = sinks;
  p.scale_log2 = (float)((double)softmax_scale * 1.4426950408889634);
  p.n_splits = n_splits;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = workspace ? p.part_o + n_splits * n_tokens * n_q_heads * cache->head_dim : nullptr;
  p.out = static_cast<uint16_t*>(out);
  p.status = d_status;
  CUtensorMap map, qmap;
  if ((st = cache_map(*cache, &map, what)) != RKV_OK) return st;
  if ((st = q_map(*cache, q, q_token_stride, q_head_stride, n_tokens, n_q_heads, p.tile_tokens, p.group, &qmap, what)) != RKV_OK)
    return st;
  cudaStream_t s = (cudaStream_t)stream;
  if (cache->dtype == RKV_GQA_BF16)
    return cache->head_dim == 64 ? launch<Bf16, 64>(p, map, qmap, s, what) : launch<Bf16, 128>(p, map, qmap, s, what);
  return cache->head_dim == 64 ? launch<F16, 64>(p, map, qmap, s, what) : launch<F16, 128>(p, map, qmap, s, what);
}
