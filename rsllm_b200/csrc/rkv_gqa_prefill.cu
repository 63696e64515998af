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
// A block is two tiles of 128 q rows of one kv head, taken against a page (64
// key rows) at a time.  A tile's rows are the group's q heads of 128 / group
// consecutive tokens, token by token, so that every K and V row fetched serves
// the whole group and a tile of a long prompt has a short diagonal.
//
// One CTA runs on each SM.  The blocks of all sequences, in (sequence, head,
// tokens) order and weighed by the rows they see, are cut into equal runs, one
// for each CTA, so that ragged prompts, few tokens behind a long prefix and the
// last wave of many leave no SM idle.  A run may begin and end inside a block
// (not within 4 pages of its ends, nor in one of up to 8); such parts are
// written as partial softmaxes (m, l, O) and joined by a second small kernel.
// While a block ends, the next one's Q, K and V are copied and its first logits
// computed.
//
//   warps 0-3, 4-7  softmax of tile 0 and of tile 1, one row a thread: S from
//                   tensor memory, running maximum and sum, P (in the cache's
//                   type) back to it; the epilogue
//   warps 8, 9      issue S = Q K^T (Q, K in shared memory) and O += P V (P in
//                   tensor memory, V in shared memory) of tile 0 and of tile 1
//   warp 10         copies Q, K and V by tensor maps into a ring of stages
//   warp 11         walks the run and hands out its blocks
//
// Tensor memory of a tile: S of a step (64 columns), P of two steps (32 each), O
// (head_dim columns).  S of the next step is issued when the softmax warps have
// loaded the last one into their registers, and is there when they are done with
// it.  Two MMAs run in the order of their issue only if they have the same
// accumulator and shape, so whatever is overwritten here has been read behind a
// barrier: S when the softmax warps say so, P of step j - 2 when S of step j
// is there (the commit behind S covers the product issued before it by the same
// thread), O by its own products.
//
// An issuing thread is held up until the tensor cores are nearly done with what it
// issued, so each tile has a warp of its own for it, and what a warp waits for
// besides is asked for by a lane each, in one instruction: a barrier takes 150 to
// 250 clocks while the operand reads fill the shared memory.  (One after another
// they were 350 clocks more a step, and the issuing warp bound the step: 580 us
// for 8192 tokens.)
//
// What bounds a step of both tiles (some 1750 clocks, head_dim 128): 1280 of
// MMAs -- S with 64 columns reads 6 KB of operands for 32 clocks of products, the
// shared memory's 128 bytes a clock make it 48 -- and a chain of the softmax
// warps: 150 for the barrier of S, 80 to 110 for loads, 160 to 250 for maxima and
// masks, 930 for 64 exponentials, conversions and sums (1070 to 1280 when both
// tiles' warps meet there; 512 each at 16 a clock).
// Measured and not kept: P over its own S, with two S buffers a tile and a wait for
// the product that reads P before the S that overwrites it (642 us for 8192 tokens);
// S issued before the product of the step before it (594: P then waits for that
// product); one S buffer of 128 columns a tile, 3400-4000 clocks a step beside
// 2400 of MMAs; two sets of softmax warps taking a tile's steps in turn; the
// tiles' warps handing each other the exponentials by named barriers; a cubic on
// the FMA pipe for a quarter of the exponentials (+2%, for half of them +12%);
// other orders of the same instructions (no change); eight more warps that write
// a block's rows out (no change).
//
// 8192 tokens, 32 q and 8 kv heads of 128, bf16: 519 to 550 us, 1.0 to 1.06
// PFLOP/s, with the clock at 1.65 to 1.7 GHz under the power limit.
#include <atomic>

#include "rkv_gqa.cuh"
#include "rkv_gqa_plan.h"

namespace rkv {
namespace gqa {
namespace pre {

constexpr int kM = 128;        // q rows of a tile
static_assert(kN == kPage, "a step is a page");
constexpr int kMmaWarp = 8, kLoadWarp = 10, kPlanWarp = 11;
constexpr int kThreads = 384;
constexpr int kGrid = 148;         // one CTA an SM
constexpr int kBlockRows = 2 * kM;
constexpr int kRunCost = 8 * kN + kBlockCost;  // no more CTAs than have this much, or a block each
constexpr int kJobs = 4;           // blocks handed out ahead
constexpr uint32_t kTmemCols = 512;
// The launch has 168 registers a thread; the two softmax warpgroups take what the
// third does without.  (Calls that are not inlined do not go with it: ptxas
// does not end.)
constexpr int kSoftmaxRegs = 192, kOtherRegs = 120;
static_assert(2 * kSoftmaxRegs + kOtherRegs <= 3 * 168, "more registers than the launch has");

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
  float* part_o;   // [2 * kGrid][256 rows of a block][head_dim]
  float* part_ml;  // [2 * kGrid][256][2]
  int4* parts;     // [2 * kGrid]: first token, tokens, kv head, 1: written, 3: and the block's last
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
  static constexpr int kJob = kRing + kStages * kStage;   // [kJobs] of 64 bytes
  static constexpr int kBars = kJob + 64 * kJobs;
  static constexpr int kBarEmpty = 8 * kStages;   // full[kStages], empty[kStages]
  static constexpr int kBarS = 16 * kStages;      // S full [2][2], of even and odd steps
  static constexpr int kBarP = kBarS + 32;        // P full [2][2]
  static constexpr int kBarPv = kBarP + 32;       // O += P V of a step done [2][2]
  static constexpr int kBarO = kBarPv + 32;       // O of a block done [2]
  static constexpr int kBarOFree = kBarO + 16;    // and read [2]
  static constexpr int kBarQ = kBarOFree + 16;    // Q full, Q free
  static constexpr int kBarJob = kBarQ + 16;      // job full[kJobs], free[kJobs]
  static constexpr int kBarDrain = kBarJob + 16 * kJobs;  // [2]
  static constexpr int kBarSFree = kBarDrain + 16;        // S read [2]
  static constexpr int kMisc = kBars + kBarSFree + 16;    // TMEM address, abort flag, start of the run
  static constexpr int kScan = kMisc + 32;                // sums of the warps: costs, blocks
  static constexpr int kTotal = kScan + 12 * (kThreads / 32) + 1024;  // slack for the 1024-byte alignment
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

// The weights 2^(x scale - m) of a row's 64 logits, stored as P in the cache's
// type; returns their sum.  (A cubic on the FMA pipe in place of a
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

// The new tokens of sequence s in q: [begin, end), cut to what q holds.
__device__ __forceinline__ int2 new_tokens(const Params& p, int s) {
  const int a = min(max(__ldg(p.cu_q + s), 0), p.n_tokens);
  return make_int2(a, min(max(__ldg(p.cu_q + s + 1), a), p.n_tokens));
}

__device__ __forceinline__ Blocks blocks_of(const Params& p, int s) {
  const int2 t = new_tokens(p, s);
  Blocks b;
  b.init(t.x, t.y - t.x, min(max(__ldg(p.kv_lens + s), 0), (int)p.pt_stride * kPage), p.tile_tokens, p.window);
  return b;
}

// A block, or a part of its steps, as handed to the warps.
struct Job {
  int head, seq;
  int token;          // first token (row of q)
  int tokens;         // of both tiles
  int pos;            // position of the first token, may be negative
  int len;            // rows of the sequence
  int step0, steps;   // pages; steps < 0: no more jobs
  int steps0;         // of which tile 0 needs the first ones only
  int slot;           // of the partial result, -1: the whole block
};
static_assert(sizeof(Job) <= 64, "job slot");

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
  volatile int* start_seq = reinterpret_cast<volatile int*>(smem + L::kMisc + 8);
  volatile long long* start_off = reinterpret_cast<volatile long long*>(smem + L::kMisc + 16);
  long long* scan = reinterpret_cast<long long*>(smem + L::kScan);
  int* block_sums = reinterpret_cast<int*>(smem + L::kScan + 8 * (kThreads / 32));

  if (tid == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(bars + 8 * i, 1);
      mbar_init(bars + L::kBarEmpty + 8 * i, 2);  // both tiles
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(bars + L::kBarS + 8 * i, 1);
      mbar_init(bars + L::kBarP + 8 * i, 128);
      mbar_init(bars + L::kBarPv + 8 * i, 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(bars + L::kBarO + 8 * t, 1);
      mbar_init(bars + L::kBarOFree + 8 * t, 4);  // warps of a tile
      mbar_init(bars + L::kBarDrain + 8 * t, 1);
      mbar_init(bars + L::kBarSFree + 8 * t, 4);
    }
    mbar_init(bars + L::kBarQ, 1);
    mbar_init(bars + L::kBarQ + 8, 2);
    for (int i = 0; i < kJobs; ++i) {
      mbar_init(bars + L::kBarJob + 8 * i, 1);
      mbar_init(bars + L::kBarJob + 8 * (kJobs + i), kPlanWarp);  // every other warp
    }
    *abort_flag = 0;
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

  // ---- this CTA's run: [u0, u1) of the cost of all blocks
  long long u0, u1;
  {
    const int per = (p.n_seq + kThreads - 1) / kThreads;
    const int s_begin = min(tid * per, p.n_seq), s_end = min(s_begin + per, p.n_seq);
    long long mine = 0, blocks = 0;
    for (int s = s_begin; s < s_end; ++s) {
      const Blocks b = blocks_of(p, s);
      mine += b.before(b.count) * p.cache.n_kv_heads;
      blocks += (long long)b.count * p.cache.n_kv_heads;
      if (blockIdx.x == 0 && (b.len != __ldg(p.kv_lens + s) || b.token != __ldg(p.cu_q + s) ||
                              b.token + b.tokens != __ldg(p.cu_q + s + 1) || (s == 0 && b.token != 0) ||
                              (s == p.n_seq - 1 && b.token + b.tokens != p.n_tokens)))
        set_status(p.status, RKV_ERR_INDEX_OUT_OF_RANGE);
    }
    // the blocks count up to one for each CTA only, beside the cost in one number
    blocks = min(blocks, (long long)kGrid);
    long long upto = mine;
    int many = (int)blocks;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
      many += __shfl_xor_sync(0xffffffffu, many, o);
    }
    if (lane == 31) scan[warp] = upto;
    if (lane == 0) block_sums[warp] = many;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    long long total = 0;
    many = 0;
    for (int i = 0; i < kThreads / 32; ++i) {
      if (i < warp) upto += scan[i];
      total += scan[i];
      many += block_sums[i];
    }
    const long long ctas = min((long long)gridDim.x, max((long long)many, total / kRunCost));
    u0 = blockIdx.x < ctas ? blockIdx.x * total / ctas : total;
    u1 = blockIdx.x < ctas ? (blockIdx.x + 1) * total / ctas : total;
    long long at = upto - mine;
    if (u0 < u1 && u0 >= at && u0 < upto) {
      for (int s = s_begin; s < s_end; ++s) {
        const Blocks b = blocks_of(p, s);
        const long long n = b.before(b.count) * p.cache.n_kv_heads;
        if (u0 < at + n) {
          *start_seq = s;
          *start_off = u0 - at;
          break;
        }
        at += n;
      }
    }
    __syncthreads();
  }
  const uint32_t tmem = *tmem_slot;
  const Job* jobs = reinterpret_cast<const Job*>(smem + L::kJob);
  // The next job, copied; false after the last one or when the CTA gives up.
  int n_jobs = 0;
  auto next_job = [&](Job& w, bool& ok) {
    const int at = n_jobs % kJobs;
    ok = __all_sync(0xffffffffu, mbar_wait(bars + L::kBarJob + 8 * at, (n_jobs / kJobs) & 1, abort_flag));
    if (!ok) return false;
    w = jobs[at];
    __syncwarp();
    if (lane == 0) mbar_arrive(bars + L::kBarJob + 8 * (kJobs + at));
    ++n_jobs;
    return w.steps >= 0;
  };
  // A warp that gives up says so; the others' waits end with it.
  auto give_up = [&]() {
    *abort_flag = 1;
    set_status(p.status, RKV_ERR_CUDA);
  };

  if (warp >= kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kPlanWarp) {
      // ---------------------------------------------------------------- planner
      // The whole warp computes the same, but for the search; lane 0 writes.
      Job* out = reinterpret_cast<Job*>(smem + L::kJob);
      bool ok = true;
      int n = 0;
      auto hand_out = [&](const Job& w) {
        const int at = n % kJobs;
        // as long as the work before takes: twenty of the usual limits
        for (int i = 0; n >= kJobs && !(ok = __all_sync(0xffffffffu, mbar_wait(bars + L::kBarJob + 8 * (kJobs + at), (n / kJobs - 1) & 1, abort_flag))); ++i)
          if (i == 20 || __any_sync(0xffffffffu, *abort_flag)) return;
        if (lane == 0) {
          out[at] = w;
          mbar_arrive(bars + L::kBarJob + 8 * at);
        }
        ++n;
      };
      int4 first = make_int4(0, 0, 0, 0), last = first;  // what the two slots hold
      long long left = u1 - u0;
      if (left > 0) {
        int s = *start_seq;
        long long off = *start_off;
        for (; left > 0 && ok && s < p.n_seq; ++s, off = 0) {
          const Blocks b = blocks_of(p, s);
          const long long per_head = b.before(b.count);
          if (per_head == 0) continue;
          int head = 0;
          if (off >= per_head) {
            head = (int)(off / per_head);
            off -= head * per_head;
          }
          int lo = 0, hi = b.count;  // the block that holds `off` is in [lo, hi): 32 places are looked at together
          while (off > 0 && hi - lo > 1) {
            const int step = (hi - lo + 31) / 32;
            const int at = min(lo + lane * step, hi - 1);
            const unsigned below = __ballot_sync(0xffffffffu, b.before(at) <= off);  // lanes from 0 on
            const int k = 31 - __clz(below);
            const int from = min(lo + k * step, hi - 1);
            hi = min(hi, from + step);
            lo = from;
          }
          long long x = off - b.before(lo);
          for (; head < p.cache.n_kv_heads && left > 0 && ok; ++head, lo = 0) {
            for (int i = lo; i < b.count && left > 0 && ok; ++i, x = 0) {
              const long long cost = b.cost(i), stop = min(cost, x + left);
              const int steps = b.steps(i), k0 = cut_step(x, cost, steps), k1 = cut_step(stop, cost, steps);
              if (k1 > k0 || (steps == 0 && x == 0)) {
                Job w;
                w.head = head;
                w.seq = s;
                w.token = b.token + i * b.span;
                w.tokens = min(b.span, b.tokens - i * b.span);
                w.pos = b.pos + i * b.span;
                w.len = b.len;
                w.step0 = b.first_step(i) + k0;
                w.steps = k1 - k0;
                const int end0 = w.pos + min(w.tokens, p.tile_tokens);
                w.steps0 = max(0, min(w.steps, (end0 > 0 ? (end0 + kN - 1) / kN : 0) - w.step0));
                w.slot = -1;
                if (k1 - k0 < steps) {
                  w.slot = 2 * blockIdx.x + (k0 == 0);
                  (k0 == 0 ? last : first) = make_int4(w.token, w.tokens, head, k1 == steps ? 3 : 1);
                }
                hand_out(w);
              }
              left -= stop - x;
            }
          }
        }
      }
      if (lane == 0) {
        p.parts[2 * blockIdx.x] = first;
        p.parts[2 * blockIdx.x + 1] = last;
      }
      Job w = {};
      w.steps = -1;
      if (ok) hand_out(w);
      if (!ok) give_up();
    } else if (warp < kMmaWarp + 2) {
      // ----------------------------------------------------------- MMA issuers
      // The whole warp waits, so that it stays converged; one lane issues.
      constexpr uint32_t kType = T::kCode == RKV_GQA_BF16 ? (1u << 7) | (1u << 10) : 0u;
      constexpr uint32_t kIdescS = (1u << 4) | kType | ((kN >> 3) << 17) | ((kM >> 4) << 24);
      constexpr uint32_t kIdescO = (1u << 4) | kType | (1u << 16) | ((D >> 3) << 17) | ((kM >> 4) << 24);
      const int t = warp - kMmaWarp;
      const uint64_t qd = sw128_desc(base + t * L::kQ, 16, 1024);
      const uint64_t kd0 = sw128_desc(base + L::kRing, 16, 1024), vd0 = sw128_desc(base + L::kRing, L::kCol, 1024);
      const uint32_t ts = tmem + t * 128, to = tmem + 256 + t * D;
      struct Place {  // in the ring: stage and parity of its phase
        int st;
        uint32_t ph;
        __device__ __forceinline__ void next() {
          if (++st == L::kStages) {
            st = 0;
            ph ^= 1u;
          }
        }
      };
      auto full = [&](const Place& at) {
        return (bool)__all_sync(0xffffffffu, mbar_wait(bars + 8 * at.st, at.ph, abort_flag));
      };
      // S of the tile's step n (one lane)
      auto qk = [&](const Place& at, int n) {
        const uint64_t kd = kd0 + (uint64_t)((at.st * L::kStage) >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_ss(ts, qd + (uint64_t)(((k >> 2) * L::kQCol + (k & 3) * 32) >> 4),
                 kd + (uint64_t)(((k >> 2) * L::kCol + (k & 3) * 32) >> 4), kIdescS, k > 0);
        mma_commit(bars + L::kBarS + 16 * t + 8 * (n & 1));
        mma_commit(bars + L::kBarEmpty + 8 * at.st);
      };
      Place at = {0, 0u};
      int n = 0;       // steps of this tile so far: of step j of a job, n + j
      int n_q = 0;     // jobs with steps
      int n_o = 0;     // of which this tile had some
      Job w;
      bool ok = true;
      while (next_job(w, ok)) {
        if (w.steps == 0) continue;
        const int tiles = w.tokens > p.tile_tokens ? 2 : 1;
        const int steps = t == tiles - 1 ? w.steps : t < tiles ? w.steps0 : 0;
        ok = __all_sync(0xffffffffu, mbar_wait(bars + L::kBarQ, n_q & 1, abort_flag));
        if (steps == 0 && elect_one()) mbar_arrive(bars + L::kBarQ + 8);
        __syncwarp();
        // K and V lie in the ring in the order K0 K1 V0 K2 V1 ... V of the last step
        ok = ok && full(at);
        for (int j = -1; ok && j < w.steps; ++j) {
          if (j + 1 < w.steps) {  // S of step j + 1, once the softmax warps have read the one before it
            if (j + 1 < steps && n + j >= 0) {
              ok = __all_sync(0xffffffffu, mbar_wait(bars + L::kBarSFree + 8 * t, (n + j) & 1, abort_flag));
              if (!ok) break;
              tc_fence_after();
            }
            if (elect_one()) {
              if (j + 1 < steps) qk(at, n + j + 1);
              else mbar_arrive(bars + L::kBarEmpty + 8 * at.st);  // the other tile's steps
              if (j + 1 == steps - 1) mma_commit(bars + L::kBarQ + 8);  // Q may be overwritten
            }
            __syncwarp();
            at.next();
          }
          if (j < 0) {
            if (w.steps > 1) ok = full(at);
            continue;
          }
          // a barrier a lane: V of this step, K of the one after next, P of this step, the O of the block before read
          const Place v = at;
          at.next();
          uint32_t bar = bars + 8 * v.st, ph = v.ph;
          if ((lane & 3) == 1 && j + 2 < w.steps) bar = bars + 8 * at.st, ph = at.ph;
          if ((lane & 3) == 2 && j < steps) bar = bars + L::kBarP + 16 * t + 8 * ((n + j) & 1), ph = ((n + j) >> 1) & 1;
          if ((lane & 3) == 3 && j == 0 && steps > 0 && n_o > 0) bar = bars + L::kBarOFree + 8 * t, ph = (n_o - 1) & 1;
          ok = __all_sync(0xffffffffu, mbar_wait(bar, ph, abort_flag));
          if (!ok) break;
          tc_fence_after();
          const int past = w.len - (w.step0 + j) * kN;  // first row past the sequence's end: zeros there (both warps do it)
          if (past < kN) {
            for (int i = lane; i < (kN - past) * (D / 8); i += 32) {
              const int r = past + i / (D / 8), c = i % (D / 8);
              *reinterpret_cast<uint4*>(smem + L::kRing + v.st * L::kStage + (c >> 3) * L::kCol + r * 128 +
                                        (((c & 7) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async();
            __syncwarp();
          }
          if (elect_one()) {
            if (j < steps) {
              const uint64_t vd = vd0 + (uint64_t)((v.st * L::kStage) >> 4);
              const uint32_t pa = ts + kN + ((n + j) & 1) * (kN / 2);
#pragma unroll
              for (int k = 0; k < kN / 16; ++k)
                mma_ts(to, pa + 8 * k, vd + (uint64_t)((k * 2048) >> 4), kIdescO, (j > 0 || k > 0) ? 1u : 0u);
              mma_commit(bars + L::kBarPv + 16 * t + 8 * ((n + j) & 1));
              if (j == steps - 1) mma_commit(bars + L::kBarO + 8 * t);
              mma_commit(bars + L::kBarEmpty + 8 * v.st);
            } else {
              mbar_arrive(bars + L::kBarEmpty + 8 * v.st);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
        n += steps;
        n_q += 1;
        n_o += steps > 0;
      }
      if (!ok) give_up();
      // every MMA is done before the tensor memory is freed
      if (elect_one()) mma_commit(bars + L::kBarDrain + 8 * t);
      __syncwarp();
      mbar_wait_copy(bars + L::kBarDrain + 8 * t, 0);
    } else if (warp == kLoadWarp) {
      // ---------------------------------------------------------------- loader
      const int rows_total = (int)row_base(p.cache, p.cache.n_layers, 0, 0, 0);  // out of range: zero rows
      const int v_off = p.cache.n_kv_heads * kPage;
      Job w;
      bool ok = true;
      int n_q = 0;   // Q loads
      int n = 0;     // places of the ring filled
      auto fill = [&](int y) {
        const int st = n % L::kStages;
        if (n >= L::kStages)
          ok = __all_sync(0xffffffffu, mbar_wait(bars + L::kBarEmpty + 8 * st, (n / L::kStages - 1) & 1, abort_flag));
        if (!ok) return;
        ++n;
        if (lane == 0) {
          const uint32_t full = bars + 8 * st, dst = base + L::kRing + st * L::kStage;
          mbar_expect_tx(full, L::kStage);
#pragma unroll
          for (int c = 0; c < D / 64; ++c) tma_load_2d(dst + c * L::kCol, &map, 64 * c, y, full);
        }
      };
      while (next_job(w, ok)) {
        if (w.steps == 0) continue;
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
        int v_rows = rows_of(0), k_rows = v_rows;  // of the 32 steps that V and K are at
        // Q, once the MMAs of the job before have read theirs (twenty of the usual limits: it may be a long one)
        for (int i = 0; n_q > 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(bars + L::kBarQ + 8, (n_q - 1) & 1, abort_flag))); ++i)
          if (i == 20 || __any_sync(0xffffffffu, *abort_flag)) break;
        if (!ok) break;
        ++n_q;
        if (lane == 0) {
          const int tiles = w.tokens > p.tile_tokens ? 2 : 1;
          mbar_expect_tx(bars + L::kBarQ, tiles * (D / 64) * used * 128);
          for (int t = 0; t < tiles; ++t)
            for (int c = 0; c < D / 64; ++c)
              asm volatile(
                  "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
                  "%4}], [%5];" ::"r"(base + t * L::kQ + c * L::kQCol),
                  "l"(&qmap), "r"(64 * c), "r"(w.head * p.group), "r"(w.token + t * p.tile_tokens), "r"(bars + L::kBarQ)
                  : "memory");
        }
        fill(__shfl_sync(0xffffffffu, k_rows, 0));
        for (int j = 0; ok && j < w.steps; ++j) {  // K of step j + 1, V of step j
          if (j + 1 < w.steps) {
            if ((j + 1) % 32 == 0) k_rows = rows_of(j + 1);
            fill(__shfl_sync(0xffffffffu, k_rows, (j + 1) % 32));
            if (!ok) break;
          }
          const int y = __shfl_sync(0xffffffffu, v_rows, j % 32);
          fill(y == rows_total ? y : y + v_off);
          if ((j + 1) % 32 == 0) v_rows = k_rows;
        }
        if (!ok) break;
      }
      if (!ok) give_up();
      // every copy has landed before the CTA ends
      if (n_q > 0) mbar_wait_copy(bars + L::kBarQ, (n_q - 1) & 1);
      for (int i = max(0, n - L::kStages); i < n; ++i)
        mbar_wait_copy(bars + 8 * (i % L::kStages), (i / L::kStages) & 1);
    }
  } else {
    // --------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int t = warp >> 2;                            // tile
    const int r = 32 * (warp & 3) + lane;               // row of the tile
    const int row_token = t * p.tile_tokens + r / p.group;  // of a job's tokens
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ts0 = tmem + lanes + t * 128;
    const uint32_t to = tmem + lanes + 256 + t * D;
    const unsigned long long c2 = dup2(p.scale_log2);
    int n = 0;    // steps of this tile so far: of step j of a job, n + j
    int n_o = 0;  // jobs in which the tile had some
    bool ok = true;
    for (int n_jobs = 0;; ++n_jobs) {
      const int slot = n_jobs % kJobs;
      const Job* job = jobs + slot;
      const uint32_t job_free = bars + L::kBarJob + 8 * (kJobs + slot);
      ok = __all_sync(0xffffffffu, mbar_wait(bars + L::kBarJob + 8 * slot, (n_jobs / kJobs) & 1, abort_flag));
      if (!ok || job->steps < 0) break;
      const int tiles = job->tokens > p.tile_tokens ? 2 : 1;
      if (t >= tiles) {
        __syncwarp();
        if (lane == 0) mbar_arrive(job_free);
        continue;
      }
      const int steps = t < tiles - 1 ? job->steps0 : job->steps;  // a row past them sees nothing there
      const int row0 = job->step0 * kN - job->pos;                 // first row of step 0 from the first token's position
      const int pos_min = t * p.tile_tokens;                       // the tile's first and last position from there
      const int pos_max = pos_min + p.tile_tokens - 1;
      float m = -INFINITY;  // exponent reference of l
      float l = 0.f;        // sum of the weights
      for (int j = 0; j < steps; ++j) {
        const int b = (n + j) & 1;
        const uint32_t ts = ts0 + kN + (kN / 2) * b;  // P
        if (!__all_sync(0xffffffffu, mbar_wait(bars + L::kBarS + 16 * t + 8 * b, ((n + j) >> 1) & 1, abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t x[kN];
#pragma unroll
        for (int i = 0; i < kN; i += 32) tmem_ld32(ts0 + i, x + i);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + L::kBarSFree + 8 * t);  // S may be overwritten
        const int key0 = row0 + j * kN;
        if (key0 + kN - 1 > pos_min || (p.window > 0 && key0 <= pos_max - p.window)) {
          const int last = row_token - key0, first = p.window > 0 ? max(last, -1) - p.window : -1;
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
        const bool up = top > m + kLazyLog2 || (m == -INFINITY && top > -INFINITY);
        if (__any_sync(0xffffffffu, up)) {
          const float a = up ? ex2(m - top) : 1.f;  // 0 from -inf
          m = up ? top : m;
          l *= a;
          if (j > 0) {
            // O holds the steps up to j - 1 once their MMAs are done.  The product before on that barrier, of step j - 3,
            // was done before P of step j - 1 was written, and the one after waits for this warp's P of step j + 1.
            if (!__all_sync(0xffffffffu, mbar_wait(bars + L::kBarPv + 16 * t + 8 * (1 - b), ((n + j - 1) >> 1) & 1, abort_flag))) {
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
      if (!ok) break;
      // ---- epilogue: one row a thread
      if (steps > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(bars + L::kBarO + 8 * t, n_o & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        n += steps;
        n_o += 1;
      }
      // the rest of the job, read (and what the row needs worked out) only here: it would not fit beside S
      int row = r;
      asm volatile("" : "+r"(row));
      const Job w = *job;
      __syncwarp();
      if (lane == 0) mbar_arrive(job_free);
      const int token = t * p.tile_tokens + row / p.group;
      const bool live = row < used && token < w.tokens;
      // a row that saw nothing: zeros, whatever O holds; one that saw nothing but NaN has a sum of NaN, and is not such a row
      const bool seen = m != -INFINITY || l != 0.f;
      const int head = w.head * p.group + row % p.group;
      float f = seen ? 1.f : 0.f;
      const int64_t at = (int64_t)w.slot * kBlockRows + t * kM + row;
      if (w.slot >= 0) {
        if (live) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(m, l);
      } else if (live && seen) {
        const float sink = p.sinks ? p.sinks[head] * 1.4426950408889634f : -INFINITY;
        const float top = fmaxf(m, sink);
        const float e = ex2(m - top);
        f = e / (l * e + ex2(sink - top));
      }
      uint16_t* dst = p.out + ((int64_t)(w.token + token) * p.n_q_heads + head) * D;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        if (steps > 0) {
          tmem_ld32(to + c, o);
          tmem_wait_ld();
          if (c + 32 == D) {  // O may be overwritten
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + L::kBarOFree + 8 * t);
          }
        } else {  // set on every path: else it would live on through the next job
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = seen ? __float_as_uint(__uint_as_float(o[i]) * f) : 0u;
        if (!live) continue;
        if (w.slot >= 0) {
          if (seen)
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              st_stream32(p.part_o + at * D + c + i, make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]),
                          make_uint4(o[i + 4], o[i + 5], o[i + 6], o[i + 7]));
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 16) {
            uint32_t v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = T::pack(__uint_as_float(o[i + 2 * k]), __uint_as_float(o[i + 2 * k + 1]));
            // 32 bytes a lane: the lanes' rows are apart, and the store unit takes one of them a clock
            st_stream32(dst + c + i, make_uint4(v[0], v[1], v[2], v[3]), make_uint4(v[4], v[5], v[6], v[7]));
          }
        }
      }
    }
    if (!ok) give_up();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// Joins the parts of the block whose first part is the end of run c, in the
// order of their rows: slot 2 c + 1, then slot 2 c' of the runs after it up to the
// block's last part.  32 rows a CTA, four a warp, whose loads go out together.
constexpr int kJoinThreads = 256;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Params p) {
  __shared__ int slots[kGrid];
  __shared__ int counts[kJoinThreads / 32];
  __shared__ int ends[kJoinThreads / 32];
  grid_dependency_wait();
  const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 block = p.parts[2 * c + 1];
  if (block.w == 0 || (blockIdx.y * 32 >= kM && block.y <= p.tile_tokens)) return;
  // the list of slots: thread i looks at run c + 1 + i; those past the block's last part do not count
  const int from = c + 1 + threadIdx.x;
  int4 part = make_int4(0, 0, 0, 0);
  if (from < kGrid) part = p.parts[2 * from];
  const bool mine = part.w != 0 && part.x == block.x && part.z == block.z;  // a run whose share was cut away has none
  const unsigned has = __ballot_sync(0xffffffffu, mine), last = __ballot_sync(0xffffffffu, mine && part.w == 3);
  const unsigned upto = last ? (last & (0u - last)) | ((last & (0u - last)) - 1u) : 0xffffffffu;  // up to the first last part
  if (lane == 0) {
    counts[warp] = __popc(has & upto);
    ends[warp] = last != 0u;
  }
  __syncthreads();
  int before = 1, n = 1;
  bool ended = false;
  for (int i = 0; i < kJoinThreads / 32; ++i) {
    if (i == warp && ended) before = -1;
    if (i < warp && before > 0) before += counts[i];
    if (!ended) n += counts[i];
    ended = ended || ends[i];
  }
  if (before > 0 && mine && ((upto >> lane) & 1u)) slots[before + __popc(has & ((1u << lane) - 1u))] = 2 * from;
  if (threadIdx.x == 0) slots[0] = 2 * c + 1;
  __syncthreads();

  constexpr int kMine = 4;
  int row[kMine];
  float m[kMine], l[kMine], o[kMine][D / 32];
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    row[k] = blockIdx.y * 32 + warp + 8 * k;
    const int head = block.z * p.group + row[k] % kM % p.group;
    m[k] = p.sinks ? p.sinks[head] * 1.4426950408889634f : -INFINITY;
    l[k] = m[k] == -INFINITY ? 0.f : 1.f;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) o[k][j] = 0.f;
  }
  for (int i = 0; i < n; ++i) {
    const int64_t at = (int64_t)slots[i] * kBlockRows;
    float2 e[kMine];
    float v[kMine][D / 32];
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      e[k] = *reinterpret_cast<const float2*>(p.part_ml + 2 * (at + row[k]));
      const float* src = p.part_o + (at + row[k]) * D + D / 32 * lane;
      if constexpr (D == 128) {
        const float4 f = *reinterpret_cast<const float4*>(src);
        v[k][0] = f.x, v[k][1] = f.y, v[k][2] = f.z, v[k][3] = f.w;
      } else {
        const float2 f = *reinterpret_cast<const float2*>(src);
        v[k][0] = f.x, v[k][1] = f.y;
      }
    }
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      if (e[k].x == -INFINITY && e[k].y == 0.f) continue;  // it saw nothing there, and wrote no O
      const float top = fmaxf(m[k], e[k].x);
      const float a = ex2(m[k] - top), w = ex2(e[k].x - top);  // 0 from -inf
      l[k] = l[k] * a + e[k].y * w;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) o[k][j] = o[k][j] * a + w * v[k][j];
      m[k] = top;
    }
  }
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    const int r = row[k] % kM, token = row[k] / kM * p.tile_tokens + r / p.group;
    if (r >= p.tile_tokens * p.group || token >= block.y) continue;
    const float inv = l[k] == 0.f ? 0.f : 1.f / l[k];
    const int head = block.z * p.group + r % p.group;
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + ((int64_t)(block.x + token) * p.n_q_heads + head) * D) + D / 64 * lane;
#pragma unroll
    for (int j = 0; j < D / 64; ++j) dst[j] = T::pack(o[k][2 * j] * inv, o[k][2 * j + 1] * inv);
  }
}

template <typename T, int D>
static rkv_status launch(const Params& p, const CUtensorMap& map, const CUtensorMap& qmap, cudaStream_t s,
                         const char* what) {
  static std::atomic<bool> ready[kMaxDevicesCached];  // the shared-memory opt-in is per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevicesCached || !ready[dev].load(std::memory_order_acquire)) {
    cudaError_t e =
        cudaFuncSetAttribute(prefill_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::kTotal);
    cudaFuncAttributes built;
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&built, prefill_kernel<T, D>);
    if (e != cudaSuccess) return fail(RKV_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    // taking more registers than the launch has would wait for ever
    if (3 * built.numRegs < 2 * kSoftmaxRegs + kOtherRegs)
      return fail(RKV_ERR_CUDA, "%s: built with %d registers a thread, which the register split exceeds", what, built.numRegs);
    if (dev >= 0 && dev < kMaxDevicesCached) ready[dev].store(true, std::memory_order_release);
  }
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kGrid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Layout<D>::kTotal;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, prefill_kernel<T, D>, p, map, qmap);
  if (e == cudaSuccess && p.pt_stride > kWhole) {
    cfg.gridDim = dim3(kGrid, kBlockRows / 32);
    cfg.blockDim = dim3(kJoinThreads);
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

extern "C" int64_t rkv_gqa_prefill_workspace_bytes(const rkv_gqa_view* cache) {
  using namespace rkv::gqa::pre;
  if (!cache || (cache->head_dim != 64 && cache->head_dim != 128)) return -1;
  return (int64_t)2 * kGrid * (kBlockRows * (cache->head_dim + 2) * 4 + 16);
}

extern "C" rkv_status rkv_gqa_prefill(const rkv_gqa_view* cache, int32_t layer, const void* q, int64_t q_token_stride,
                                      int64_t q_head_stride, int64_t n_tokens, int32_t n_q_heads, const int32_t* cu_q,
                                      int32_t n_seq, const int32_t* page_table, int64_t pt_stride,
                                      const int32_t* kv_lens, int32_t window, const float* sinks, float softmax_scale,
                                      void* workspace, void* out, uint32_t* d_status, rkv_stream_t stream) {
  using namespace rkv;
  using namespace rkv::gqa;
  using namespace rkv::gqa::pre;
  static const char* what = "rkv_gqa_prefill";
  rkv_status st = check_cache(cache, layer, what);
  if (st != RKV_OK) return st;
  if ((st = check_heads(cache, n_q_heads, what)) != RKV_OK) return st;
  if (n_tokens < 0 || n_tokens > INT32_MAX / 2) return fail_shape("n_tokens", 0, n_tokens, "%s: bad n_tokens", what);
  if (n_seq < 0) return fail_shape("n_seq", 0, n_seq, "%s: n_seq < 0", what);
  if (n_tokens == 0 || n_seq == 0) {
    if (n_tokens > 0) return fail_shape("n_tokens", 0, n_tokens, "%s: tokens without a sequence", what);
    clear_error();
    return RKV_OK;
  }
  const AttendArgs args = {*cache,     layer,   q,      q_token_stride, q_head_stride, n_tokens, n_q_heads, page_table,
                           pt_stride,  kv_lens, window, sinks,          softmax_scale, out,      d_status};
  if ((st = check_attend(args, what)) != RKV_OK) return st;
  // q is copied by a tensor map, whose strides are not zero; one that nothing follows may be anything
  if ((n_tokens > 1 && q_token_stride == 0) || (n_q_heads > 1 && q_head_stride == 0))
    return fail(RKV_ERR_SHAPE_MISMATCH, "%s: q must not be a broadcast view (a stride of 0)", what);
  if (n_tokens == 1) q_token_stride = (int64_t)n_q_heads * cache->head_dim;
  if (n_q_heads == 1) q_head_stride = cache->head_dim;
  if (!cu_q) return fail(RKV_ERR_INVALID_ARGUMENT, "%s: cu_q is required", what);
  if (!workspace || !aligned(workspace, 32) || !aligned(out, 32))
    return fail(RKV_ERR_INVALID_ARGUMENT, "%s: out and a workspace, both 32-byte aligned, are required", what);
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
  p.window = window_of(window, pt_stride);
  p.sinks = sinks;
  p.scale_log2 = (float)((double)softmax_scale * 1.4426950408889634);
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + (int64_t)2 * kGrid * kBlockRows * cache->head_dim;
  p.parts = reinterpret_cast<int4*>(p.part_ml + 2 * kGrid * kBlockRows * 2);
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
