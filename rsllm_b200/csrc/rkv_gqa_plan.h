// rkv_gqa_plan.h -- how the attentions of the grouped-head cache divide their
// work: the blocks of a prefill's sequence, what they weigh, where they may be
// cut; what decode's join takes.  Plain arithmetic, the same on the device and
// on the host.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define RKV_PLAN_FN __host__ __device__ __forceinline__
#else
#define RKV_PLAN_FN inline
#endif

namespace rkv {
namespace gqa {

// The window as the kernels take it: one as wide as the page tables hides nothing (the largest int is a usual way to
// say so) and is none.
RKV_PLAN_FN int32_t window_of(int32_t window, int64_t pt_stride) { return window < pt_stride * 64 ? window : 0; }

namespace pre {

constexpr int kN = 64;             // key rows of a step: a page
constexpr int kBlockCost = 192;    // what a block costs beside its rows, in rows
constexpr int kWhole = 8;          // steps that are not shared out: with page tables no wider, no join is launched

RKV_PLAN_FN int lesser(int a, int b) { return a < b ? a : b; }
RKV_PLAN_FN int larger(int a, int b) { return a > b ? a : b; }

// A sequence's blocks for one kv head.  Block i has the tokens [i span, (i + 1)
// span) and sees the rows [begin(i), end(i)); it weighs as many and kBlockCost.
struct Blocks {
  int token, tokens, len, pos, span, window, count;
  // `tokens_` tokens from `token_` on, the last of the sequence's `len_` rows; `window_` 0: none
  RKV_PLAN_FN void init(int token_, int tokens_, int len_, int tile_tokens, int window_) {
    token = token_;
    tokens = tokens_;
    len = len_;
    pos = len - tokens;  // position of the first token, may be negative
    span = 2 * tile_tokens;
    window = window_;
    count = (tokens + span - 1) / span;
  }
  RKV_PLAN_FN int end(int i) const { return larger(0, pos + lesser(tokens, (i + 1) * span)); }
  RKV_PLAN_FN int begin(int i) const {
    // in 64 bits: with a negative position and a wide window it does not fit in 32
    const long long row = (long long)pos + i * span - window + 1;
    return window > 0 && row > 0 ? (int)row : 0;
  }
  RKV_PLAN_FN long long cost(int i) const { return (long long)kBlockCost + end(i) - lesser(begin(i), end(i)); }
  // sum over i < n of max(0, a + i span)
  RKV_PLAN_FN long long ramp(long long n, long long a) const {
    const long long i0 = a > 0 ? 0 : (-a) / span + 1;  // the first above zero
    if (i0 >= n) return 0;
    return (n - i0) * a + span * (n * (n - 1) / 2 - i0 * (i0 - 1) / 2);
  }
  // cost of the blocks before n
  RKV_PLAN_FN long long before(int n) const {
    long long c = (long long)n * kBlockCost + ramp(n, (long long)pos + span);
    if (window > 0) c -= ramp(n, (long long)pos - window + 1);
    if (n == count && n > 0) c -= (long long)pos + (long long)n * span - len;  // the last one may be short
    return c;
  }
  RKV_PLAN_FN int first_step(int i) const { return begin(i) / kN; }
  RKV_PLAN_FN int steps(int i) const { return end(i) > begin(i) ? (end(i) + kN - 1) / kN - begin(i) / kN : 0; }
};
// Where a cut at `at` of a block's cost goes: its step.  Blocks of up to kWhole
// steps stay whole, longer ones are not cut within 4 of their ends.
RKV_PLAN_FN int cut_step(long long at, long long cost, int steps) {
  if (at <= 0) return 0;
  if (at >= cost) return steps;
  if (steps <= kWhole) return 2 * at >= cost ? steps : 0;
  const int k = (int)(at * steps / cost);
  return k < 4 ? 0 : steps - k < 4 ? steps : k;
}

}  // namespace pre

namespace dec {

// Whether an entry of the join's list can be followed: its first slot, the last run, the sequence and the item of it.
// A launch that gave up (a wait that ran out) leaves entries unwritten, with whatever the workspace held.
RKV_PLAN_FN bool join_holds(int slot, int last, int seq, int item, int runs, int n_seq, int items) {
  return slot >= 0 && slot / 2 <= last && last < runs && seq >= 0 && seq < n_seq && item >= 0 && item < items;
}

}  // namespace dec
}  // namespace gqa
}  // namespace rkv
