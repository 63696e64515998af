"""How the attentions of the grouped-head cache divide their work: the arithmetic that the kernels compile, compiled
for the host and held to the definition of what a token sees."""
import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "rsllm_b200" / "csrc"
INT_MAX = 2 ** 31 - 1

WRAPPER = """
#include "rkv_gqa_plan.h"
using namespace rkv::gqa;
namespace dec = rkv::gqa::dec;
using namespace rkv::gqa::pre;
static Blocks make(int tokens, int len, int tile, int window) {
  Blocks b;
  b.init(0, tokens, len, tile, window);
  return b;
}
extern "C" {
int count(int tokens, int len, int tile, int window) { return make(tokens, len, tile, window).count; }
// begin, end, first step, steps, cost of block i, and the cost of the blocks before it and up to it
void block(int tokens, int len, int tile, int window, int i, long long* out) {
  const Blocks b = make(tokens, len, tile, window);
  out[0] = b.begin(i), out[1] = b.end(i), out[2] = b.first_step(i), out[3] = b.steps(i), out[4] = b.cost(i);
  out[5] = b.before(i), out[6] = b.before(i + 1);
}
int window(int w, long long pt_stride) { return window_of(w, pt_stride); }
int joins(int slot, int last, int seq, int item, int runs, int n_seq, int items) {
  return dec::join_holds(slot, last, seq, item, runs, n_seq, items);
}
int cut(long long at, long long cost, int steps) { return cut_step(at, cost, steps); }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    cxx = shutil.which("g++")
    assert cxx, "g++ is needed to compile the plan for the host"
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cpp").write_text(WRAPPER)
    # a sum past 32 bits wraps, as it does on the device
    subprocess.run([cxx, "-std=c++17", "-O1", "-fwrapv", "-fPIC", "-shared", "-I", str(CSRC), "-o", str(at / "plan.so"),
                    str(at / "plan.cpp")], check=True)
    lib = ctypes.CDLL(str(at / "plan.so"))
    lib.block.argtypes = [ctypes.c_int] * 5 + [ctypes.POINTER(ctypes.c_longlong)]
    lib.window.argtypes = [ctypes.c_int, ctypes.c_longlong]
    lib.cut.argtypes = [ctypes.c_longlong, ctypes.c_longlong, ctypes.c_int]
    return lib


def blocks(plan, tokens, len_, tile, window):
    out = (ctypes.c_longlong * 7)()
    for i in range(plan.count(tokens, len_, tile, window)):
        plan.block(tokens, len_, tile, window, i, out)
        yield i, list(out)


def check(plan, tokens, len_, tile, window):
    total = 0
    for i, (begin, end, first, steps, cost, before, upto) in blocks(plan, tokens, len_, tile, window):
        # rows that some token of the block sees: token t at position p sees max(0, p - window + 1) .. p
        lo = len_ - tokens + i * 2 * tile
        hi = len_ - tokens + min(tokens, (i + 1) * 2 * tile) - 1
        want_end = max(0, hi + 1)
        want_begin = max(0, lo - window + 1) if window else 0
        assert (begin, end) == (want_begin, want_end), (tokens, len_, tile, window, i)
        assert steps == ((end + 63) // 64 - begin // 64 if end > begin else 0) and first == begin // 64
        assert cost == 192 + end - begin
        assert before == total and upto == total + cost, (tokens, len_, tile, window, i)
        total += cost


@pytest.mark.parametrize("window", [0, 1, 7, 4096, 1 << 30, INT_MAX - 1, INT_MAX])
@pytest.mark.parametrize("tokens,len_", [(50, 20), (50, 0), (3, 0), (700, 699), (1, 1), (1, 100000), (513, 513),
                                         (40, 33554431 * 64)])
def test_blocks_at_the_ends_of_the_ranges(plan, tokens, len_, window):
    for tile in (2, 18, 64, 128):
        check(plan, tokens, len_, tile, window)


def test_blocks_drawn(plan):
    r = random.Random(0)
    for _ in range(1500):
        tokens = r.randint(1, 10 ** r.randint(1, 4))
        len_ = r.choice([r.randint(0, tokens), tokens, tokens + r.randint(0, 100000)])
        check(plan, tokens, len_, 128 // r.randint(1, 64), r.choice([0, r.randint(1, 2 * len_ + 2), INT_MAX]))


def test_cuts_are_in_order(plan):
    r = random.Random(1)
    for _ in range(300):
        rows = r.randint(1, 5000)
        cost, steps = rows + 192, (rows + 63) // 64
        at = [plan.cut(x, cost, steps) for x in range(cost + 1)]
        assert at[0] == 0 and at[-1] == steps and at == sorted(at)
        inner = set(at) - {0, steps}
        assert not inner or (steps > 8 and min(inner) >= 4 and max(inner) <= steps - 4)


def test_a_window_as_wide_as_the_tables_is_none(plan):
    for stride in (1, 9, 33554431):
        for w in (0, 1, 63, 64, 65, 575, 576, 577, 33554431 * 64 - 1, 33554431 * 64, INT_MAX):
            assert plan.window(w, stride) == (w if w < stride * 64 else 0)


def test_join_entries_that_cannot_be_followed(plan):
    """Entries that a launch which gave up never wrote hold anything: none may lead the join out of its tables."""
    runs, n_seq, items = 296, 3, 8
    for slot, last, seq, item in [(0, 0, 0, 0), (1, 0, 2, 7), (591, 295, 0, 3), (0, 295, 2, 0)]:
        assert plan.joins(slot, last, seq, item, runs, n_seq, items)
    for slot, last, seq, item in [(-1, 0, 0, 0), (592, 296, 0, 0), (2, 0, 0, 0), (0, 296, 0, 0), (0, -1, 0, 0),
                                  (0, 5, 3, 0), (0, 5, -1, 0), (0, 5, 0, 8), (0, 5, 0, -1), (INT_MAX, INT_MAX, 0, 0),
                                  (-1, -1, -1, -1), (0x7f7f7f7f,) * 4, (0, 5, INT_MAX, 0)]:
        assert not plan.joins(slot, last, seq, item, runs, n_seq, items)
    r = random.Random(2)
    for _ in range(20000):
        e = [r.randint(-2 ** 31, 2 ** 31 - 1) if r.random() < 0.5 else r.randint(-3, 700) for _ in range(4)]
        if plan.joins(*e, runs, n_seq, items):  # every slot that the join reads, and the row it writes, exists
            first = e[0] // 2
            assert all(0 <= s < 2 * runs for s in (e[0], 2 * first, 2 * e[1])) and e[1] - first + 1 <= runs
            assert 0 <= e[2] < n_seq and 0 <= e[3] < items
