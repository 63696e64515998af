"""The grouped-head paged cache on the GPU: rotary append, page copies, prefill and decode attention against plain
64-bit implementations, at the sizes, masks and strides where they can go wrong."""
import numpy as np
import pytest
import torch

import rsllm_b200 as rk
from rsllm_b200 import GqaKvPool, RotaryTable
from tests.gqa_cases import PAGE, UNIT, Batch, close, rotate

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


# ---------------------------------------------------------------- prefill
PREFILL = [
    # q_lens, kv_lens (None: no cached prefix), hq, hkv, d, dtype, window, sinks
    ([1], None, 8, 2, 128, BF, 0, False),
    ([5], None, 8, 2, 64, HF, 0, False),
    ([63], None, 8, 8, 128, BF, 0, False),
    ([64], None, 8, 1, 128, HF, 0, True),
    ([65], None, 4, 4, 64, BF, 0, False),
    ([127, 128, 129], None, 8, 2, 128, BF, 0, False),
    ([255, 256, 257], None, 2, 2, 128, HF, 0, False),
    ([300, 1, 0, 77, 513], None, 14, 2, 128, BF, 0, True),
    ([300, 1, 0, 77, 513], None, 14, 2, 64, HF, 0, False),
    ([33, 200], [1000, 777], 16, 2, 128, HF, 0, False),
    ([33, 200], [1000, 777], 12, 4, 64, BF, 100, True),
    ([700], None, 8, 2, 128, BF, 64, False),
    ([700], None, 8, 2, 128, HF, 1, False),
    ([700, 40], [900, 1300], 8, 2, 64, BF, 129, False),
    ([50, 300], [20, 0], 8, 2, 128, BF, 0, False),     # more new tokens than rows: the first see nothing
    ([50, 300], [20, 0], 8, 2, 64, HF, 7, True),
    ([3, 2, 4], [1, 64, 65], 64, 1, 128, BF, 0, True),  # a group of 64
    ([40], [500], 40, 8, 128, HF, 0, False),            # a group of 5
    ([9] * 40, None, 8, 8, 64, BF, 0, False),
    ([1100], None, 6, 2, 128, BF, 0, False),            # a group of 3
    ([4], [5000], 8, 2, 128, BF, 0, True),
    ([2, 1], [9000, 4097], 16, 2, 64, HF, 0, False),
]


@pytest.mark.parametrize("case", range(len(PREFILL)))
def test_prefill(cuda, case):
    q_lens, kv_lens, hq, hkv, d, dtype, window, sinks = PREFILL[case]
    b = Batch(q_lens, kv_lens or q_lens, hq, hkv, d, dtype, seed=case)
    pool = GqaKvPool.over(b.cache)
    out = pool.prefill(0, b.q, b.cu_q, b.table, b.kv_lens, window=window, sinks=b.sinks if sinks else None)
    pool.check("prefill")
    close(out, *b.want(window=window, sinks=sinks), dtype)


@pytest.mark.parametrize("window", [0, 200, 3000])
@pytest.mark.parametrize("d,dtype", [(128, BF), (64, HF)])
def test_prefill_parts(cuda, window, d, dtype):
    """Few tokens and long prefixes: the rows of a token are shared out and joined, in more parts for some tokens than
    for others; tokens without a row, short ones and one long prompt among them."""
    q_lens, kv_lens = [10, 1, 33, 0, 130, 1, 700], [7000, 1, 15000, 40, 100, 0, 700]
    b = Batch(q_lens, kv_lens, 14, 2, d, dtype, seed=3)
    pool = GqaKvPool.over(b.cache)
    ws = torch.full((1 << 26,), 255, dtype=torch.uint8, device=cuda)
    out = pool.prefill(0, b.q, b.cu_q, b.table, b.kv_lens, window=window, sinks=b.sinks, workspace=ws)
    pool.check("prefill")
    close(out, *b.want(window=window, sinks=True), dtype)
    again = pool.prefill(0, b.q, b.cu_q, b.table, b.kv_lens, window=window, sinks=b.sinks, workspace=ws)
    assert torch.equal(out, again)


@pytest.mark.parametrize("seed", range(12))
def test_prefill_random_batches(cuda, seed):
    """Drawn lengths, prefixes, heads, windows: every block boundary and cut somewhere."""
    rng = np.random.default_rng(1000 + seed)
    n = int(rng.integers(1, 40))
    q_lens = [int(x) for x in rng.integers(0, [3, 60, 300, 900][seed % 4], n)]
    q_lens[0] += 1
    kv_lens = [q + int(x) for q, x in zip(q_lens, rng.integers(0, [1, 2000, 300, 64][seed // 3], n))]
    hq, hkv = [(4, 4), (14, 2), (8, 1), (12, 4), (10, 2)][seed % 5]
    dtype, d = (BF, HF)[seed % 2], (64, 128)[seed // 2 % 2]
    window = [0, 0, 37, 500][seed % 4]
    b = Batch(q_lens, kv_lens, hq, hkv, d, dtype, seed=seed)
    pool = GqaKvPool.over(b.cache)
    out = pool.prefill(0, b.q, b.cu_q, b.table, b.kv_lens, window=window, sinks=b.sinks if seed % 3 == 0 else None)
    pool.check("prefill")
    close(out, *b.want(window=window, sinks=seed % 3 == 0), dtype)


def test_prefill_strided_q_layer_scale_and_stream(cuda):
    """q as a view of a fused projection, the second of three layers, its own scale, on a stream of its own."""
    b = Batch([100, 37], [100, 200], 8, 2, 128, BF, seed=4, layers=3)
    fused = torch.full((137, 20, 128), float("nan"), dtype=BF, device=cuda)
    fused[:, 5:13] = b.q
    pool = GqaKvPool.over(b.cache)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = pool.prefill(1, fused[:, 5:13], b.cu_q, b.table, b.kv_lens, softmax_scale=0.21, stream=s)
    pool.check("prefill", stream=s)
    close(out, *b.want(layer=1, scale=0.21), BF)


def test_prefill_head_major_q(cuda):
    """Heads outermost: the head stride is larger than the token stride."""
    b = Batch([90], [150], 4, 2, 64, HF, seed=5)
    q = b.q.transpose(0, 1).contiguous().transpose(0, 1)
    pool = GqaKvPool.over(b.cache)
    close(pool.prefill(0, q, b.cu_q, b.table, b.kv_lens), *b.want(), HF)


def test_prefill_large_logits(cuda):
    """Logits of some hundreds, in growing order along a sequence, so that the running maximum keeps moving."""
    b = Batch([400], None or [400], 4, 2, 64, BF, seed=6, q_scale=40.0)
    pool = GqaKvPool.over(b.cache)
    out = pool.prefill(0, b.q, b.cu_q, b.table, b.kv_lens)
    want, mag = b.want()
    # logits of |x| < 1000 carry 2^-24 of themselves through each of their few f32 steps: 2^-12 covers 1000 * 2^-22
    close(out, want, mag, BF)


# ----------------------------------------------------------------- decode
DECODE = [
    # kv_lens, hq, hkv, d, dtype, window, sinks
    ([1], 8, 2, 128, BF, 0, False),
    ([0, 1, 2], 8, 2, 64, HF, 0, True),
    ([63, 64, 65, 0, 127, 128, 129], 8, 8, 128, HF, 0, False),
    ([1000, 1, 4000, 0, 333], 14, 2, 128, BF, 0, True),
    ([1000, 1, 4000, 0, 333], 14, 2, 64, HF, 0, False),
    ([20000], 8, 1, 128, BF, 0, False),
    ([20000, 3], 16, 2, 64, HF, 0, True),
    ([5000, 100, 64], 64, 1, 128, BF, 0, False),      # a group of 64
    ([500, 700], 34, 2, 128, HF, 0, True),            # a group of 17
    ([5000, 4096, 4097, 10], 8, 2, 128, BF, 4096, True),
    ([5000, 130, 129, 128, 127], 12, 4, 64, BF, 128, False),
    ([900, 10], 8, 2, 128, HF, 1, False),
    ([77] * 300, 4, 2, 64, BF, 0, False),
    ([int(x) for x in range(1, 400, 3)], 4, 4, 128, HF, 0, True),
]


@pytest.mark.parametrize("case", range(len(DECODE)))
def test_decode(cuda, case):
    kv_lens, hq, hkv, d, dtype, window, sinks = DECODE[case]
    b = Batch([1] * len(kv_lens), kv_lens, hq, hkv, d, dtype, seed=100 + case)
    pool = GqaKvPool.over(b.cache)
    out = pool.decode(0, b.q, b.table, b.kv_lens, window=window, sinks=b.sinks if sinks else None)
    pool.check("decode")
    close(out, *b.want(window=window, sinks=sinks), dtype)


def test_decode_is_repeatable_and_keeps_nothing(cuda):
    """The same call gives the same bits; a call in between on other data changes nothing, nor does what the
    workspace held."""
    a = Batch([1] * 9, [3000, 10, 0, 700, 64, 65, 1, 9000, 4], 16, 2, 128, BF, seed=7)
    b = Batch([1] * 3, [100, 5000, 2], 8, 2, 128, BF, seed=8)
    pa, pb = GqaKvPool.over(a.cache), GqaKvPool.over(b.cache)
    ws = torch.full((1 << 26,), 255, dtype=torch.uint8, device=cuda)
    one = pa.decode(0, a.q, a.table, a.kv_lens, workspace=ws)
    two = pb.decode(0, b.q, b.table, b.kv_lens, workspace=ws)
    three = pa.decode(0, a.q, a.table, a.kv_lens, workspace=ws)
    assert torch.equal(one, three)
    close(one, *a.want(), BF)
    close(two, *b.want(), BF)


def test_decode_in_a_graph(cuda):
    """Captured once, replayed with new lengths and new rows in the same tensors."""
    b = Batch([1] * 4, [500, 40, 1000, 7], 8, 2, 128, BF, seed=9)
    pool = GqaKvPool.over(b.cache)
    out = torch.empty_like(b.q)
    ws = torch.empty(1 << 26, dtype=torch.uint8, device=cuda)
    pool.decode(0, b.q, b.table, b.kv_lens, out=out, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pool.decode(0, b.q, b.table, b.kv_lens, out=out, workspace=ws)
    g.replay()
    torch.cuda.synchronize()
    close(out, *b.want(), BF)
    shorter = Batch([1] * 4, [300, 40, 64, 0], 8, 2, 128, BF, seed=9)
    shorter.k = [k[:, :n] for k, n in zip(b.k, [300, 40, 64, 0])]
    shorter.v = [v[:, :n] for v, n in zip(b.v, [300, 40, 64, 0])]
    shorter.q_cpu = b.q_cpu
    b.kv_lens.copy_(torch.tensor([300, 40, 64, 0], dtype=torch.int32))
    g.replay()
    torch.cuda.synchronize()
    close(out, *shorter.want(), BF)


def test_workspace_is_kept_by_stream_and_fits_every_call(cuda):
    """Calls of different head counts, on two streams and in a capture, one after another without a workspace given."""
    a = Batch([1] * 3, [3000, 700, 1], 16, 2, 128, BF, seed=20)
    b = Batch([1] * 2, [900, 2000], 64, 2, 128, BF, seed=21)
    pa, pb = GqaKvPool.over(a.cache), GqaKvPool.over(b.cache)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for pool, batch in ((pa, a), (pb, b), (pa, a)):
        with torch.cuda.stream(side):
            two = pool.decode(0, batch.q, batch.table, batch.kv_lens)
        one = pool.decode(0, batch.q, batch.table, batch.kv_lens)
        torch.cuda.synchronize()
        assert torch.equal(one, two)
        close(one, *batch.want(), BF)
    # another group of q heads on the same cache needs another size
    small = Batch([1] * 3, [3000, 700, 1], 4, 2, 128, BF, seed=22)
    small.k, small.v = a.k, a.v
    close(pa.decode(0, small.q, a.table, a.kv_lens), *small.want(), BF)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = pa.decode(0, a.q, a.table, a.kv_lens)
    eager = pa.decode(0, a.q, a.table, a.kv_lens)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, eager)


@pytest.mark.parametrize("rows", [8 * 64 - 1, 8 * 64, 8 * 64 + 1])
@pytest.mark.parametrize("op", ["prefill", "decode"])
def test_around_the_widest_table_without_a_join(cuda, rows, op):
    """Page tables of 8 pages (no join is launched) and of 9, many sequences, so that cuts fall inside them."""
    n = 70
    b = Batch([1 if op == "decode" else 5] * n, [rows - i % 40 for i in range(n)], 12, 4, 64, HF, seed=rows)
    width = (rows + 63) // 64
    table = b.table[:, :width].contiguous()
    pool = GqaKvPool.over(b.cache)
    out = pool.decode(0, b.q, table, b.kv_lens, sinks=b.sinks) if op == "decode" else \
        pool.prefill(0, b.q, b.cu_q, table, b.kv_lens, sinks=b.sinks)
    pool.check(op)
    close(out, *b.want(sinks=True), HF)


@pytest.mark.parametrize("op", ["prefill", "decode"])
def test_bad_pages_and_lengths(cuda, op):
    """A page id outside the cache reads as zero rows and is reported; a length past the page table is cut and
    reported; the call after it is clean again."""
    b = Batch([1, 1], [200, 130], 8, 2, 128, BF, seed=10, rest=0.0)
    pool = GqaKvPool.over(b.cache)
    table = b.table.clone()
    table[0, 1] = b.cache.shape[1]
    b.k[0][:, 64:128] = 0
    b.v[0][:, 64:128] = 0

    def call(table, lens):
        if op == "decode":
            return pool.decode(0, b.q, table, lens)
        return pool.prefill(0, b.q, b.cu_q, table, lens)

    out = call(table, b.kv_lens)
    assert pool.take_status() == 1 << rk.IndexOutOfRange.status
    close(out, *b.want(), BF)
    table[0, 1] = -5
    out = call(table, b.kv_lens)
    assert pool.take_status() == 1 << rk.IndexOutOfRange.status
    close(out, *b.want(), BF)
    table = b.table[:, :2].contiguous()  # 128 rows a sequence at most
    out = call(table, b.kv_lens)
    assert pool.take_status() == 1 << rk.IndexOutOfRange.status
    cut = Batch([1, 1], [128, 128], 8, 2, 128, BF, seed=10)
    cut.k, cut.v, cut.q_cpu = [k[:, :128] for k in b.k], [v[:, :128] for v in b.v], b.q_cpu
    cache_rows = b.cache[0, b.table[0, 1].long()].cpu()  # the real second page of sequence 0
    cut.k[0][0, 64:128] = cache_rows[0].transpose(0, 1)
    cut.v[0][0, 64:128] = cache_rows[1].transpose(0, 1)
    close(out, *cut.want(), BF)
    call(b.table, torch.tensor([-3, 130], dtype=torch.int32, device=cuda))
    assert pool.take_status() == 1 << rk.IndexOutOfRange.status
    call(b.table, b.kv_lens)
    assert pool.take_status() == 0


def test_cache_past_32_bit_offsets(cuda):
    """Pages whose element and byte offsets do not fit in 32 bits."""
    hkv, d, pages = 8, 128, 35000  # 4.6e9 elements
    small = Batch([1, 70], [300, 70], 16, hkv, d, BF, seed=11, rest=0.0)
    cache = torch.empty((1, pages, 2, hkv, PAGE, d), dtype=BF, device=cuda)
    used = small.cache.shape[1]
    cache[0, pages - used:] = small.cache[0]
    pool = GqaKvPool.over(cache)
    table = torch.where(small.table >= 0, small.table + pages - used, small.table)
    out = pool.prefill(0, small.q, small.cu_q, table, small.kv_lens)
    want, mag = small.want()
    close(out, want, mag, BF)
    k = torch.randn((2, hkv, d), device=cuda).to(BF)
    slots = torch.tensor([(pages - 1) * 64 + 63, (pages - 2) * 64], dtype=torch.int32, device=cuda)
    pool.append(0, k, k, slots)
    assert torch.equal(cache[0, pages - 1, 1, :, 63], k[0]) and torch.equal(cache[0, pages - 2, 0, :, 0], k[1])
    src, dst = torch.tensor([[pages - 1], [3]], dtype=torch.int32, device=cuda)
    pool.copy_pages(src, dst)
    assert torch.equal(cache[0, 3], cache[0, pages - 1])
    pool.check()
    one = Batch([1], [300], 16, hkv, d, BF, seed=11, rest=0.0)
    one.k, one.v, one.q_cpu = small.k[:1], small.v[:1], small.q_cpu[:1]
    cache[0, pages - used:] = small.cache[0]
    close(pool.decode(0, small.q[:1], table[:1], small.kv_lens[:1]), *one.want(), BF)


# ------------------------------------------------------------------ append
APPEND = [
    # tokens, hq, hkv, d, dtype, rot, sections, interleaved
    (1, 8, 2, 128, BF, 128, None, False),
    (77, 14, 2, 64, HF, 64, None, True),
    (130, 5, 5, 128, HF, 64, None, False),
    (33, 8, 1, 128, BF, 128, (16, 24, 24), False),
    (33, 8, 1, 128, BF, 128, (3, 60, 1), True),
    (20, 3, 3, 64, HF, 32, (5, 5, 3, 3), False),
    (300, 28, 4, 64, BF, 16, (4, 4), True),
]


@pytest.mark.parametrize("case", range(len(APPEND)))
@pytest.mark.parametrize("fused", [False, True])
def test_append(cuda, case, fused):
    n, hq, hkv, d, dtype, rot, sections, inter = APPEND[case]
    g = torch.Generator().manual_seed(case)
    rows, pages = 500, (n + PAGE - 1) // PAGE + 2
    qkv = torch.randn((n, hq + 2 * hkv, d), generator=g).to(dtype)
    rt = RotaryTable.build(rows, rot, sections=sections, interleaved=inter, device=cuda)
    axes = len(rt.sections)
    pos = torch.randint(0, rows, (axes, n), generator=g, dtype=torch.int32)
    slots = torch.randperm(pages * PAGE, generator=g)[:n].to(torch.int32)
    slots[n // 2] = -1  # a token that is rotated but not stored
    x = qkv.to(cuda)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    cache = torch.full((2, pages, 2, hkv, PAGE, d), 7.0, dtype=dtype, device=cuda)
    pool = GqaKvPool.over(cache)
    got = pool.append(1, k, v, slots.to(cuda), q=q, rotary=rt, pos=pos.to(cuda) if axes > 1 else pos[0].to(cuda))
    pool.check("append")
    table = rt.table.cpu()
    u = UNIT[dtype]
    for part, have in ((qkv[:, :hq], got.cpu()), (qkv[:, hq:hq + hkv], None)):
        want = rotate(part, table, pos, rt.sections, inter)
        if have is None:
            kept = slots >= 0
            s = slots[kept].long()
            have, want, part = cache[1].cpu()[s // PAGE, 0, :, s % PAGE], want[kept], part[kept]
        # two products and a sum in f32, one rounding to the type
        bound = u * want.abs() + 2.0 ** -22 * part.double().abs().amax(-1, keepdim=True) + 2.0 ** -25
        assert ((have.double() - want).abs() <= bound).all()
    s = slots[slots >= 0].long()
    assert torch.equal(cache[1].cpu()[s // PAGE, 1, :, s % PAGE], qkv[:, hq + hkv:][slots >= 0])
    untouched = torch.ones(pages * PAGE, dtype=torch.bool)
    untouched[s] = False
    r = torch.arange(pages * PAGE)[untouched]
    assert (cache[1].cpu()[r // PAGE, :, :, r % PAGE] == 7).all() and (cache[0] == 7).all()


def test_append_without_rotary_and_in_place_q(cuda):
    k, v = torch.randn((2, 100, 4, 64), device=cuda).to(HF)
    pool = GqaKvPool(4, 4, 64, dtype=HF)
    slots = torch.arange(100, dtype=torch.int32, device=cuda) + 64
    assert pool.append(0, k, v, slots) is None
    got = pool.cache[0, 1:3].permute(0, 3, 1, 2, 4).reshape(128, 2, 4, 64)[:100]
    assert torch.equal(got[:, 0], k) and torch.equal(got[:, 1], v)
    rt = RotaryTable.build(200, 64, device=cuda)
    q = torch.randn((100, 8, 64), device=cuda).to(HF)
    pos = torch.arange(100, dtype=torch.int32, device=cuda)
    apart = pool.append(0, k, v, slots, q=q, rotary=rt, pos=pos)
    same = pool.append(0, k, v, slots, q=q, rotary=rt, pos=pos, q_out=q)
    assert same is q and torch.equal(apart, q)
    pool.check()


def test_append_refuses_rows_on_the_device(cuda):
    """Not finite: that head's row is not written; a bad slot or position: none of the token's."""
    hkv, d = 4, 128
    cache = torch.full((1, 3, 2, hkv, PAGE, d), 7.0, dtype=BF, device=cuda)
    pool = GqaKvPool.over(cache)
    k, v = torch.randn((2, 6, hkv, d), device=cuda).to(BF)
    k[1, 2, 127] = float("inf")
    v[2, 0, 0] = float("nan")
    slots = torch.tensor([0, 1, 2, 3, 192, 5], dtype=torch.int32, device=cuda)
    pool.append(0, k, v, slots)
    assert pool.take_status() == (1 << rk.NonFiniteInput.status) | (1 << rk.IndexOutOfRange.status)
    rows = cache[0, 0, :, :, :6]  # [2, hkv, 6, d]
    want = torch.stack((k, v)).transpose(1, 2).clone()
    want[0, 2, 1] = 7
    want[1, 0, 2] = 7
    want[:, :, 4] = 7
    assert torch.equal(rows, want)
    rt = RotaryTable.build(10, 128, device=cuda)
    cache.fill_(7)
    pos = torch.tensor([0, 9, 10, -1, 3, 4], dtype=torch.int32, device=cuda)
    q = torch.randn((6, 8, d), device=cuda).to(BF)
    slots = torch.arange(6, dtype=torch.int32, device=cuda)
    k, v = torch.randn((2, 6, hkv, d), device=cuda).to(BF)
    got = pool.append(0, k, v, slots, q=q, rotary=rt, pos=pos)
    assert pool.take_status() == 1 << rk.IndexOutOfRange.status
    assert (got[2:4] == 0).all() and (got[:2] != 0).any() and (got[4:] != 0).any()
    assert (cache[0, 0, :, :, 2:4] == 7).all()
    assert torch.equal(cache[0, 0, 1, :, 4:6], v[4:6].transpose(0, 1))
    # a value that overflows only when it is rotated and rounded
    big = torch.full((1, hkv, d), 60000.0, dtype=HF, device=cuda)
    half = GqaKvPool(1, hkv, d, dtype=HF)
    half.append(0, big, big, slots[:1], rotary=rt, pos=pos[4:5])
    assert half.take_status() == 1 << rk.NonFiniteInput.status
    assert (half.cache[0, 0, 0] == 0).all() and torch.equal(half.cache[0, 0, 1, :, 0], big[0])


# ------------------------------------------------------------------- copies
@pytest.mark.parametrize("hkv,d,layers,n", [(1, 64, 1, 1), (2, 64, 3, 5), (8, 128, 2, 33), (5, 128, 1, 7)])
def test_copy_pages(cuda, hkv, d, layers, n):
    total = 2 * n + 2
    cache = torch.randn((layers, total, 2, hkv, PAGE, d), device=cuda).to(BF)
    before = cache.clone()
    ids = torch.randperm(total).to(torch.int32).to(cuda)
    pool = GqaKvPool.over(cache)
    pool.copy_pages(ids[:n].contiguous(), ids[n:2 * n].contiguous())
    pool.check("copy")
    before[:, ids[n:2 * n].long()] = before[:, ids[:n].long()]
    assert torch.equal(cache, before)


def test_copy_pages_bad_ids_and_empty(cuda):
    cache = torch.randn((2, 6, 2, 2, PAGE, 64), device=cuda).to(HF)
    before = cache.clone()
    pool = GqaKvPool.over(cache)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    pool.copy_pages(i32(0, 6, 1, -1), i32(2, 3, 7, 4))
    assert pool.take_status() == 1 << rk.IndexOutOfRange.status
    before[:, 2] = before[:, 0]
    assert torch.equal(cache, before)
    pool.copy_pages(i32(), i32())
    pool.check()


def test_apply_moves_keeps_their_order(cuda):
    rng = np.random.default_rng(0)
    cache = torch.randn((2, 30, 2, 1, PAGE, 64), device=cuda).to(BF)
    want = cache.clone()
    src, dst = rng.integers(0, 30, 60), rng.integers(0, 30, 60)
    keep = src != dst
    src, dst = src[keep], dst[keep]
    for a, b in zip(src, dst):
        want[:, b] = want[:, a]
    pool = GqaKvPool.over(cache)
    pool.apply_moves(src, dst)
    pool.check()
    assert torch.equal(cache, want)


# ----------------------------------------------------------------- refusals
def test_python_refusals(cuda):
    pool = GqaKvPool(4, 2, 128)
    q = torch.zeros((1, 8, 128), dtype=BF, device=cuda)
    kv = torch.zeros((1, 2, 128), dtype=BF, device=cuda)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    table = i32(0, 1).view(1, 2)
    bad = [
        lambda: pool.decode(0, q.half(), table, i32(5)),
        lambda: pool.decode(0, q.cpu(), table, i32(5)),
        lambda: pool.decode(0, q[:, :, :64], table, i32(5)),
        lambda: pool.decode(0, q, table, i32(5, 6)),
        lambda: pool.decode(0, q, table.long(), i32(5)),
        lambda: pool.decode(0, q[:, :7], table, i32(5)),
        lambda: pool.decode(0, q, table, i32(5), window=-1),
        lambda: pool.decode(0, q, table, i32(5), sinks=torch.zeros(7, device=cuda)),
        lambda: pool.decode(0, q, table, i32(5), out=q[:, :4]),
        lambda: pool.decode(0, q, table, i32(5), workspace=torch.zeros(8, device=cuda, dtype=torch.uint8)),
        lambda: pool.prefill(0, q, i32(0, 1, 1), table, i32(5)),
        lambda: pool.prefill(0, q, i32(0, 1), table, i32(5), workspace=torch.zeros(8, device=cuda, dtype=torch.uint8)),
        lambda: pool.prefill(0, torch.zeros((1, 8, 132), dtype=BF, device=cuda)[:, :, :128], i32(0, 1), table, i32(5)),
        lambda: pool.append(0, kv, kv[:0], i32(1)),
        lambda: pool.append(0, kv, kv, i32(1, 2)),
        lambda: pool.append(0, kv[:, :1], kv, i32(1)),
        lambda: pool.append(0, kv, kv, i32(1), rotary=RotaryTable.build(4, 64), pos=None),
        lambda: pool.append(0, kv, kv, i32(1), rotary=RotaryTable.build(4, 64, sections=(8, 8)), pos=i32(0, 0).view(2, 1)),
        lambda: pool.append(0, kv, kv, i32(1), rotary=RotaryTable.build(4, 40), pos=i32(0)),
        lambda: pool.copy_pages(i32(1), i32(1, 2)),
        lambda: GqaKvPool.over(torch.zeros((1, 2, 2, 2, 32, 64), dtype=BF, device=cuda)),
        lambda: GqaKvPool(4, 2, 96),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(rk.ShapeMismatch):
            f()
            pytest.fail(f"call {i} was accepted")
    with pytest.raises(rk.InvalidLayer):
        pool.decode(1, q, table, i32(5))
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(rk.InvalidArgument):
            pool.decode(0, q, table, i32(5), softmax_scale=scale)
    with pytest.raises(rk.InvalidArgument):
        pool.append(0, kv, kv, i32(1), q=q)
    with pytest.raises(rk.InvalidArgument):
        GqaKvPool(4, 2, 64, dtype=torch.float32)
    # nothing to do is no error
    assert pool.decode(0, q[:0], table[:0], i32()).shape == (0, 8, 128)
    assert pool.prefill(0, q[:0], i32(0, 0), table, i32(5)).shape == (0, 8, 128)
    pool.append(0, kv[:0], kv[:0], i32())
    pool.check()
