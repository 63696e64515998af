"""More of the grouped-head paged cache on the GPU: what only shows over many steps, at the ends of the arguments'
ranges, with values that are not finite, and from several threads."""
import random
import threading

import pytest
import torch

import rsllm_b200 as rk
from rsllm_b200 import GqaKvPool
from tests.gqa_cases import UNIT, Batch, close

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


# ---------------------------------------------------------- tensor memory
@pytest.mark.parametrize("d,dtype", [(128, BF), (64, HF)])
def test_prefill_repeats_itself(cuda, d, dtype):
    """Every run gives the same bits: the buffers of S, P and O in tensor memory are never overwritten before they are
    read, whatever else the tensor cores are at.  The logits grow along the sequences, so that O is rescaled too."""
    b = Batch([1500, 700, 3], [1500, 2700, 4000], 8, 2, d, dtype, seed=30, q_scale=8.0)
    pool = GqaKvPool.over(b.cache)
    first = pool.prefill(0, b.q, b.cu_q, b.table, b.kv_lens)
    close(first, *b.want(), dtype)
    for _ in range(40):
        assert torch.equal(pool.prefill(0, b.q, b.cu_q, b.table, b.kv_lens), first)
    pool.check("prefill")


# ------------------------------------------------------- windows without end
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 30, 2 ** 30, 640, 639])
@pytest.mark.parametrize("op", ["prefill", "decode"])
def test_widest_windows(cuda, op, window):
    """The largest int as "no window", with fewer rows than new tokens among the sequences; and windows of just the
    rows that the page tables hold (10 pages) and one fewer."""
    q_lens, kv_lens = ([50, 300, 4, 70], [20, 0, 1, 576]) if op == "prefill" else ([1] * 4, [576, 0, 1, 130])
    b = Batch(q_lens, kv_lens, 8, 2, 128, BF, seed=31)
    assert b.table.shape[1] == 10
    pool = GqaKvPool.over(b.cache)
    if op == "prefill":
        out = pool.prefill(0, b.q, b.cu_q, b.table, b.kv_lens, window=window)
    else:
        out = pool.decode(0, b.q, b.table, b.kv_lens, window=window)
    pool.check(op)
    close(out, *b.want(window=window), BF)


# ---------------------------------------------------------------- threads
@pytest.mark.parametrize("op", ["prefill", "decode"])
def test_two_threads_on_one_stream(cuda, op):
    """Both queue calls whose rows are shared out and joined, on the default stream; each gets its own results."""
    batches = [Batch([1] * 3 if op == "decode" else [3, 20, 1], lens, 8, 2, 128, BF, seed=33 + i)
               for i, lens in enumerate(([3000, 7000, 900], [9000, 400, 2500]))]
    cache = torch.cat([b.cache for b in batches], dim=1)
    tables = [batches[0].table, torch.where(batches[1].table >= 0, batches[1].table + batches[0].cache.shape[1], -1)]
    pool = GqaKvPool.over(cache)

    def call(i):
        b = batches[i]
        if op == "decode":
            return pool.decode(0, b.q, tables[i], b.kv_lens)
        return pool.prefill(0, b.q, b.cu_q, tables[i], b.kv_lens)

    alone = [call(i) for i in range(2)]
    for out, b in zip(alone, batches):
        close(out, *b.want(), BF)
    torch.cuda.synchronize()
    results = [[], []]
    start = threading.Barrier(2)

    def work(i):
        start.wait()
        for _ in range(300):
            results[i].append(call(i))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    pool.check(op)
    for i in range(2):
        assert len(results[i]) == 300 and all(torch.equal(r, alone[i]) for r in results[i])


# ------------------------------------------------------------------- NaN
@pytest.mark.parametrize("kv", [1, 40, 700, 9000])
@pytest.mark.parametrize("d,dtype", [(128, BF), (64, HF)])
@pytest.mark.parametrize("op", ["prefill", "decode"])
def test_nan_is_not_taken_for_an_empty_row(cuda, op, d, dtype, kv):
    """A q row, or every K row that a token sees, of NaN: the result is NaN, not the zeros of a token that sees nothing,
    with rows shared out or not, with sinks or not; every other result keeps its bits."""
    q_lens = [1, 1, 1] if op == "decode" else [min(kv, 30), 5, 1]
    b = Batch(q_lens, [kv, 300, 0], 8, 2, d, dtype, seed=35)
    pool = GqaKvPool.over(b.cache)

    def call(q, sinks):
        if op == "decode":
            return pool.decode(0, q, b.table, b.kv_lens, sinks=sinks)
        return pool.prefill(0, q, b.cu_q, b.table, b.kv_lens, sinks=sinks)

    for sinks in (None, b.sinks):
        clean = call(b.q, sinks)
        close(clean, *b.want(sinks=sinks is not None), dtype)
        q = b.q.clone()
        q[0, 5] = float("nan")
        out = call(q, sinks)
        assert out[0, 5].isnan().all()
        out[0, 5] = clean[0, 5]
        assert torch.equal(out, clean)
        # row 0 of kv head 1 in the first sequence: the tokens that see no other row see nothing else
        page = int(b.table[0, 0])
        kept = b.cache[0, page, 0, 1].clone()
        b.cache[0, page, 0, 1, 0] = float("nan")
        out = call(b.q, sinks)
        b.cache[0, page, 0, 1] = kept
        assert out[:q_lens[0], 4:].isnan().all()
        out[:q_lens[0], 4:] = clean[:q_lens[0], 4:]
        assert torch.equal(out, clean)
        pool.check(op)


# ------------------------------------------------------------- the weights
@pytest.mark.parametrize("hq,hkv,d,dtype,sinks", [(16, 2, 128, BF, False), (8, 8, 64, BF, True), (34, 2, 128, HF, False),
                                                  (4, 4, 64, HF, True)])
def test_decode_weights_keep_their_bits(cuda, hq, hkv, d, dtype, sinks):
    """Few rows, so that their weights are large and their errors do not average out.  The weights' two terms hold them
    to 2^-16, the exponentials and logits are good to 2^-13 each in numerator and denominator (2^-12 sum w |v| in
    all), and the output is rounded once (u |out|); 1e-6 for f16 results near the subnormals.  One term would
    add u sum w |v|."""
    kv_lens = [1, 2, 3, 4, 5, 7, 9, 16, 17, 33, 64, 65, 100, 900]
    b = Batch([1] * len(kv_lens), kv_lens, hq, hkv, d, dtype, seed=36)
    pool = GqaKvPool.over(b.cache)
    out = pool.decode(0, b.q, b.table, b.kv_lens, sinks=b.sinks if sinks else None).double().cpu()
    pool.check("decode")
    want, mag = b.want(sinks=sinks)
    over = (out - want).abs() - ((2.0 ** -12 + 2.0 ** -16) * mag + UNIT[dtype] * want.abs() + 1e-6)
    assert over.max().item() <= 0, f"off by {over.max().item():.3g} more than the bound"


# ---------------------------------------------------------------- strides
def test_broadcast_q_k_and_v(cuda):
    """One q row for every sequence, and one k and v row for every token, as expanded views: decode and append take
    them as they are, prefill refuses them."""
    b = Batch([1] * 3, [70, 1, 300], 8, 2, 128, BF, seed=37)
    pool = GqaKvPool.over(b.cache)
    q = b.q[:1].expand(3, 8, 128)
    assert torch.equal(pool.decode(0, q, b.table, b.kv_lens), pool.decode(0, q.contiguous(), b.table, b.kv_lens))
    with pytest.raises(rk.ShapeMismatch):
        pool.prefill(0, q, b.cu_q, b.table, b.kv_lens)
    one = pool.prefill(0, b.q[:1], b.cu_q[:2], b.table[:1], b.kv_lens[:1])
    row = torch.randn((1, 1, 128), device=cuda).to(BF).expand(5, 2, 128)
    slots = torch.arange(5, dtype=torch.int32, device=cuda) + 64 * int(b.table[2, 4])
    pool.append(0, row, row, slots)
    pool.check()
    assert (b.cache[0, int(b.table[2, 4]), :, :, :5] == row[0, 0]).all()
    close(one, *[x[:1] for x in b.want()], BF)


# ------------------------------------------------------------- the ring
@pytest.mark.parametrize("n,least,most,hq,hkv,d,dtype,window", [
    (9, 626, 5713, 40, 8, 64, HF, 0),
    (30, 0, 4110, 4, 4, 64, HF, 0),
    (35, 71, 1602, 28, 4, 64, BF, 0),
    (30, 0, 27158, 8, 8, 64, BF, 1024),
    (36, 0, 4379, 4, 4, 128, BF, 1024),
])
def test_decode_repeats_itself_close_behind(cuda, n, least, most, hq, hkv, d, dtype, window):
    """Launches close behind one another, their pages in L2, so that a page is overwritten as soon as it may be: every
    one gives the same bits."""
    r = random.Random(7)
    kv_lens = [most if i == 0 else r.randint(least, most) for i in range(n)]
    b = Batch([1] * n, kv_lens, hq, hkv, d, dtype, seed=38)
    pool = GqaKvPool.over(b.cache)
    first = pool.decode(0, b.q, b.table, b.kv_lens, window=window)
    close(first, *b.want(window=window), dtype)
    other = torch.zeros(1, dtype=torch.int64, device=cuda)
    for _ in range(100):
        torch.cuda._sleep(2_000_000)  # the launches queue up behind it
        for out in [pool.decode(0, b.q, b.table, b.kv_lens, window=window) for _ in range(40)]:
            other += (out != first).any()
    pool.check("decode")
    assert int(other) == 0
