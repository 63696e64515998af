"""The grouped-head paged cache on the GPU at the sizes that its kernels are built for: several tokens and several
blocks of heads a CTA in the append, decode items in many parts, a prefill captured in a graph."""
import random

import pytest
import torch

from rsllm_b200 import GqaKvPool, RotaryTable
from tests.gqa_cases import PAGE, UNIT, Batch, close, rotate

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


# ----------------------------------------------------------------- append
@pytest.mark.parametrize("n", [593, 1500, 20011])
@pytest.mark.parametrize("hq,hkv,d,dtype,rot,sections,inter", [
    (28, 4, 128, HF, 128, (16, 24, 24), False),
    (28, 4, 64, BF, 64, None, True),
    (64, 8, 128, BF, 64, None, False),
    (64, 8, 64, HF, 64, (8, 12, 12), True),
    (0, 8, 128, BF, 128, None, False),
])
def test_append_of_many_tokens(cuda, n, hq, hkv, d, dtype, rot, sections, inter):
    """A CTA takes token after token, a thread several heads, and more heads than a CTA's go to a second one; with q
    as a view of one projection, and then in place."""
    g = torch.Generator(cuda).manual_seed(n + hq)
    rows, pages = 4000, (n + PAGE - 1) // PAGE + 1
    qkv = torch.randn((n, hq + 2 * hkv, d), generator=g, device=cuda).to(dtype)
    rt = RotaryTable.build(rows, rot, sections=sections, interleaved=inter, device=cuda)
    axes = len(rt.sections)
    pos = torch.randint(0, rows, (axes, n), generator=g, device=cuda, dtype=torch.int32)
    slots = torch.randperm(pages * PAGE, generator=g, device=cuda)[:n].to(torch.int32)
    skipped = torch.arange(n, device=cuda) % 97 == 5
    slots[skipped] = -1
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    cache = torch.full((1, pages, 2, hkv, PAGE, d), 7.0, dtype=dtype, device=cuda)
    pool = GqaKvPool.over(cache)
    got = pool.append(0, k, v, slots, q=q if hq else None, rotary=rt, pos=pos if axes > 1 else pos[0])
    pool.check("append")
    s = slots[~skipped].long()
    stored = cache[0, s // PAGE, :, :, s % PAGE]  # [tokens, 2, hkv, d]
    assert torch.equal(stored[:, 1], v[~skipped])
    u = UNIT[dtype]
    for part, have in ((q, got), (k[~skipped], stored[:, 0])):
        if have is None or not part.shape[1]:
            continue
        want = rotate(part, rt.table, pos if have is got else pos[:, ~skipped], rt.sections, inter)
        # two products and a sum in f32, one rounding to the type
        bound = u * want.abs() + 2.0 ** -22 * part.double().abs().amax(-1, keepdim=True) + 2.0 ** -25
        assert ((have.double() - want).abs() <= bound).all()
    touched = torch.zeros(pages * PAGE, dtype=torch.bool, device=cuda)
    touched[s] = True
    assert (cache[0].permute(0, 3, 1, 2, 4).flatten(0, 1)[~touched] == 7).all()
    if hq:
        own = q.contiguous()
        again = pool.append(0, k, v, slots, q=own, rotary=rt, pos=pos if axes > 1 else pos[0], q_out=own)
        assert again is own and torch.equal(own, got)


# ----------------------------------------------------------------- decode
@pytest.mark.parametrize("n,hq,hkv,d,dtype,window,sinks", [
    (20, 16, 2, 128, BF, 0, True),      # 40 items, the long ones in a dozen parts
    (12, 12, 4, 64, HF, 3000, False),
    (12, 28, 4, 64, BF, 0, True),
    (11, 34, 2, 128, HF, 0, False),     # groups of 17: two chunks of heads
    (38, 40, 1, 64, BF, 2000, True),    # a group of 40: three
    (64, 16, 8, 128, HF, 0, False),     # 512 items, a few parts each
])
def test_decode_items_in_many_parts(cuda, n, hq, hkv, d, dtype, window, sinks):
    """Enough (sequence, kv head) items that runs are joined run by run, some of many parts and some of one."""
    r = random.Random(n)
    kv_lens = [r.randint(600, 10000 if n * hkv < 100 else 1500) for _ in range(n)]
    kv_lens[1], kv_lens[-1] = 0, 65
    b = Batch([1] * n, kv_lens, hq, hkv, d, dtype, seed=n)
    pool = GqaKvPool.over(b.cache)
    ws = torch.full((1 << 24,), 255, dtype=torch.uint8, device=cuda)
    out = pool.decode(0, b.q, b.table, b.kv_lens, window=window, sinks=b.sinks if sinks else None, workspace=ws)
    pool.check("decode")
    close(out, *b.want(window=window, sinks=sinks), dtype)
    again = pool.decode(0, b.q, b.table, b.kv_lens, window=window, sinks=b.sinks if sinks else None, workspace=ws)
    assert torch.equal(out, again)


# ---------------------------------------------------------------- prefill
def test_prefill_in_a_graph(cuda):
    """Captured once, replayed with other lengths in the same tensors: the work is divided anew, on the device."""
    b = Batch([40, 3, 200], [3000, 90, 200], 8, 2, 128, BF, seed=41)
    pool = GqaKvPool.over(b.cache)
    out = torch.empty_like(b.q)
    pool.prefill(0, b.q, b.cu_q, b.table, b.kv_lens, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pool.prefill(0, b.q, b.cu_q, b.table, b.kv_lens, out=out)
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    close(out, *b.want(), BF)
    # the same 243 tokens shared out otherwise over shorter sequences
    lens, cu = [700, 60, 183], [0, 30, 60, 243]
    other = Batch([30, 30, 183], lens, 8, 2, 128, BF, seed=41)
    other.k = [k[:, :m] for k, m in zip(b.k, lens)]
    other.v = [v[:, :m] for v, m in zip(b.v, lens)]
    other.q_cpu = b.q_cpu
    b.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    b.cu_q.copy_(torch.tensor(cu, dtype=torch.int32))
    g.replay()
    torch.cuda.synchronize()
    close(out, *other.want(), BF)
    pool.check("prefill")
