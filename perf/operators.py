"""The operators of the grouped-head (GQA) paged KV cache, case by case: what a
serving engine calls for a model with separate K and V heads.

* ``append``  rotary positions of q and k (one or several axes) and the store of
              k and v into their pages,
* ``copy``    whole-page moves (copy-on-write, compaction),
* ``prefill`` causal attention of packed prompts over the pages, cached prefix
              included,
* ``decode``  attention of one new token per sequence over the pages.

``run`` computes them in elementary torch operations in 32 bits, or, where
``own`` is true, through ``rsllm_b200.GqaKvPool``.  The cache is a tensor
``[layers, pages, 2 (k, v), kv_heads, 64, head_dim]``; a slot is page * 64 + row.
"""
import math
import random

import torch

own = False

PAGE = 64
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
TABLE_ROWS = 32768  # positions the rotary table covers


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of 256 running sequences: each token rotated and stored in its sequence's last page
        _append("append_step", 256, True, 32, 8, 128, "bf16", 128, False, 1),
        # a long prompt with images: three position axes (time, height, width), consecutive slots
        _append("append_axes_prompt", 20011, False, 28, 4, 128, "f16", 128, False, 3),
        # forks of a small model's sequences writing into shared last pages
        _copy("copy_on_write", 9, 1, 2, 64, "bf16"),
        # compaction of a pool after an eviction
        _copy("copy_compaction", 2500, 1, 8, 128, "bf16"),
        # a single chat user early in a conversation: latency of one token
        _decode("decode_single", 1, 777, 777, 32, 8, 128, "bf16", 0, False),
        # the attention read of the 64-sequence batch at context 32768
        _decode("decode_batch", 64, 32768, 32768, 32, 8, 128, "bf16", 0, False),
        # a mixed batch, some slots of it empty, of a model with a sliding window, sinks and 7 heads a group
        _decode("decode_ragged_window", 256, 0, 8192, 28, 4, 64, "f16", 4096, True),
        # one user with a very long document, two kv heads
        _decode("decode_long", 1, 131072, 131072, 16, 2, 128, "bf16", 0, False),
        # a few short questions prefilled together: latency to the first token
        _prefill("prefill_short", 3, 1, 90, 0, 0, 32, 8, 128, "bf16", 0, False),
        # sixteen prompts of very different lengths packed in one call
        _prefill("prefill_packed", 16, 1, 2048, 0, 0, 28, 4, 128, "f16", 0, False),
        # one long prompt
        _prefill("prefill_long", 1, 8192, 8192, 0, 0, 32, 8, 128, "bf16", 0, False),
        # new turns on a shared 8192-token prefix that is already in the pages
        _prefill("prefill_cached", 8, 64, 256, 8192, 8192, 64, 8, 64, "f16", 0, True),
    ]


def draw(rng):
    """One more case of the same ranges."""
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "copy", "prefill", "prefill", "decode", "decode"])
    dtype = rng.choice(["bf16", "f16"])
    heads = [(hq, hkv, d) for hq, hkv in ((32, 8), (64, 8), (16, 2), (28, 4), (8, 8), (40, 8), (14, 2), (32, 1), (4, 4), (12, 4))
             for d in (64, 128) if 3072 not in (hq * d, (hq + 2 * hkv) * d)]
    hq, hkv, d = rng.choice(heads)
    if op == "append":
        rot = rng.choice([r for r in (0, 32, 64, 128) if r <= d])
        axes = rng.choice([1, 1, 3]) if rot else 1
        return _append(None, log(1, 20000), rng.random() < 0.5, hq, hkv, d, dtype, rot, rng.random() < 0.4, axes)
    if op == "copy":
        layers = rng.choice([1, 2, 5])
        return _copy(None, max(1, log(1, 2500) // layers), layers, hkv, d, dtype)
    window = rng.choice([0, 0, 128, 1024, 4096])
    sinks = rng.random() < 0.4
    if op == "decode":
        most = log(1, 131072)
        per = 2 * hkv * d * 2  # bytes of a token
        n_seq = log(1, max(1, min(256, 64 * 32768 * 4096 // max(1, most * per * 2))))
        least = rng.choice([most, rng.randrange(0, most + 1), 0])
        return _decode(None, n_seq, least, most, hq, hkv, d, dtype, window, sinks)
    cached = rng.choice([0, 0, log(1, 8192)])
    q_max = log(1, 4096)
    n_seq = log(1, max(1, min(64, 1_500_000_000 // (hq * q_max * (q_max + cached)))))
    return _prefill(None, n_seq, rng.randrange(0, q_max + 1), q_max, rng.randrange(0, cached + 1), cached, hq, hkv, d,
                    dtype, window, sinks, lens_seed=rng.randrange(1000))


def _named(name, case):
    return case if name is None else dict(case, name=name)


def _append(name, tokens, step, q_heads, kv_heads, head_dim, dtype, rot_dim, interleaved, axes):
    return _named(name, dict(op="append", tokens=tokens, step=step, q_heads=q_heads, kv_heads=kv_heads,
                             head_dim=head_dim, dtype=dtype, rot_dim=rot_dim, interleaved=interleaved, axes=axes))


def _copy(name, pages, layers, kv_heads, head_dim, dtype):
    return _named(name, dict(op="copy", pages=pages, layers=layers, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype))


def _decode(name, n_seq, kv_min, kv_max, q_heads, kv_heads, head_dim, dtype, window, sinks, lens_seed=7):
    return _named(name, dict(op="decode", n_seq=n_seq, kv_min=kv_min, kv_max=kv_max, q_heads=q_heads,
                             kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, window=window, sinks=sinks,
                             lens_seed=lens_seed))


def _prefill(name, n_seq, q_min, q_max, cached_min, cached_max, q_heads, kv_heads, head_dim, dtype, window, sinks,
             lens_seed=11):
    return _named(name, dict(op="prefill", n_seq=n_seq, q_min=q_min, q_max=q_max, cached_min=cached_min,
                             cached_max=cached_max, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                             dtype=dtype, window=window, sinks=sinks, lens_seed=lens_seed))


def _lengths(case):
    """(new tokens, key rows) of each sequence; they belong to the case, not to the seed.  The first sequence has
    the most of both."""
    r = random.Random(case["lens_seed"])
    n = case["n_seq"]
    if case["op"] == "decode":
        return [1] * n, [case["kv_max"] if i == 0 else r.randint(case["kv_min"], case["kv_max"]) for i in range(n)]
    q = [case["q_max"] if i == 0 else r.randint(case["q_min"], case["q_max"]) for i in range(n)]
    return q, [a + (case["cached_max"] if i == 0 else r.randint(case["cached_min"], case["cached_max"]))
               for i, a in enumerate(q)]


def _visible(q, kv, window):
    """How many keys the q last positions of a sequence of kv rows see in all."""
    full = q * (2 * kv - q + 1) // 2
    if not window:
        return full
    inside = max(0, min(q, window - (kv - q)))  # positions that see fewer than `window` keys, or just as many
    first = kv - q + 1
    return inside * (2 * first + inside - 1) // 2 + (q - inside) * window


def work(case):
    d, hkv = case["head_dim"], case["kv_heads"]
    if case["op"] == "copy":
        return {"bytes": 2 * case["pages"] * case["layers"] * 2 * hkv * PAGE * d * 2 + 8 * case["pages"], "flops": 0}
    hq = case["q_heads"]
    if case["op"] == "append":
        n = case["tokens"]
        table = min(n * case["axes"], TABLE_ROWS) * case["rot_dim"] * 4 // case["axes"]
        return {"bytes": 2 * n * (hq + 2 * hkv) * d * 2 + n * 4 * (1 + case["axes"]) + table,
                "flops": 3 * n * (hq + hkv) * case["rot_dim"]}
    q, kv = _lengths(case)
    w = case["window"]
    rows = sum(min(b, w + a - 1) if w else b for a, b in zip(q, kv))  # key rows that some position sees
    seen = sum(_visible(a, b, w) for a, b in zip(q, kv) if b)
    return {"bytes": rows * 2 * hkv * d * 2 + 2 * sum(q) * hq * d * 2 + 4 * (rows // PAGE + 2 * len(q)),
            "flops": 4 * seen * hq * d}


# --------------------------------------------------------------- the inputs
def prepare(case, seed):
    g = torch.Generator(DEV)
    g.manual_seed(seed)
    dtype, d, hkv = DTYPES[case["dtype"]], case["head_dim"], case["kv_heads"]

    def normal(*shape, dtype=dtype):
        return torch.randn(shape, generator=g, device=DEV, dtype=dtype)

    state = {"case": case, "status": torch.zeros(1, dtype=torch.int32, device=DEV)}
    if case["op"] == "copy":
        total = 2 * case["pages"] + 3
        state["cache"] = normal(case["layers"], total, 2, hkv, PAGE, d)
        order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
        state["src"], state["dst"] = order[:case["pages"]].contiguous(), order[case["pages"]:2 * case["pages"]].contiguous()
        return state
    hq = case["q_heads"]
    if case["op"] == "append":
        n = case["tokens"]
        pages = n if case["step"] else (n + PAGE - 1) // PAGE
        state["cache"] = normal(1, pages + 2, 2, hkv, PAGE, d)
        perm = torch.randperm(pages + 2, generator=g, device=DEV)
        t = torch.arange(n, device=DEV)
        where = (t, torch.randint(0, PAGE, (n,), generator=g, device=DEV)) if case["step"] else (t // PAGE, t % PAGE)
        state["slots"] = (perm[where[0]] * PAGE + where[1]).to(torch.int32)
        qkv = normal(n, (hq + 2 * hkv) * d)  # one projection's output: q, k and v are views of it
        state["q"] = qkv[:, :hq * d].unflatten(1, (hq, d))
        state["k"] = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
        state["v"] = qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d))
        half = case["rot_dim"] // 2
        if half:
            freq = 10000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
            angle = torch.arange(TABLE_ROWS, device=DEV, dtype=torch.float64)[:, None] * freq
            state["table"] = torch.stack((angle.cos(), angle.sin()), dim=-1).float().contiguous()
            shape = (n,) if case["axes"] == 1 else (case["axes"], n)
            state["pos"] = torch.randint(0, TABLE_ROWS, shape, generator=g, device=DEV).to(torch.int32) \
                if case["step"] or case["axes"] > 1 else t.to(torch.int32) % TABLE_ROWS
            state["sections"] = _sections(case)
        return state
    q_lens, kv_lens = _lengths(case)
    need = [(k + PAGE - 1) // PAGE for k in kv_lens]
    total = sum(need) + 2
    state["cache"] = normal(1, total, 2, hkv, PAGE, d)
    width = max(1, max(need))
    perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(need), width), -1, dtype=torch.int32, device=DEV)
    held = torch.arange(width, device=DEV)[None, :] < torch.tensor(need, device=DEV)[:, None]
    table[held] = perm[:sum(need)]
    state["page_table"] = table
    state["kv_lens"] = torch.tensor(kv_lens, dtype=torch.int32, device=DEV)
    state["max_q"], state["max_kv"] = max(q_lens), max(1, max(kv_lens))
    state["q"] = normal(sum(q_lens), hq, d) * 1.5
    state["sinks"] = normal(hq, dtype=torch.float32) if case["sinks"] else None
    if case["op"] == "prefill":
        state["cu_q"] = torch.tensor([0] + q_lens, device=DEV).cumsum(0).to(torch.int32)
    return state


def _sections(case):
    """Pairs of each position axis: a quarter of them time, the rest height and width; one axis has them all."""
    half = case["rot_dim"] // 2
    if case["axes"] == 1:
        return (half,)
    a = half // 4
    b = (half - a) // 2
    return (a, b, half - a - b)


# ---------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    return {"append": _plain_append, "copy": _plain_copy, "prefill": _plain_prefill, "decode": _plain_decode}[op](state)


def _own(s, op):
    if "pool" not in s:  # the pool object that a program keeps beside its cache tensor
        from rsllm_b200 import GqaKvPool, RotaryTable

        s["pool"] = GqaKvPool.over(s["cache"], status=s["status"])
        s["rotary"] = RotaryTable(s["table"], sections=s["sections"], interleaved=s["case"]["interleaved"]) \
            if "table" in s else None
    pool = s["pool"]
    if op == "append":
        if s["rotary"] is None:
            pool.append(0, s["k"], s["v"], s["slots"])
            return {"cache": s["cache"]}
        q = pool.append(0, s["k"], s["v"], s["slots"], q=s["q"], rotary=s["rotary"], pos=s["pos"])
        return {"q": q, "cache": s["cache"]}
    if op == "copy":
        pool.copy_pages(s["src"], s["dst"])
        return {"cache": s["cache"]}
    if op == "decode":
        return {"out": pool.decode(0, s["q"], s["page_table"], s["kv_lens"], window=s["case"]["window"], sinks=s["sinks"])}
    return {"out": pool.prefill(0, s["q"], s["cu_q"], s["page_table"], s["kv_lens"], window=s["case"]["window"],
                                sinks=s["sinks"])}


def _axis_of_pair(sections):
    return torch.repeat_interleave(torch.arange(len(sections), device=DEV), torch.tensor(sections, device=DEV))


def _rotated(x, cos, sin, interleaved):
    """x [n, heads, d] with its first 2 * pairs lanes rotated; cos and sin [n, pairs]."""
    half = cos.shape[1]
    rot, rest = x[..., :2 * half], x[..., 2 * half:]
    cos, sin = cos[:, None, :], sin[:, None, :]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        out = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = rot[..., :half], rot[..., half:]
        out = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((out, rest), dim=-1)


def _plain_append(s):
    cache, slots = s["cache"], s["slots"].long()
    page, row = slots // PAGE, slots % PAGE
    cache[0, page, 1, :, row] = s["v"]
    if "table" not in s:
        cache[0, page, 0, :, row] = s["k"]
        return {"cache": cache}
    half = s["table"].shape[1]
    pos = s["pos"].long().reshape(-1, s["k"].shape[0])
    cs = s["table"][pos[_axis_of_pair(s["sections"])].T, torch.arange(half, device=DEV)]  # [n, pairs, 2]
    k = _rotated(s["k"].float(), cs[..., 0], cs[..., 1], s["case"]["interleaved"])
    q = _rotated(s["q"].float(), cs[..., 0], cs[..., 1], s["case"]["interleaved"])
    cache[0, page, 0, :, row] = k.to(cache.dtype)
    return {"q": q.to(cache.dtype), "cache": cache}


def _plain_copy(s):
    s["cache"][:, s["dst"].long()] = s["cache"][:, s["src"].long()]
    return {"cache": s["cache"]}


def _rows(s, which):
    """Every sequence's key (0) or value (1) rows in order, f32 [n_seq, kv_heads, rows, d], padded."""
    pages = s["cache"][0, s["page_table"].clamp(min=0).long(), which]
    return pages.transpose(1, 2).flatten(2, 3).float()


def _attend(q, seen, s):
    """q f32 [n, kv_heads, m, d]; seen [n, m, rows] -> [n, kv_heads, m, d]; rows that see nothing give zeros."""
    n, hkv, m, d = q.shape
    group = s["case"]["q_heads"] // hkv
    x = q @ _rows(s, 0).transpose(2, 3)
    x *= 1.0 / math.sqrt(d)
    x.masked_fill_(~seen[:, None], -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(hkv, 1, group).expand(hkv, m // group, group).reshape(1, hkv, m, 1)
        top = torch.maximum(top, sink)
    top = top.clamp(min=-3.0e38)
    x -= top
    x.exp_()
    total = x.sum(dim=-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + (sink - top).exp()
    return (x @ _rows(s, 1)) / torch.where(total > 0, total, 1.0)


def _plain_decode(s):
    n, hq, d = s["q"].shape
    hkv, w = s["case"]["kv_heads"], s["case"]["window"]
    key = torch.arange(s["page_table"].shape[1] * PAGE, device=DEV)[None, None, :]
    kv = s["kv_lens"].view(n, 1, 1)
    seen = key < kv
    if w:
        seen = seen & (key >= kv - w)
    out = _attend(s["q"].float().view(n, hkv, hq // hkv, d), seen.expand(n, hq // hkv, -1), s)
    return {"out": out.reshape(n, hq, d).to(s["q"].dtype)}


def _plain_prefill(s):
    tokens, hq, d = s["q"].shape
    hkv, w = s["case"]["kv_heads"], s["case"]["window"]
    group = hq // hkv
    cu = s["cu_q"].long()
    n = cu.numel() - 1
    lens = cu[1:] - cu[:-1]
    i = torch.arange(s["max_q"], device=DEV)[None, :]
    real = i < lens[:, None]
    at = (cu[:-1, None] + i)[real]  # every packed row, sequence after sequence
    q = torch.zeros((n, s["max_q"], hkv, group, d), device=DEV)
    q[real] = s["q"].float().view(tokens, hkv, group, d)[at]
    q = q.permute(0, 2, 1, 3, 4).reshape(n, hkv, s["max_q"] * group, d)
    pos = (s["kv_lens"].long() - lens)[:, None] + i
    key = torch.arange(s["page_table"].shape[1] * PAGE, device=DEV)[None, None, :]
    seen = (key <= pos[:, :, None]) & (key < s["kv_lens"].view(n, 1, 1))
    if w:
        seen = seen & (key > pos[:, :, None] - w)
    out = _attend(q, seen.repeat_interleave(group, dim=1), s)
    out = out.view(n, hkv, s["max_q"], group, d).permute(0, 2, 1, 3, 4)[real]
    return {"out": out.reshape(tokens, hq, d).to(s["q"].dtype)}


# ------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        cache = s["cache"].double()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            cache[:, b] = cache[:, a]
        return {"cache": cache}
    if case["op"] == "append":
        return _exact_append(case, s)
    q_lens, kv_lens = _lengths(case)
    hq, hkv, d, w = case["q_heads"], case["kv_heads"], case["head_dim"], case["window"]
    group = hq // hkv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    first = 0
    for i, (m, kv) in enumerate(zip(q_lens, kv_lens)):
        pages = s["page_table"][i, :(kv + PAGE - 1) // PAGE].long()
        for h in range(hkv if kv and m else 0):
            keys = s["cache"][0, pages, 0, h].reshape(-1, d)[:kv].double()
            values = s["cache"][0, pages, 1, h].reshape(-1, d)[:kv].double()
            for a in range(0, m, 1024):  # positions a .. b of the sequence's new tokens
                b = min(m, a + 1024)
                t = torch.arange(kv - m + a, kv - m + b, device=DEV)[:, None]
                j = torch.arange(kv, device=DEV)[None, :]
                hidden = (j > t) | (j <= t - w) if w else j > t
                for g in range(h * group, (h + 1) * group):
                    x = s["q"][first + a:first + b, g].double() @ keys.T / math.sqrt(d)
                    x[hidden] = -math.inf
                    top = x.max(dim=1, keepdim=True).values
                    if s["sinks"] is not None:
                        top = top.clamp(min=float(s["sinks"][g]))
                    e = (x - top).exp()
                    total = e.sum(dim=1, keepdim=True)
                    if s["sinks"] is not None:
                        total += (s["sinks"][g].double() - top).exp()
                    out[first + a:first + b, g] = (e / total) @ values
        first += m
    return {"out": out}


def _exact_append(case, s):
    cache = s["cache"].double()
    n, half = case["tokens"], case["rot_dim"] // 2
    slots = s["slots"].long()
    k, q = s["k"].double(), s["q"].double()
    if half:
        pos = s["pos"].long().reshape(-1, n)
        cos = torch.empty((n, half), dtype=torch.float64, device=DEV)
        sin = torch.empty_like(cos)
        axis = [a for a, count in enumerate(s["sections"]) for _ in range(count)]
        for i in range(half):
            cos[:, i] = s["table"][pos[axis[i]], i, 0].double()
            sin[:, i] = s["table"][pos[axis[i]], i, 1].double()
        for x in (k, q):
            for i in range(half):
                a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
                u, v = x[:, :, a].clone(), x[:, :, b].clone()
                x[:, :, a] = u * cos[:, i, None] - v * sin[:, i, None]
                x[:, :, b] = v * cos[:, i, None] + u * sin[:, i, None]
    cache[0, slots // PAGE, 0, :, slots % PAGE] = k
    cache[0, slots // PAGE, 1, :, slots % PAGE] = s["v"].double()
    return {"q": q, "cache": cache} if half else {"cache": cache}
