"""Serving a grouped-head model over the paged cache: prompts that share a prefix,
prefilled together, then decoded token by token.

    python examples/gqa_serve.py

A small random-weight transformer (two layers, 8 q heads on 2 kv heads of 64
lanes) runs on the calls an engine would make: ``PrefixKvPool`` plans the pages
(radix prefix store, copy-on-write, slots), ``GqaKvPool`` holds the rows --
rotary append, prefill over what is cached and what is new, decode -- and
``apply_moves`` copies the pages the plan moves.  The tokens are compared with a
plain recomputation of every sequence from its first token.
"""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from rsllm_b200 import GqaKvPool, RotaryTable  # noqa: E402
from rsllm_b200.prefix_pool import PrefixKvPool  # noqa: E402

VOCAB, WIDTH, LAYERS, Q_HEADS, KV_HEADS, HEAD_DIM = 97, 256, 2, 8, 2, 64
DTYPE = torch.bfloat16


class Model:
    """Embedding, attention blocks without an MLP, tied output."""

    def __init__(self, device, seed: int = 0):
        g = torch.Generator(device).manual_seed(seed)

        def weight(*shape):
            return torch.randn(shape, generator=g, device=device) / shape[-1] ** 0.5

        self.embed = torch.randn((VOCAB, WIDTH), generator=g, device=device)
        self.qkv = [weight((Q_HEADS + 2 * KV_HEADS) * HEAD_DIM, WIDTH) for _ in range(LAYERS)]
        self.out = [8 * weight(WIDTH, Q_HEADS * HEAD_DIM) for _ in range(LAYERS)]  # attention decides the next token

    @staticmethod
    def norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)

    def project(self, layer, x):
        """q, k, v as views of one projection, in the cache's type."""
        fused = (self.norm(x) @ self.qkv[layer].T).to(DTYPE).unflatten(1, (Q_HEADS + 2 * KV_HEADS, HEAD_DIM))
        return fused[:, :Q_HEADS], fused[:, Q_HEADS:Q_HEADS + KV_HEADS], fused[:, Q_HEADS + KV_HEADS:]

    def add(self, layer, x, attention):
        return x + attention.float().flatten(1) @ self.out[layer].T

    def logits(self, x):
        return self.norm(x) @ self.embed.T


class Server:
    def __init__(self, device, pages: int = 64):
        self.device = device
        self.model = Model(device)
        self.plan = PrefixKvPool(pages, LAYERS, device=None)  # decides pages; holds no device memory
        self.cache = GqaKvPool(pages, KV_HEADS, HEAD_DIM, n_layers=LAYERS, dtype=DTYPE, device=device)
        self.rotary = RotaryTable.build(4096, HEAD_DIM, device=device)

    def _i32(self, a):
        return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(self.device)

    def _step(self, seqs, new_tokens):
        """Runs new_tokens[i] (a list) of every sequence and returns the logits of each one's last token."""
        counts = [len(t) for t in new_tokens]
        before = [self.plan.seq_len(s) for s in seqs]
        slots = self._i32(self.plan.reserve(seqs, counts))
        self.cache.apply_moves(*self.plan.take_moves())  # a shared, partly filled page was copied
        tables = [self.plan.page_table(s) for s in seqs]
        table = np.full((len(seqs), max(map(len, tables))), -1, np.int32)
        for row, t in zip(table, tables):
            row[:len(t)] = t
        table = self._i32(table)
        lens = self._i32([b + c for b, c in zip(before, counts)])
        cu = self._i32(np.concatenate(([0], np.cumsum(counts))))
        pos = self._i32(np.concatenate([np.arange(b, b + c) for b, c in zip(before, counts)]))
        x = self.model.embed[torch.tensor([t for new in new_tokens for t in new], device=self.device)]
        for layer in range(LAYERS):
            q, k, v = self.model.project(layer, x)
            q = self.cache.append(layer, k, v, slots, q=q, rotary=self.rotary, pos=pos)
            if max(counts) == 1:
                attention = self.cache.decode(layer, q, table, lens)
            else:
                attention = self.cache.prefill(layer, q, cu, table, lens)
            x = self.model.add(layer, x, attention)
        return self.model.logits(x[cu[1:].long() - 1])

    def generate(self, prompts, n_new: int):
        """Greedy continuations of the prompts.  Returns (tokens, reused prefix lengths, the logits of every step)."""
        seqs, reused, todo = [], [], []
        for p in prompts:
            n, seq = self.plan.match_prefix(p[:-1])  # at least one token is left to run
            seqs.append(seq)
            reused.append(n)
            todo.append(p[n:])
        tokens, steps = [[] for _ in prompts], []
        for _ in range(n_new):
            logits = self._step(seqs, todo)
            steps.append(logits)
            todo = [[int(t)] for t in logits.argmax(-1).tolist()]
            for got, t in zip(tokens, todo):
                got += t
        self.cache.check("generate")
        for p, seq in zip(prompts, seqs):  # later prompts find these
            self.plan.insert_prefix(p, seq)
            self.plan.release(seq)
        return tokens, reused, steps


def plain_logits(model: Model, rotary: RotaryTable, tokens) -> torch.Tensor:
    """The last token's logits from the whole sequence, attention in f32 torch operations."""
    device = model.embed.device
    n = len(tokens)
    x = model.embed[torch.tensor(tokens, device=device)]
    cos, sin = rotary.table[:n, None, :, 0], rotary.table[:n, None, :, 1]

    def turn(a):
        u, w = a.float().chunk(2, dim=-1)
        return torch.cat((u * cos - w * sin, w * cos + u * sin), dim=-1).to(DTYPE).float()

    hidden = torch.ones((n, n), dtype=torch.bool, device=device).triu(1)
    for layer in range(LAYERS):
        q, k, v = model.project(layer, x)
        q, k, v = turn(q), turn(k), v.float()
        k, v = (a.repeat_interleave(Q_HEADS // KV_HEADS, dim=1) for a in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) / HEAD_DIM ** 0.5
        p = s.masked_fill(hidden, float("-inf")).softmax(-1)
        x = model.add(layer, x, torch.einsum("hij,jhd->ihd", p, v).to(DTYPE))
    return model.logits(x[-1:])


def main() -> float:
    device = torch.device("cuda", 0)
    rng = np.random.default_rng(1)
    shared = rng.integers(0, VOCAB, 150).tolist()  # two whole pages and part of a third
    prompts = [shared + rng.integers(0, VOCAB, n).tolist() for n in (1, 40, 7)] + [rng.integers(0, VOCAB, 90).tolist()]
    server = Server(device)
    server.generate([shared + [3]], 2)  # puts the prefix into the store
    tokens, reused, steps = server.generate(prompts, 12)
    worst = 0.0
    for i, p in enumerate(prompts):
        for j, logits in enumerate(steps):
            want = plain_logits(server.model, server.rotary, p + tokens[i][:j])[0]
            worst = max(worst, float((logits[i] - want).abs().max() / want.abs().max()))
        print(f"prompt {i}: {len(p)} tokens, {reused[i]} from the prefix store -> {tokens[i]}")
    print(f"logits against a plain recomputation: within {worst:.2g} of the largest")
    return worst


if __name__ == "__main__":
    main()
