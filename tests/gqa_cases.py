"""Inputs and a plain 64-bit implementation for the grouped-head cache tests."""
import math

import torch

PAGE = 64
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # largest relative rounding error of the type


class Batch:
    """Sequences of ``kv_lens`` rows in scattered pages of a one-layer cache, each ending with its ``q_lens`` new
    tokens.  Rows past a sequence's length and pages of no sequence hold ``rest``."""

    def __init__(self, q_lens, kv_lens, hq, hkv, d, dtype, seed=0, rest=float("nan"), layers=1, q_scale=1.5,
                 device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.q_lens, self.kv_lens_list = list(q_lens), list(kv_lens)
        self.hq, self.hkv, self.d, self.dtype, self.layers = hq, hkv, d, dtype, layers
        need = [(n + PAGE - 1) // PAGE for n in kv_lens]
        total = sum(need) + 3
        cache = torch.full((layers, total, 2, hkv, PAGE, d), rest, dtype=dtype)
        perm = torch.randperm(total, generator=g).tolist()
        self.k, self.v = [], []  # per sequence [layers, kv, hkv, d]
        table = torch.full((len(need), max(need + [1]) + 1), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(kv_lens):
            rows = torch.randn((2, layers, n, hkv, d), generator=g).to(dtype)
            self.k.append(rows[0])
            self.v.append(rows[1])
            for i in range(need[s]):
                page = perm[at]
                at += 1
                table[s, i] = page
                part = rows[:, :, i * PAGE:(i + 1) * PAGE]
                cache[:, page, :, :, :part.shape[2]] = part.permute(1, 0, 3, 2, 4)
        self.q_cpu = (torch.randn((sum(q_lens), hq, d), generator=g) * q_scale).to(dtype)
        self.sinks_cpu = torch.randn(hq, generator=g)
        cu = [0]
        for n in q_lens:
            cu.append(cu[-1] + n)
        self.cu = cu
        self.cache = cache.to(device)
        self.table = table.to(device)
        self.q = self.q_cpu.to(device)
        self.sinks = self.sinks_cpu.to(device)
        self.kv_lens = torch.tensor(kv_lens, dtype=torch.int32, device=device)
        self.cu_q = torch.tensor(cu, dtype=torch.int32, device=device)

    def want(self, layer=0, window=0, sinks=False, scale=None):
        """(outputs, sum_j |weight_j v_j|) in 64 bits, [tokens, hq, d]."""
        scale = 1.0 / math.sqrt(self.d) if scale is None else scale
        group = self.hq // self.hkv
        out = torch.zeros((self.cu[-1], self.hq, self.d), dtype=torch.float64)
        mag = torch.zeros_like(out)
        for s, (m, n) in enumerate(zip(self.q_lens, self.kv_lens_list)):
            if m == 0 or n == 0:
                continue
            k = self.k[s][layer].double().repeat_interleave(group, dim=1).transpose(0, 1)
            v = self.v[s][layer].double().repeat_interleave(group, dim=1).transpose(0, 1)
            q = self.q_cpu[self.cu[s]:self.cu[s + 1]].double().transpose(0, 1)
            x = q @ k.transpose(1, 2) * scale
            pos = torch.arange(n - m, n)[:, None]
            j = torch.arange(n)[None, :]
            x.masked_fill_((j > pos) | ((j <= pos - window) if window else (j < 0)), -math.inf)
            top = x.amax(-1, keepdim=True)
            if sinks:
                top = torch.maximum(top, self.sinks_cpu.double()[:, None, None])
            top = top.clamp(min=-1e300)
            e = (x - top).exp()
            den = e.sum(-1, keepdim=True)
            if sinks:
                den = den + (self.sinks_cpu.double()[:, None, None] - top).exp()
            w = e / torch.where(den > 0, den, torch.ones_like(den))
            out[self.cu[s]:self.cu[s + 1]] = (w @ v).transpose(0, 1)
            mag[self.cu[s]:self.cu[s + 1]] = (w @ v.abs()).transpose(0, 1)
        return out, mag


def close(got, want, mag, dtype, what=""):
    """Every element within what the roundings allow: each weight is rounded to the type once (u sum w |v|), its
    exponential and the logits are good to 2^-13 each in numerator and denominator (2^-12 sum w |v|), and the
    output is rounded once (u |out|); 1e-6 for f16 results near the subnormals."""
    u = UNIT[dtype]
    got = got.double().cpu()
    assert got.shape == want.shape
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - ((u + 2.0 ** -12) * mag + u * want.abs() + 1e-6)
    assert over.max().item() <= 0 if over.numel() else True, \
        f"{what}: off by {over.max().item():.3g} more than the bound at {over.argmax().item()}"


def rotate(x, table, pos, sections, interleaved):
    """x [n, heads, d] rotated in 64 bits; pos [axes, n]."""
    x = x.double().clone()
    half = table.shape[1]
    axis = [a for a, c in enumerate(sections) for _ in range(c)]
    for i in range(half):
        cs = table[pos[axis[i]].long(), i].double()
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        u, w = x[:, :, a].clone(), x[:, :, b].clone()
        x[:, :, a] = u * cs[:, :1] - w * cs[:, 1:]
        x[:, :, b] = w * cs[:, :1] + u * cs[:, 1:]
    return x
