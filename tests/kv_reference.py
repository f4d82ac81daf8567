"""Plain 64-bit restatement of the paged 8-bit cache and the attention over it
(include/q4k.h), on CPU tensors; used by the GPU tests."""
from __future__ import annotations

import math

import torch

BLOCK = 16


def scale_of(amax: torch.Tensor) -> torch.Tensor:
    """2^E, E the smallest with amax <= 448 * 2^E, in [-60, 60] (f64)."""
    out = torch.full_like(amax, 2.0**-60)
    for e in range(-60, 60):
        out = torch.where(amax > 448.0 * 2.0**e, torch.full_like(amax, 2.0 ** (e + 1)), out)
    return out


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [..., D] f64, cos/sin [..., R/2]: pairs (j, j + R/2)."""
    h = cos.shape[-1]
    a, b = x[..., :h], x[..., h : 2 * h]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h :]], -1)


def rope_table(positions: int, rot: int, theta: float = 10000.0) -> torch.Tensor:
    f = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * f[None]
    return torch.stack([ang.cos(), ang.sin()], -1).float()


def dequant(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """[pages, heads, page, D] codes and their scales -> f64 values."""
    return codes.view(torch.uint8).view(torch.float8_e4m3fn).to(torch.float64) * scale.double().repeat_interleave(
        BLOCK, -1)[..., None]


def gather(values: torch.Tensor, table_row: torch.Tensor, n: int) -> torch.Tensor:
    """The first n positions of a sequence: [heads, n, D]."""
    page = values.shape[2]
    pages = table_row[: max(1, -(-n // page))].long()
    return values[pages].transpose(0, 1).reshape(values.shape[1], -1, values.shape[3])[:, :n]


def attention(q, k_val, v_val, table, q_start, kv_len, scale, window=0) -> torch.Tensor:
    """q [tokens, Hq, D] f64; k_val, v_val dequantised caches f64; lists of ints."""
    tokens, hq, d = q.shape
    hkv = k_val.shape[1]
    out = torch.zeros(tokens, hq, d, dtype=torch.float64)
    for b in range(len(kv_len)):
        n, kv = q_start[b + 1] - q_start[b], kv_len[b]
        if n == 0 or kv == 0:
            continue
        k, v = gather(k_val, table[b], kv), gather(v_val, table[b], kv)
        pos = torch.arange(kv - n, kv)
        j = torch.arange(kv)
        seen = j[None] <= pos[:, None]
        if window:
            seen &= j[None] > pos[:, None] - window
        for h in range(hq):
            kh = h // (hq // hkv)
            s = (q[q_start[b] : q_start[b + 1], h] @ k[kh].T) * scale
            s = s.masked_fill(~seen, -math.inf)
            p = torch.exp(s - s.amax(1, keepdim=True).clamp(min=-1e300))
            tot = p.sum(1, keepdim=True)
            o = (p @ v[kh]) / tot
            out[q_start[b] : q_start[b + 1], h] = torch.where(tot > 0, o, torch.zeros_like(o))
    return out


class Problem:
    """A batch of sequences over a filled cache, on the CPU."""

    def __init__(self, new, kv, hq, hkv, d, page, seed=0, extra_pages=3, spread=4.0, v_mix=False):
        g = torch.Generator().manual_seed(seed)
        self.new, self.kv, self.page, self.hq, self.hkv, self.d = list(new), list(kv), page, hq, hkv, d
        per = [max(1, -(-x // page)) for x in kv]
        cols, pages = max(per), sum(per) + extra_pages
        order = torch.randperm(pages, generator=g)
        self.table = torch.zeros(len(kv), cols, dtype=torch.int32)
        at = 0
        for b, p in enumerate(per):
            self.table[b, :p] = order[at : at + p]
            at += p
        self.q_start = [0]
        for n in new:
            self.q_start.append(self.q_start[-1] + n)
        self.tokens = self.q_start[-1]
        self.pages = pages
        self.q = torch.randn(self.tokens, hq, d, generator=g, dtype=torch.float64)

        def fill(amp):
            x = torch.randn(pages, hkv, page, d, generator=g, dtype=torch.float64) * amp
            if v_mix:  # blocks of very different magnitude
                mix = torch.randint(-12, 6, (pages, hkv, page // BLOCK, 1), generator=g)
                x = (x.view(pages, hkv, page // BLOCK, -1) * 2.0**mix).view_as(x)
            s = scale_of(x.abs().view(pages, hkv, page // BLOCK, BLOCK * d).amax(-1))
            c = (x / s.repeat_interleave(BLOCK, -1)[..., None]).float().to(torch.float8_e4m3fn)
            return c, s.float()

        amp = torch.ones(d, dtype=torch.float64)
        amp[:: max(1, d // 4)] = spread
        self.k, self.k_scale = fill(amp)
        self.v, self.v_scale = fill(torch.ones(d, dtype=torch.float64))

    def device(self, dev, q4k, dtype):
        cache = q4k.KVCache(self.k.to(dev), self.v.to(dev), self.k_scale.to(dev), self.v_scale.to(dev))
        i32 = dict(dtype=torch.int32, device=dev)
        return cache, self.q.to(dtype).to(dev), self.table.to(dev), torch.tensor(self.q_start, **i32), torch.tensor(
            self.kv, **i32)

    def expected(self, dtype, scale, window=0):
        return attention(self.q.to(dtype).double(), dequant(self.k, self.k_scale), dequant(self.v, self.v_scale),
                         self.table, self.q_start, self.kv, scale, window)
