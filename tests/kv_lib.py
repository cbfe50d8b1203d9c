"""The paged int4 key / value cache in plain terms: quantising rows, reading values back, attention and the rest in 64 bits on the CPU."""
from __future__ import annotations

import math

import torch

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}  # a rounding's relative error


def quantize(x: torch.Tensor, group: int):
    """rows [..., d] -> (codes int8 [..., d], scale, offset f16 [..., d / group]), the definition's fp32 operations one by one"""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=math.inf, neginf=-math.inf).clamp(-61440.0, 61440.0)
    x = x.unflatten(-1, (-1, group))
    lo, hi = x.amin(dim=-1), x.amax(dim=-1)
    s = ((hi - lo) / torch.full_like(lo, 15.0)).half()
    o = (lo + 8.0 * s.float()).half()
    inv = torch.where(s > 0, torch.ones_like(lo) / s.float(), 0.0)
    c = ((x - o.float()[..., None]) * inv[..., None]).round().clamp(-8, 7)
    return c.flatten(-2).to(torch.int8), s, o


def pack(c: torch.Tensor) -> torch.Tensor:
    c = c.int() & 15
    return (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """uint8 [..., d / 2] and f16 [..., d / group, 2] -> the values they stand for, f16 in 64 bits"""
    u = codes.int()
    c = torch.stack([u & 15, u >> 4], dim=-1).flatten(-2)
    c = torch.where(c > 7, c - 16, c).double()
    group = c.shape[-1] // scales.shape[-2]
    s = scales.double().repeat_interleave(group, dim=-2)
    return (c * s[..., 0] + s[..., 1]).half().double()


class Problem:
    """a filled cache, page tables in random order, queries; everything on the CPU"""

    def __init__(self, seed, lengths, queries=None, heads=8, kv=2, d=128, group=32, page=16, dt="f16", spare=3, q_size=1.0,
                 kv_size=1.0, columns=None):
        g = self.g = torch.Generator().manual_seed(seed)
        self.lengths, self.heads, self.kv, self.d, self.group, self.page, self.dt = lengths, heads, kv, d, group, page, dt
        self.queries = queries if queries is not None else [1] * len(lengths)
        self.ragged = queries is not None
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + spare
        self.columns = columns or max(need + [1])
        order = torch.randperm(pages, generator=g).int()
        self.table = torch.full((len(lengths), self.columns), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.spare = order[at:]
        x = torch.randn(2, pages, kv, page, d, generator=g) * kv_size
        x[0] += 2 * kv_size * torch.randn(kv, 1, d, generator=g) * (torch.rand(kv, 1, d, generator=g) < 0.1)
        c, s, o = quantize(x, group)
        packed, pairs = pack(c), torch.stack([s, o], dim=-1)
        self.cache = [packed[0].contiguous(), packed[1].contiguous(), pairs[0].contiguous(), pairs[1].contiguous()]
        rows = sum(self.queries)
        self.q = (torch.randn(rows, heads, d, generator=g) * q_size).to(DT[dt])
        self.starts = torch.tensor([0] + list(torch.tensor(self.queries).cumsum(0))).int() if lengths else torch.zeros(1).int()

    def gpu(self, ascq):
        return ascq.KvCache(*(t.cuda() for t in self.cache))

    def args(self, ascq, cache=None):
        """positional and keyword arguments of kv_attention"""
        kw = dict(starts=self.starts.cuda(), max_queries=max(self.queries + [0])) if self.ragged else {}
        return ((self.q.cuda(), cache or self.gpu(ascq), self.table.cuda(), torch.tensor(self.lengths).int().cuda()), kw)

    def rows_of(self, b, which):
        """values [tokens of the table's pages, kv, d] of sequence b and whether a token's page exists"""
        col = self.table[b].long()
        ok = (col >= 0) & (col < self.cache[which].shape[0])
        p = torch.where(ok, col, 0)
        v = values(self.cache[which][p], self.cache[which + 2][p])  # [pages, kv, page, d]
        return v.transpose(1, 2).flatten(0, 1), ok.repeat_interleave(self.page)


def attention(p: Problem, scale=None, causal=True, window=0):
    """(out, lse, bound of out without the output's rounding, bound of lse, weights) in 64 bits.  Bounds: with S = scale sum |q k| of a
    score, its fp32 sum of d products is off by (d + 8) 2^-24 S, its conversion to base 2 and the exponential by 2^-21 (|score| + 1):
    e per score.  A weight is off by 2 e relatively (its own score and the sum) and by its rounding to f16, 2^-11, or 2^-33 of the
    largest weight where f16 has no smaller step; the sums of n terms add n 2^-24."""
    scale = p.d ** -0.5 if scale is None else scale
    rows = p.q.shape[0]
    out = torch.zeros(rows, p.heads, p.d, dtype=torch.float64)
    lse = torch.full((rows, p.heads), -math.inf, dtype=torch.float64)
    tol, tol_lse = torch.zeros_like(out), torch.zeros(rows, p.heads, dtype=torch.float64)
    weights, tol_w = [], []
    ratio = p.heads // p.kv
    for b, length in enumerate(p.lengths):
        k, ok = p.rows_of(b, 0)
        v, _ = p.rows_of(b, 1)
        cap = k.shape[0]
        length = max(0, min(length, cap))
        n = p.queries[b]
        got, err = torch.zeros(p.kv, cap, dtype=torch.float64), torch.zeros(p.kv, cap, dtype=torch.float64)
        t = torch.arange(cap)
        k, v = torch.where(((t < length) & ok)[:, None, None], k, 0.0), torch.where(((t < length) & ok)[:, None, None], v, 0.0)
        for i in range(n):
            r = int(p.starts[b]) + i if p.ragged else b
            at = length - n + i
            seen = (t < length) & ok
            if causal:
                seen &= t <= at
            if window:
                seen &= t > at - window
            if not seen.any():
                continue
            for h in range(p.heads):
                q = p.q[r, h].double()
                kk, vv = k[:, h // ratio], v[:, h // ratio]
                x = (kk @ q) * scale
                e = (abs(scale) * (p.d + 8) * 2.0 ** -24 * (kk.abs() @ q.abs()))[seen].max() + 2.0 ** -21 * (x[seen].abs().max() + 1)
                e = e + t.numel() * 2.0 ** -24
                x = torch.where(seen, x, -math.inf)
                lse[r, h] = torch.logsumexp(x, 0)
                w = torch.exp(x - lse[r, h])
                out[r, h] = w @ vv
                small = 2.0 ** -33 * w.max()
                tol[r, h] = (w * (2.0 ** -11 + 2 * e) + small * seen) @ vv.abs()
                tol_lse[r, h] = e + 2.0 ** -22 * lse[r, h].abs()
                got[h // ratio] += w
                err[h // ratio] += w * (2 * e + 2.0 ** -20 * (1 + lse[r, h].abs()))
        weights.append(got)
        tol_w.append(err)
    return out, lse, tol, tol_lse, weights, tol_w


def evict(weights: torch.Tensor, length: int, keep: int, recent: int):
    """positions that stay of one row of weights"""
    if length <= keep:
        return list(range(length))
    old = length - recent
    key = [(-math.inf if math.isnan(w) else w) for w in weights[:old].tolist()]
    return sorted(sorted(range(old), key=lambda i: (-key[i], i))[:keep - recent]) + list(range(old, length))
