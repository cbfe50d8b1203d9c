"""A quantised attention layer over a 4-bit key / value cache that is kept to a budget of tokens.

    python examples/quantized_attention.py [--prompt 4096] [--steps 64] [--budget 1024] [--hidden 4096] [--heads 32]

Every tensor operation of the layer is one of the library's: add_rms_norm_quant, quant_linear (one projection to queries, keys
and values, and the output projection, added to the residual stream), kv_append, kv_attention, kv_weights and kv_evict.  The
prompt goes through in chunks; its last queries give the first weights, the cache is cut to the budget, and decode steps follow,
which cut it again whenever it has grown by a page.  The command compares the layer's output with the same attention in fp32
(without eviction, over the unquantised keys and values) and prints errors and times.  Weights and inputs are random.
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "asc-devkit_clone_amd"))
import ascq  # noqa: E402


def quantize_weight(w: torch.Tensor):
    """[out, in] -> int8 codes and one fp32 scale per output channel"""
    scale = w.abs().amax(dim=-1) / 127
    return (w / scale[:, None]).round().to(torch.int8).contiguous(), scale.contiguous()


class QuantizedAttention:
    """weights: dict of fp32 tensors -- gamma [H], qkv [(heads + 2 kv_heads) d, H], out [H, heads d]"""

    def __init__(self, weights: dict, batch: int, heads: int, kv_heads: int, room: int, page: int = 64, group: int = 64):
        self.heads, self.kv_heads, self.page, self.batch = heads, kv_heads, page, batch
        self.d = weights["out"].shape[1] // heads
        self.gamma = weights["gamma"].to(torch.bfloat16)
        self.qkv, self.out = quantize_weight(weights["qkv"]), quantize_weight(weights["out"])
        device = self.gamma.device
        columns = -(-room // page)
        self.cache = ascq.kv_cache(batch * columns, kv_heads, page, self.d, group, device)
        self.table = torch.randperm(batch * columns, device=device).int().view(batch, columns).contiguous()
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.weights = torch.zeros(batch, kv_heads, columns * page, device=device)

    def forward(self, x: torch.Tensor, residual: torch.Tensor, queries: int, watch: bool):
        """x, residual [batch * queries, H] bf16, the sequences' next `queries` tokens one after the other -> the new residual
        stream; watch: add these queries' attention to the cached tokens' weights"""
        b, n = self.batch, queries
        q8, scale, h = ascq.add_rms_norm_quant(x, self.gamma, residual=residual)
        qkv = ascq.quant_linear(q8, scale, *self.qkv).view(b * n, -1, self.d)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        at = self.lengths[:, None].long() + torch.arange(n, device=x.device)
        slots = self.table.long().gather(1, at // self.page) * self.page + at % self.page
        ascq.kv_append(self.cache, k, v, slots.reshape(-1))
        self.lengths += n
        where = dict(starts=torch.arange(0, b * n + 1, n, dtype=torch.int32, device=x.device), max_queries=n)
        y, lse = ascq.kv_attention(q, self.cache, self.table, self.lengths, need_lse=watch, **where)
        if watch:
            ascq.kv_weights(q, lse, self.cache, self.table, self.lengths, self.weights, out=self.weights, **where)
        y8, y_scale = ascq.quant_dynamic_per_token(y.view(b * n, -1))
        ascq.quant_linear(y8, y_scale, *self.out, residual=h, out=h)
        return h

    def cut(self, budget: int, recent: int) -> torch.Tensor:
        """keeps the `budget` heaviest tokens of every sequence and head, the last `recent` among them"""
        kept, self.lengths, _ = ascq.kv_evict(self.cache, self.table, self.lengths, self.weights, budget, recent)
        return kept


def reference(weights: dict, heads: int, kv_heads: int, x: torch.Tensor, residual: torch.Tensor, batch: int):
    """the layer in fp32 over whole sequences: x, residual [batch * tokens, H], sequence by sequence"""
    h = (x.float() + residual.float()).to(x.dtype).float()
    n = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + 1e-6) * weights["gamma"].to(torch.bfloat16).float()
    d = weights["out"].shape[1] // heads
    qkv = (n @ weights["qkv"].t()).view(batch, -1, heads + 2 * kv_heads, d)
    out = torch.empty(batch, qkv.shape[1], heads, d, device=x.device)
    mask = torch.ones(qkv.shape[1], qkv.shape[1], dtype=torch.bool, device=x.device).tril()
    for b in range(batch):
        for g in range(heads):
            kv = heads + g // (heads // kv_heads)
            s = (qkv[b, :, g] @ qkv[b, :, kv].t().contiguous()) / math.sqrt(d)
            out[b, :, g] = torch.softmax(torch.where(mask, s, -math.inf), dim=1) @ qkv[b, :, kv + kv_heads]
    return h + out.view(x.shape[0], -1) @ weights["out"].t()


def random_weights(hidden: int, heads: int, kv_heads: int, d: int, device="cuda"):
    g = torch.Generator(device=device).manual_seed(0)
    w = lambda *s: torch.randn(s, generator=g, device=device) / s[-1] ** 0.5  # noqa: E731
    return dict(gamma=1 + 0.1 * torch.randn(hidden, generator=g, device=device), qkv=w((heads + 2 * kv_heads) * d, hidden),
                out=w(hidden, heads * d))


def run(batch: int, prompt: int, steps: int, budget: int, hidden: int, heads: int, kv_heads: int, d: int, chunk: int = 512):
    """errors of the prompt's and the decode steps' outputs relative to what the layer adds, and the layer"""
    weights = random_weights(hidden, heads, kv_heads, d)
    page = 64
    layer = QuantizedAttention(weights, batch, heads, kv_heads, max(prompt, budget) + 2 * page)
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens = prompt + steps
    x, residual = (torch.randn(batch, tokens, hidden, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    want = reference(weights, heads, kv_heads, x.flatten(0, 1), residual.flatten(0, 1), batch).view(batch, tokens, hidden)
    added = want - (x.float() + residual.float())
    part = lambda t, a, b: t[:, a:b].reshape(-1, hidden)  # noqa: E731
    errors = []
    for a in range(0, prompt, chunk):
        b = min(prompt, a + chunk)
        out = layer.forward(part(x, a, b), part(residual, a, b), b - a, watch=b == prompt)
        errors.append(((out.float() - part(want, a, b)).norm() / part(added, a, b).norm()).item())
    full = max(errors)
    errors = []
    length = prompt
    for i in range(prompt, tokens):
        if length > budget + page or (i == prompt and length > budget):
            layer.cut(budget, budget // 4)
            length = budget
        out = layer.forward(part(x, i, i + 1), part(residual, i, i + 1), 1, watch=True)
        length += 1
        errors.append(((out.float() - part(want, i, i + 1)).norm() / part(added, i, i + 1).norm()).item())
    return full, errors, layer


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, default in (("batch", 4), ("prompt", 4096), ("steps", 64), ("budget", 1024), ("hidden", 4096), ("heads", 32),
                          ("kv-heads", 8), ("d", 128)):
        ap.add_argument(f"--{name}", type=int, default=default)
    a = ap.parse_args()
    full, errors, layer = run(a.batch, a.prompt, a.steps, a.budget, a.hidden, a.heads, a.kv_heads, a.d)
    x = torch.randn(a.batch, a.hidden, device="cuda").to(torch.bfloat16)
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    before = layer.lengths.clone()
    start.record()
    for _ in range(20):
        layer.forward(x, x, 1, watch=True)
        layer.lengths.copy_(before)
    stop.record()
    torch.cuda.synchronize()
    print(f"error of what the layer adds: {full:.4f} over the whole cache, {sum(errors) / max(1, len(errors)):.4f} over the "
          f"budget of {a.budget}; {start.elapsed_time(stop) / 20 * 1e3:.0f} us a decode step")
    return 0


if __name__ == "__main__":
    sys.exit(main())
