"""Attention over a paged key / value cache held in 4 bits, measured through the public Python binding.

A case is a dict of plain values with an "op":
  append     rows of keys and values into the cache: int4 codes with a scale and an offset per group of channels
  attention  softmax(scale q k + mask) v over the cached tokens of every sequence, and its log-sum-exp
  weights    the attention each cached token received from some queries, added to what it had
  evict      the heaviest and the last tokens of each sequence and head, moved together into other pages
Sizes are generic: 32 heads over 8 key heads of 128, one to 131072 cached tokens, one to 64 sequences; group sizes 32, 64 and
128 as in the repository's weight-only products; rows of 4096.

The cache holds value(code) = f16(code * scale + offset), codes -8 .. 7 two to a byte (even channel in the low nibble), in
pages [page, key head, token of the page, channel].  A sequence's token t lies in page table[t // page_size].

Where `own` is false, `run` computes the operators from elementary torch operations in 32 bits; where it is true, it makes the
library's calls.  Codes, scales and offsets follow from fp32 operations in a fixed order and are the same in both.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
FLOAT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
LIMIT = 61440.0  # keys and values beyond are taken as this: codes * scale + offset stays a finite f16
HEAVY = 8 * 131072 * 8 * 128  # cached elements (of keys) of the largest listed attention

_ascq = None


def _lib():
    global _ascq
    if _ascq is None:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "asc-devkit_clone_amd"))
        import ascq

        _ascq = ascq
    return _ascq


def listed():
    base = dict(heads=32, kv=8, d=128, group=32, page=64, dtype="bf16")
    return [
        # one decode step of 16 sequences: the smallest call, latency
        dict(base, name="append_decode", op="append", tokens=16, fused=True),
        # the keys and values of a large prompt, sliced from the fused projection's rows: HBM
        dict(base, name="append_8192", op="append", tokens=8192, group=128, dtype="f16", fused=True),
        # one decode step of a single conversation: latency, few rows, the cached tokens split over the card
        dict(base, name="attention_one", op="attention", batch=1, queries=1, length=4096, ragged=False, window=0),
        # one decode step of a serving batch, conversations of all lengths, small pages
        dict(base, name="attention_batch", op="attention", batch=32, queries=1, length=8192, ragged=True, window=0, page=16,
             dtype="f16"),
        # decode steps over very long documents, coarse groups: the cache's bytes from HBM; the largest
        dict(base, name="attention_long", op="attention", batch=8, queries=1, length=131072, ragged=False, window=0, group=128,
             page=128),
        # five drafted tokens of each sequence verified at once
        dict(base, name="attention_drafts", op="attention", batch=16, queries=5, length=4099, ragged=True, window=0, group=64),
        # a chunk of a prompt's queries over what is cached of it: matrix products
        dict(base, name="attention_chunk", op="attention", batch=2, queries=1024, length=8192, ragged=False, window=0),
        # small heads of their own keys, a sliding window, lengths that divide nothing
        dict(base, name="attention_window", op="attention", batch=13, queries=1, length=5003, ragged=True, window=1021, heads=12,
             kv=12, d=64, group=64, page=32),
        # the statistics of one decode step of a serving batch
        dict(base, name="weights_decode", op="weights", batch=16, queries=1, length=8192, ragged=True, window=0, before=True),
        # those of a prompt's last 64 queries
        dict(base, name="weights_prompt", op="weights", batch=2, queries=64, length=16384, ragged=False, window=0, before=False),
        # half of what every sequence of a batch holds goes
        dict(base, name="evict_batch", op="evict", batch=16, length=4096, ragged=True, keep=2048, recent=256),
        # a very long prompt cut to an eighth before decoding
        dict(base, name="evict_long", op="evict", batch=2, length=131072, ragged=False, keep=16384, recent=1024, page=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["append", "attention", "attention", "attention", "attention", "weights", "weights", "evict"])
        kv, ratio = rng.choice([(8, 4), (8, 4), (8, 8), (4, 7), (1, 8), (2, 6), (12, 1), (5, 3), (16, 2), (1, 32)])
        d = rng.choice([64, 128, 128, 256])
        c = dict(op=op, heads=kv * ratio, kv=kv, d=d, group=rng.choice([g for g in (32, 64, 128) if g <= d]),
                 page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["f16", "bf16"]))
        if op == "append":
            c.update(tokens=_log(rng, 1, 16384), fused=rng.random() < 0.5, dtype=rng.choice(["f16", "bf16", "f32"]))
            if c["tokens"] * kv * d <= 8192 * 8 * 128:
                return c
            continue
        c.update(batch=_log(rng, 1, 64), length=_log(rng, 1, 131072), ragged=rng.random() < 0.6)
        if op == "evict":
            c["keep"] = max(1, int(c["length"] * rng.uniform(0.1, 0.8)))
            c["recent"] = int(c["keep"] * rng.uniform(0.0, 0.5))
        else:
            c["queries"] = min(c["length"], rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 1024)]))
            c["window"] = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
            if op == "weights":
                c["before"] = rng.random() < 0.5
        cached = c["batch"] * c["length"] * kv * d
        pairs = cached * ratio * c.get("queries", 1)  # products of a query and a key, element by element
        if cached <= (HEAVY // 2 if op == "attention" else HEAVY // 8) and pairs <= 2 * 1024 * 8192 * 32 * 128 // 2:
            return c


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _lengths(c):
    """cached tokens per sequence, queries included (the last is the longest)"""
    rng = random.Random(c["length"] * 64 + c["batch"])
    least = max(1, c.get("queries", 1))
    out = [rng.randint(least, c["length"]) if c["ragged"] else c["length"] for _ in range(c["batch"] - 1)]
    return out + [c["length"]]


def _span(c):
    return -(-c["length"] // c["page"])  # columns of the page table


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, shape):
    return torch.randn(shape, generator=g, device=DEV)


def _quantize(x, group):
    """codes (two to a byte), and scale and offset per group, of rows x [..., channels]"""
    x = x.float()
    x = torch.where(torch.isnan(x), 0.0, x).clamp(-LIMIT, LIMIT)
    x = x.reshape(*x.shape[:-1], -1, group)
    lo, hi = x.amin(dim=-1, keepdim=True), x.amax(dim=-1, keepdim=True)
    # (divided by a tensor: torch multiplies by the reciprocal of a number)
    s = ((hi - lo) / torch.full_like(lo, 15.0)).half()
    o = (lo + 8 * s.float()).half()
    inv = torch.where(s > 0, 1 / s.float(), 0.0)
    code = ((x - o.float()) * inv).round_().clamp_(-8, 7).to(torch.int8).reshape(*x.shape[:-2], -1, 2)
    packed = ((code[..., 0] & 15) | (code[..., 1] << 4)).view(torch.uint8)
    return packed, torch.cat([s, o], dim=-1)


def _filled_cache(g, c, pages):
    """a cache of `pages` pages: keys with a few strong channels, as projections have, and normal values; every page is
    made from its own numbers, some pages at a time"""
    kv, d, ps, gr = c["kv"], c["d"], c["page"], c["group"]
    cache = [torch.empty((pages, kv, ps, d // 2), dtype=torch.uint8, device=DEV) for _ in range(2)]
    cache += [torch.empty((pages, kv, ps, d // gr, 2), dtype=torch.float16, device=DEV) for _ in range(2)]
    bias = 2.0 * _normal(g, (kv, 1, d)) * (torch.rand((kv, 1, d), generator=g, device=DEV) < 0.1)
    step = max(1, (1 << 28) // (kv * ps * d))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        cache[0][at:at + n], cache[2][at:at + n] = _quantize(_normal(g, (n, kv, ps, d)) + bias, gr)
        cache[1][at:at + n], cache[3][at:at + n] = _quantize(_normal(g, (n, kv, ps, d)), gr)
    return dict(zip(("k", "v", "k_scale", "v_scale"), cache))


def _inputs(c, seed):
    g, op = _gen(seed), c["op"]
    kv, d, ps = c["kv"], c["d"], c["page"]
    if op == "append":
        t, dt = c["tokens"], FLOAT[c["dtype"]]
        pages = -(-2 * t // ps)
        cache = dict(k=torch.zeros((pages, kv, ps, d // 2), dtype=torch.uint8, device=DEV))
        cache["v"] = torch.zeros_like(cache["k"])
        cache["k_scale"] = torch.zeros((pages, kv, ps, d // c["group"], 2), dtype=torch.float16, device=DEV)
        cache["v_scale"] = torch.zeros_like(cache["k_scale"])
        width = (c["heads"] + 2 * kv) if c["fused"] else 2 * kv
        rows = _normal(g, (t, width, d)).to(dt)  # queries, keys, values of a token side by side
        rows[:, -2 * kv:-kv, ::17] *= 4
        slots = torch.randperm(pages * ps, generator=g, device=DEV)[:t]  # (int64)
        slots[torch.rand(t, generator=g, device=DEV) < 0.03] = -1  # padding of the batch: not written
        k, v = rows[:, -2 * kv:-kv], rows[:, -kv:]
        return dict(cache=cache, slots=slots, **(dict(k=k, v=v) if c["fused"] else dict(k=k.contiguous(), v=v.contiguous())))
    lengths, span = _lengths(c), _span(c)
    used = [-(-n // ps) for n in lengths]
    into = -(-c["keep"] // ps) if op == "evict" else 0
    pages = sum(used) + c["batch"] * into + 3
    order = torch.randperm(pages, generator=g, device=DEV).int()
    table = torch.full((c["batch"], span), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    s = dict(cache=_filled_cache(g, c, pages), table=table, host=lengths,
             lengths=torch.tensor(lengths, dtype=torch.int32).to(DEV))
    cap = span * ps
    reached = torch.arange(cap, device=DEV)[None, None, :] < s["lengths"][:, None, None]
    if op == "evict":
        w = torch.exp(2 * _normal(g, (c["batch"], kv, cap)) - 4)
        w = torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.3, 0.0, w)  # (many were never looked at)
        return dict(s, weights=torch.where(reached, w, 0.0),
                    into=order[at:at + c["batch"] * into].reshape(c["batch"], into).contiguous())
    rows = c["batch"] * c["queries"]
    s["q"] = (_normal(g, (rows, c["heads"], d)) * 1.5).to(FLOAT[c["dtype"]])
    if c["queries"] > 1:
        s["starts"] = torch.arange(0, rows + 1, c["queries"], dtype=torch.int32, device=DEV)
    else:
        s["starts"] = None
    if op == "weights":
        s["lse"] = _plain_attention(c, s)["lse"]
        s["weights"] = torch.where(reached, torch.rand((c["batch"], kv, cap), generator=g, device=DEV), 0.0) if c["before"] else None
    return s


def prepare(case, seed):
    """inputs, the cache, and the output buffers and workspaces that a serving loop keeps"""
    c = case
    s = dict(c=c, **_inputs(c, seed))
    op = c["op"]
    empty = lambda shape, dt: torch.empty(shape, dtype=dt, device=DEV)  # noqa: E731
    if op == "attention":
        s["buf"] = dict(out=empty(s["q"].shape, s["q"].dtype), lse=empty(s["q"].shape[:2], torch.float32))
    elif op == "weights":
        s["buf"] = dict(out=torch.zeros((c["batch"], c["kv"], _span(c) * c["page"]), device=DEV))
    elif op == "evict":
        s["buf"] = dict(kept=empty((c["batch"], c["kv"], c["keep"]), torch.int32), lengths_out=empty(c["batch"], torch.int32),
                        weights_out=empty(s["weights"].shape, torch.float32))
    if own:
        s["kv"] = _lib().KvCache(**s["cache"])
        if op == "attention":
            bytes_ = _lib().kv_attention_workspace_size(s["q"], s["kv"], s["table"], starts=s["starts"], max_queries=c["queries"],
                                                        window=c["window"])
            s["buf"]["workspace"] = empty(max(bytes_, 1), torch.uint8)
    return s


# ------------------------------------------------------------------------------------------------
# the plain forms: elementary operations in 32 bits
# ------------------------------------------------------------------------------------------------
def _plain_append(c, s):
    cache, slots, ps = s["cache"], s["slots"], c["page"]
    total = cache["k"].shape[0] * ps
    # (a row that is not written rewrites what the last slot holds; no shape depends on the data)
    live = (slots >= 0) & (slots < total)
    for name in ("k", "v"):
        packed, scale = _quantize(s[name], c["group"])
        for pool, new in ((cache[name], packed), (cache[name + "_scale"], scale)):
            flat = pool.transpose(1, 2).reshape(total, *new.shape[1:])  # [slot, key head, ...]
            wide = torch.cat([flat, flat[:1]])  # the last row takes what is not written
            wide[torch.where(live, slots, total)] = new
            pool.copy_(wide[:-1].reshape(pool.shape[0], ps, *new.shape[1:]).transpose(1, 2))
    return cache


def _rows(c, cache, name, pages, n):
    """the first n tokens of a row of pages, in 32 bits: [key head, token, channel]"""
    code = cache[name][pages].transpose(0, 1)
    code = code.reshape(code.shape[0], -1, code.shape[-1])[:, :n]
    scale = cache[name + "_scale"][pages].transpose(0, 1)
    scale = scale.reshape(scale.shape[0], -1, *scale.shape[3:])[:, :n].float()
    low = ((code & 15) ^ 8).float() - 8
    high = ((code >> 4) ^ 8).float() - 8
    x = torch.stack([low, high], dim=-1).reshape(*code.shape[:2], -1, c["group"])
    return (x * scale[..., :1] + scale[..., 1:]).half().float().reshape(*code.shape[:2], -1)


def _scores(c, s, b):
    """scaled products of a sequence's queries [key head, query of the group, token], what they see, and its pages"""
    n, kv, d, per = s["host"][b], c["kv"], c["d"], c["queries"]
    pages = s["table"][b, :-(-n // c["page"])].long()
    k = _rows(c, s["cache"], "k", pages, n)
    q = s["q"][b * per:(b + 1) * per].float()
    q = q.reshape(per, kv, -1, d).transpose(0, 1).reshape(kv, -1, d)
    x = (q @ k.transpose(1, 2).contiguous()) * (1 / math.sqrt(d))
    at = torch.arange(n, device=DEV)[None, :]
    last = (n - per + torch.arange(per, device=DEV))[:, None]  # a query's own position
    seen = at <= last
    if c["window"]:
        seen = seen & (at > last - c["window"])
    return x, seen.repeat_interleave(c["heads"] // kv, dim=0)[None], pages


def _plain_attention(c, s):
    kv, d, per = c["kv"], c["d"], c["queries"]
    out, lse = torch.empty_like(s["q"]), torch.empty(s["q"].shape[:2], device=DEV)
    for b, n in enumerate(s["host"]):
        x, seen, pages = _scores(c, s, b)
        x = torch.where(seen, x, -math.inf)
        top = x.amax(dim=-1, keepdim=True)
        p = torch.exp(x - top)
        total = p.sum(dim=-1, keepdim=True)
        o = (p @ _rows(c, s["cache"], "v", pages, n)) / total
        o = o.reshape(kv, per, -1, d).transpose(0, 1).reshape(per, c["heads"], d)
        out[b * per:(b + 1) * per] = o.to(out.dtype)
        lse[b * per:(b + 1) * per] = (top + torch.log(total)).reshape(kv, per, -1).transpose(0, 1).reshape(per, -1)
    return dict(out=out, lse=lse)


def _plain_weights(c, s):
    out = s["buf"]["out"]
    for b, n in enumerate(s["host"]):
        x, seen, _ = _scores(c, s, b)
        lse = s["lse"][b * c["queries"]:(b + 1) * c["queries"]]
        lse = lse.reshape(c["queries"], c["kv"], -1).transpose(0, 1).reshape(c["kv"], -1, 1)
        new = torch.where(seen, torch.exp(x - lse), 0.0).sum(dim=1)
        out[b, :, :n] = new if s["weights"] is None else s["weights"][b, :, :n] + new
    return out


def _plain_evict(c, s):
    keep, recent, ps = c["keep"], c["recent"], c["page"]
    cap = s["weights"].shape[2]
    at = torch.arange(cap, device=DEV)[None, None, :]
    n = s["lengths"][:, None, None]
    # heaviest first, of equal ones the first; the last `recent` before all, what was not reached behind all
    w = torch.where(at >= n - recent, math.inf, s["weights"])
    w = torch.where(at < n, w, -math.inf)
    order = torch.argsort(w, dim=2, descending=True, stable=True)[:, :, :keep]
    at = torch.arange(keep, device=DEV)[None, None, :]
    kept = torch.sort(torch.where(at < n, order, cap), dim=2).values
    live = at < n
    if kept.shape[2] < keep:
        kept = torch.nn.functional.pad(kept, (0, keep - kept.shape[2]), value=cap)
    buf = s["buf"]
    buf["kept"].copy_(torch.where(live, kept, -1))
    buf["lengths_out"].copy_(s["lengths"].clamp_max(keep))
    buf["weights_out"].zero_()
    buf["weights_out"][:, :, :keep] = torch.where(live, s["weights"].gather(2, kept.clamp_max(cap - 1)), 0.0)
    page = s["table"].long().gather(1, (kept.clamp_max(cap - 1) // ps).reshape(c["batch"], -1)).reshape(kept.shape)
    page, row = torch.where(live, page, 0), kept % ps
    head = torch.arange(c["kv"], device=DEV)[None, :, None].expand_as(kept)
    target = s["into"].long().gather(1, (at // ps).expand(c["batch"], 1, keep).reshape(c["batch"], -1)).reshape(-1, 1, keep)
    target, place = target.expand_as(kept), (at % ps).expand_as(kept)
    for pool in s["cache"].values():
        moved = pool[page, head, row]
        mask = live.expand_as(kept).reshape(*kept.shape, *[1] * (moved.dim() - 3))
        pool[target, head, place] = torch.where(mask, moved, pool[target, head, place])
    return dict(kept=buf["kept"], lengths=buf["lengths_out"], weights=buf["weights_out"], **s["cache"])


# ------------------------------------------------------------------------------------------------
# the library's calls
# ------------------------------------------------------------------------------------------------
def _run_own(s):
    a, c, op = _lib(), s["c"], s["c"]["op"]
    if op == "append":
        a.kv_append(s["kv"], s["k"], s["v"], s["slots"])
        return s["cache"]
    if op == "attention":
        out, lse = a.kv_attention(s["q"], s["kv"], s["table"], s["lengths"], starts=s["starts"], max_queries=c["queries"],
                                  window=c["window"], **s["buf"])
        return dict(out=out, lse=lse)
    if op == "weights":
        return a.kv_weights(s["q"], s["lse"], s["kv"], s["table"], s["lengths"], weights=s["weights"], starts=s["starts"],
                            max_queries=c["queries"], window=c["window"], **s["buf"])
    kept, lengths, weights = a.kv_evict(s["kv"], s["table"], s["lengths"], s["weights"], c["keep"], c["recent"],
                                        into=s["into"], **s["buf"])
    return dict(kept=kept, lengths=lengths, weights=weights, **s["cache"])


def run(state):
    if own:
        return _run_own(state)
    c = state["c"]
    return {"append": _plain_append, "attention": _plain_attention, "weights": _plain_weights,
            "evict": _plain_evict}[c["op"]](c, state)


def work(case):
    c, op = case, case["op"]
    kv, d, heads = c["kv"], c["d"], c["heads"]
    half = d // 2 + 4 * (d // c["group"])  # bytes of a token's keys (or values) in a head's cache
    if op == "append":
        es = {"f16": 2, "bf16": 2, "f32": 4}[c["dtype"]]
        return dict(bytes=2 * c["tokens"] * kv * (d * es + half) + 8 * c["tokens"], flops=10 * c["tokens"] * kv * d)
    lengths = _lengths(c)
    if op == "evict":
        moved = sum(min(n, c["keep"]) for n in lengths) * kv
        return dict(bytes=sum(lengths) * kv * 4 + moved * (4 * half + 4 + 4), flops=4 * sum(lengths) * kv)
    per, window = c["queries"], c["window"]
    read = pairs = 0
    for n in lengths:
        read += min(n, window + per - 1) if window else n
        first = n - per + 1  # tokens that the first query sees; each later one sees one more
        pairs += sum(min(first + i, window) if window else first + i for i in range(per))
    rows = len(lengths) * per * heads
    if op == "attention":
        return dict(bytes=read * kv * 2 * half + rows * (2 * d * 2 + 4), flops=4 * pairs * heads * d)
    return dict(bytes=read * kv * half + sum(lengths) * kv * 4 * (2 if c["before"] else 1) + rows * (2 * d + 4),
                flops=2 * pairs * heads * d)


# ------------------------------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ------------------------------------------------------------------------------------------------
def _exact_tokens(c, s, name, b, h, n):
    """tokens 0 .. n - 1 of sequence b in key head h as the cache's values [n, d]"""
    ps, t = c["page"], torch.arange(n, device=DEV)
    where = s["table"][b].long()[t // ps]
    byte = s["cache"][name][where, h, t % ps].int()
    nibble = torch.empty((n, c["d"]), dtype=torch.int32, device=DEV)
    nibble[:, 0::2], nibble[:, 1::2] = byte % 16, byte // 16
    code = torch.where(nibble < 8, nibble, nibble - 16).double()
    pair = s["cache"][name + "_scale"][where, h, t % ps].double().repeat_interleave(c["group"], dim=1)
    return (code * pair[..., 0] + pair[..., 1]).half().double()


def exact(case, seed):
    c, op = case, case["op"]
    s = _inputs(c, seed)
    if op == "append":
        out = dict(k=None, v=None)
        live = s["slots"] >= 0
        at = s["slots"][live]
        for name in ("k", "v"):
            rows = s[name][live].double().clamp(-LIMIT, LIMIT).unflatten(2, (-1, c["group"]))
            low = rows.min(dim=3).values
            scale = (rows.max(dim=3).values - low) / 15
            offset = low + 8 * scale.half().double()  # (by the scale as it is kept)
            pairs = torch.zeros(s["cache"][name + "_scale"].shape, dtype=torch.float64, device=DEV)
            pairs[at // c["page"], :, at % c["page"]] = torch.stack([scale, offset], dim=-1)
            out[name + "_scale"] = pairs
        return out
    if op == "evict":
        w = torch.zeros(s["weights"].shape, dtype=torch.float64, device=DEV)
        for b, n in enumerate(s["host"]):
            old = max(0, n - c["recent"])
            for h in range(c["kv"]):
                row = s["weights"][b, h].double()
                light = torch.sort(row[:old], stable=True, descending=True).indices[:max(0, min(n, c["keep"]) - (n - old))]
                stay = torch.zeros(row.shape, dtype=torch.bool, device=DEV)
                stay[light] = True
                stay[old:n] = True
                picked = row[stay][:c["keep"]]
                w[b, h, :picked.numel()] = picked
        return dict(kept=None, lengths=None, weights=w, k=None, v=None, k_scale=None, v_scale=None)
    per, heads, kv, d = c["queries"], c["heads"], c["kv"], c["d"]
    g = heads // kv
    out = torch.zeros((len(s["host"]) * per, heads, d), dtype=torch.float64, device=DEV)
    lse = torch.zeros((len(s["host"]) * per, heads), dtype=torch.float64, device=DEV)
    got = torch.zeros((c["batch"], kv, _span(c) * c["page"]), dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["host"]):
        i = torch.arange(per, device=DEV)[:, None]
        t = torch.arange(n, device=DEV)[None, :]
        hidden = t > n - per + i
        if c["window"]:
            hidden = hidden | (t <= n - per + i - c["window"])
        at = slice(b * per, (b + 1) * per)
        for h in range(kv):
            k = _exact_tokens(c, s, "k", b, h, n)
            v = _exact_tokens(c, s, "v", b, h, n) if op == "attention" else None
            for j in range(h * g, (h + 1) * g):
                x = torch.mm(s["q"][at, j].double(), k.t().contiguous()) / d ** 0.5
                x = x.masked_fill(hidden, -math.inf)
                if op == "attention":
                    lse[at, j] = torch.logsumexp(x, dim=1)
                    out[at, j] = torch.mm(torch.softmax(x, dim=1), v)
                else:
                    got[b, h, :n] += torch.exp(x - s["lse"][at, j, None].double()).sum(dim=0)
        if op == "weights" and c["before"]:
            got[b, :, :n] += s["weights"][b, :, :n].double()
    return dict(out=out, lse=lse) if op == "attention" else got
