"""The operators of a quantised transformer block around its matrix products, measured through the public Python binding.

A case is a dict of plain values with an "op":
  norm          h = x + residual, RMS norm of h, 8-bit codes with one scale per token
  linear        8-bit activations (a scale per token) times an 8-bit weight (a scale per channel), bias, activation and
                residual in the epilogue
  route         top-k experts of a token, their weights, the tokens per expert, the rows' order by expert, balance loss
  route_grad    the gradient of the balance loss and of the weights with respect to the logits
  dispatch      the tokens' 8-bit rows and scales into the order of the experts
  combine       the experts' rows back into the tokens' order: their weighted sum and the residual
  combine_grad  the gradients of that sum with respect to the weights and to the experts' rows
Sizes are those of the repository's benchmark and tests -- rows of 4096, 8192 and 11008, 1 to 8192 tokens, 8192 x 8192 x
8192, 1030 x 4100 x 4095 -- and ordinary expert counts (8 to 256, 2 to 8 per token).

Where `own` is false, `run` computes them from elementary torch operations in 32 bits; where it is true, it makes the
library's calls.  int8 codes are whole numbers, the same in both; e4m3 codes are float8 values.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
FLOAT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "fp8": 448.0}  # the largest code
EPS = 1e-6
CUBE = 8192 ** 3  # M N K of the largest listed linear

_ascq = None


def _lib():
    global _ascq
    if _ascq is None:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "asc-devkit_clone_amd"))
        import ascq

        _ascq = ascq
    return _ascq


def listed():
    return [
        # the input of a W8A8 layer in one decode step of 16 sequences: the smallest call, latency
        dict(name="norm_decode", op="norm", m=16, n=4096, dtype="f16", codes="int8", residual=True, pad=0),
        # a large prefill's rows for an fp8 layer: HBM
        dict(name="norm_8192", op="norm", m=8192, n=8192, dtype="bf16", codes="fp8", residual=True, pad=0),
        # up projection at a decode batch: the weight stream
        dict(name="linear_decode", op="linear", m=16, n=11008, k=4096, codes="int8", out="f16", act="silu", bias=True,
             residual=False, w_trans=True),
        # fp8 down projection of a prefill batch, added to the residual stream
        dict(name="linear_fp8_2048", op="linear", m=2048, n=4096, k=11008, codes="fp8", out="bf16", act="none", bias=False,
             residual=True, w_trans=True),
        # the largest
        dict(name="linear_8192", op="linear", m=8192, n=8192, k=8192, codes="int8", out="bf16", act="gelu", bias=True,
             residual=True, w_trans=False),
        # sizes that divide nothing (an odd batch, a K and an N that were never padded), f32 out as for logits
        dict(name="linear_ragged", op="linear", m=1030, n=4100, k=4095, codes="int8", out="f32", act="relu", bias=True,
             residual=True, w_trans=True),
        # the router in one decode step of 16 sequences: latency
        dict(name="route_decode", op="route", tokens=16, experts=16, k=2, dtype="f32", padded=0.0, masked=False,
             renormalize=True),
        # a large batch over many experts, an eighth of it padding
        dict(name="route_16384", op="route", tokens=16384, experts=64, k=6, dtype="f32", padded=0.125, masked=False,
             renormalize=True),
        # its backward pass in a training step of the router
        dict(name="route_grad_16384", op="route_grad", tokens=16384, experts=64, k=6, dtype="f32", padded=0.125,
             masked=False, renormalize=True),
        # 4096 tokens of 4096 to two experts of 16 each, int8
        dict(name="dispatch_4096", op="dispatch", tokens=4096, experts=16, k=2, n=4096, codes="int8", padded=0.0),
        # and back
        dict(name="combine_4096", op="combine", tokens=4096, experts=16, k=2, n=4096, dtype="bf16", residual=True,
             padded=0.0),
        # its backward pass
        dict(name="combine_grad_4096", op="combine_grad", tokens=4096, experts=16, k=2, n=4096, dtype="bf16", padded=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, step):
    return max(lo, _log(rng, lo, hi) // step * step)


def draw(rng):
    op = rng.choice(["norm", "norm", "linear", "linear", "linear", "route", "route", "route_grad", "dispatch", "combine",
                     "combine_grad"])
    odd = rng.random() < 0.3
    while True:
        if op == "norm":
            c = dict(op=op, m=_log(rng, 1, 16384), n=_size(rng, 512, 16384, 1 if odd else 64),
                     dtype=rng.choice(["f16", "bf16", "f32"]), codes=rng.choice(["int8", "fp8"]),
                     residual=rng.random() < 0.7, pad=rng.choice([0, 0, 64, 8192]))
            cost, most = c["m"] * c["n"] * (2 if c["dtype"] == "f32" else 1), 8192 * 8192
        elif op == "linear":
            codes = rng.choice(["int8", "fp8"])
            c = dict(op=op, m=rng.choice([_log(rng, 1, 64), _log(rng, 1, 8192)]), n=_size(rng, 512, 14336, 1 if odd else 64),
                     k=_size(rng, 512, 14336, (1 if codes == "int8" else 16) if odd else 128), codes=codes,
                     # (16-bit outputs from fp8 operands, whose products the matrix unit aligns in groups of 16)
                     out=rng.choice(["f16", "bf16", "f32"] if codes == "int8" else ["f16", "bf16"]),
                     act=rng.choice(["none", "none", "relu", "gelu", "silu", "faster_gelu"]), bias=rng.random() < 0.6,
                     residual=rng.random() < 0.5, w_trans=rng.random() < 0.6)
            cost, most = c["m"] * c["n"] * c["k"], CUBE // (8 if odd else 1)
        else:
            experts, k = rng.choice([(8, 2), (16, 2), (16, 4), (64, 6), (64, 8), (128, 8), (256, 8), (60, 4), (7, 1)])
            c = dict(op=op, tokens=_log(rng, 1, 16384), experts=experts, k=k, padded=rng.choice([0.0, 0.0, 0.25]))
            if op in ("route", "route_grad"):
                c.update(dtype=rng.choice(["f32", "bf16", "f16"]), masked=rng.random() < 0.3, renormalize=rng.random() < 0.6)
                cost, most = c["tokens"] * experts, 16384 * 256
            else:
                c["n"] = _size(rng, 512, 8192, 1 if odd else 64)
                if op == "dispatch":
                    c["codes"] = rng.choice(["int8", "fp8"])
                else:
                    c["dtype"] = rng.choice(["f16", "bf16", "f32"])
                if op == "combine":
                    c["residual"] = rng.random() < 0.7
                cost, most = c["tokens"] * k * c["n"], 16384 * 2 * 4096
        if cost <= most:
            return c


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, shape):
    return torch.randn(shape, generator=g, device=DEV)


def _uniform(g, shape):
    return torch.rand(shape, generator=g, device=DEV)


def _code_tensor(g, shape, codes):
    """8-bit codes of normal data: int8 as absmax quantisation leaves it, or e4m3 values"""
    if codes == "int8":
        return (_normal(g, shape) * 32).round_().clamp_(-127, 127).to(torch.int8)
    return (_normal(g, shape) * 64).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _logits(g, c):
    """router logits: some experts are more popular than others; padding tokens have every expert masked"""
    t, e = c["tokens"], c["experts"]
    x = _normal(g, (t, e)) * 1.5 + _normal(g, (e,)) * 0.7
    if c.get("masked"):  # choices limited to some of the experts
        x = torch.where(_uniform(g, (t, e)) < 0.4, -math.inf, x)
    pad = _uniform(g, (t, 1)) < c["padded"]
    return torch.where(pad, -math.inf, x).to(FLOAT[c.get("dtype", "f32")] if c["op"].startswith("route") else torch.float32)


def _inputs(c, seed):
    g, op = _gen(seed), c["op"]
    if op == "norm":
        m, n, dt = c["m"], c["n"], FLOAT[c["dtype"]]
        outlier = 1 + 20 * (_uniform(g, (n,)) < 0.004).float()  # a few large channels, as residual streams have
        x = torch.empty((m, n + c["pad"]), dtype=dt, device=DEV)[:, :n]
        x.copy_(_normal(g, (m, n)))
        return dict(x=x, gamma=(0.5 + _uniform(g, (n,))).to(dt),
                    residual=(_normal(g, (m, n)) * outlier).to(dt) if c["residual"] else None)
    if op == "linear":
        m, n, k, dt = c["m"], c["n"], c["k"], FLOAT[c["out"]]
        code = 32.0 if c["codes"] == "int8" else 64.0
        return dict(x=_code_tensor(g, (m, k), c["codes"]), x_scale=(0.5 + _uniform(g, (m,))) / code,
                    w=_code_tensor(g, (n, k) if c["w_trans"] else (k, n), c["codes"]),
                    w_scale=(0.5 + _uniform(g, (n,))) / (code * math.sqrt(k)),
                    bias=_normal(g, (n,)) * 0.3 if c["bias"] else None,
                    residual=_normal(g, (m, n)).to(dt) if c["residual"] else None)
    t = dict(logits=_logits(g, c))
    if op == "route":
        return t
    routing = _plain_route(t["logits"], c["k"], c.get("renormalize", True))
    rows = c["tokens"] * c["k"]
    if op == "route_grad":
        return dict(t, **{key: routing[key] for key in ("weights", "experts", "counts", "routed")},
                    grad_weights=_normal(g, (c["tokens"], c["k"])) * 0.1, grad_loss=_uniform(g, (1,)) * 0.01 * c["tokens"])
    t = {key: routing[key] for key in ("weights", "slots", "tokens")}
    if op == "dispatch":
        t.update(q=_code_tensor(g, (c["tokens"], c["n"]), c["codes"]), scale=0.01 + 0.02 * _uniform(g, (c["tokens"],)))
    else:
        dt = FLOAT[c["dtype"]]
        t["y"] = _normal(g, (rows, c["n"])).to(dt)
        other = _normal(g, (c["tokens"], c["n"])).to(dt)
        if op == "combine_grad":
            t["grad_out"] = other
        else:
            t["residual"] = other if c["residual"] else None
    return t


def prepare(case, seed):
    """inputs, weights and the output buffers that a serving or training loop keeps"""
    c = case
    s = dict(c=c, **_inputs(c, seed))
    empty = lambda shape, dt: torch.empty(shape, dtype=dt, device=DEV)  # noqa: E731
    op = c["op"]
    if op == "norm":
        shape, dt = (c["m"], c["n"]), FLOAT[c["dtype"]]
        s["buf"] = dict(out=empty(shape, CODES[c["codes"]]), scale_out=empty(c["m"], torch.float32),
                        residual_out=empty(shape, dt) if c["residual"] else None)
    elif op == "linear":
        s["buf"] = dict(out=empty((c["m"], c["n"]), FLOAT[c["out"]]))
    elif op == "route":
        t, e, k = c["tokens"], c["experts"], c["k"]
        s["buf"] = dict(weights=empty((t, k), torch.float32), experts=empty((t, k), torch.int32),
                        slots=empty((t, k), torch.int32), tokens=empty(t * k, torch.int32), counts=empty(e, torch.int64),
                        routed=empty(1, torch.int64), loss=empty(1, torch.float32))
    elif op == "route_grad":
        s["buf"] = dict(out=torch.empty_like(s["logits"]))
    elif op == "dispatch":
        rows = c["tokens"] * c["k"]
        s["buf"] = dict(out=empty((rows, c["n"]), CODES[c["codes"]]), scale_out=empty(rows, torch.float32))
    elif op == "combine":
        s["buf"] = dict(out=empty((c["tokens"], c["n"]), FLOAT[c["dtype"]]))
    else:
        s["buf"] = dict(out=empty((c["tokens"], c["k"]), torch.float32), grad_y_out=torch.empty_like(s["y"]))
    return s


# ------------------------------------------------------------------------------------------------
# the plain forms: elementary operations in 32 bits
# ------------------------------------------------------------------------------------------------
def _plain_norm(x, residual, gamma, codes):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    f = h.float()
    rstd = torch.rsqrt((f * f).mean(dim=1) + EPS)
    t = f * gamma.float()
    top = t.abs().amax(dim=1)
    # (the row's rstd cancels in its codes)
    q = t * torch.where(top > 0, TOP[codes] / top, 0.0)[:, None]
    q = q.round().to(torch.int8) if codes == "int8" else q.clamp(-448, 448).to(torch.float8_e4m3fn)
    out = dict(q=q, scale=top * rstd / TOP[codes])
    return out if residual is None else dict(out, h=h)


def _activate(v, act):
    if act == "relu":
        return torch.clamp_min(v, 0)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "faster_gelu":
        return v / (1 + torch.exp(-1.702 * v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return v


def _plain_linear(x, x_scale, w, w_scale, bias, residual, act, w_trans, dtype):
    w = w.float()
    v = (x.float() @ (w.t() if w_trans else w)) * w_scale * x_scale[:, None]
    v = _activate(v if bias is None else v + bias, act)
    return (v if residual is None else v + residual.float()).to(dtype)


def _probabilities(logits):
    """softmax of finite logits, -inf and NaN counting nothing; a row without any is all zeros"""
    f = torch.nan_to_num(logits.double() if logits.dtype == torch.float64 else logits.float(), nan=-math.inf,
                         posinf=math.inf, neginf=-math.inf)
    top = f.amax(dim=1, keepdim=True)
    routed = top > -math.inf
    p = torch.exp(f - torch.where(routed, top, 0.0))
    return f, p / torch.where(routed, p.sum(dim=1, keepdim=True), 1.0), routed[:, 0]


def _plain_route(logits, k, renormalize):
    f, p, routed = _probabilities(logits)
    tokens, experts = f.shape
    value, index = torch.sort(f, dim=1, descending=True, stable=True)
    value, index = value[:, :k], index[:, :k]
    chosen = value > -math.inf
    w = torch.where(chosen, p.gather(1, index), 0.0)
    if renormalize:
        total = w.sum(dim=1, keepdim=True)
        w = w / torch.where(total > 0, total, 1.0)
    key = torch.where(chosen, index, experts).reshape(-1)
    order = torch.argsort(key, stable=True)  # rows by expert, then token; choices of nobody last
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device=order.device)
    counts = (key[:, None] == torch.arange(experts, device=key.device)).sum(dim=0)
    total = counts.sum()
    routed = routed.sum()
    share = counts.to(f.dtype) / torch.clamp_min(total, 1)
    mean = p.sum(dim=0) / torch.clamp_min(routed, 1)
    return dict(weights=w, experts=torch.where(chosen, index, -1).int(),
                slots=torch.where(chosen, slots.reshape(chosen.shape), -1).int(),
                tokens=torch.where(torch.arange(order.numel(), device=order.device) < total, order // k, -1).int(),
                counts=counts, routed=routed.reshape(1), loss=(experts * (share * mean).sum()).reshape(1))


def _plain_route_grad(logits, weights, experts, counts, routed, grad_weights, grad_loss, renormalize):
    f, p, row = _probabilities(logits)
    total = torch.clamp_min(counts.sum(), 1)
    g = grad_loss.to(f.dtype) * f.shape[1] * counts.to(f.dtype) / (total * torch.clamp_min(routed, 1))
    g = g.expand_as(f)
    chosen = experts >= 0
    dw = torch.where(chosen, grad_weights.to(f.dtype), 0.0)
    at = torch.where(chosen, experts, 0).long()
    w = weights.to(f.dtype)
    if not renormalize:
        g = g.scatter_add(1, at, dw)
    d = p * (g - (p * g).sum(dim=1, keepdim=True))
    if renormalize:
        d = d.scatter_add(1, at, w * (dw - (dw * w).sum(dim=1, keepdim=True)))
    return torch.where(row[:, None], d, 0.0).to(logits.dtype)


def _plain_dispatch(q, scale, tokens):
    used, at = tokens >= 0, tokens.clamp_min(0).long()
    rows = q.view(torch.int8)[at]
    return dict(q=torch.where(used[:, None], rows, 0).view(q.dtype), scale=torch.where(used, scale[at], 0.0))


def _plain_combine(y, slots, weights, residual):
    w = torch.where(slots >= 0, weights, 0.0)
    rows = y.float()[slots.clamp_min(0).long()]
    v = (w[:, :, None] * rows).sum(dim=1)
    return (v if residual is None else v + residual.float()).to(y.dtype)


def _plain_combine_grad(grad_out, y, slots, tokens, weights):
    used, d = slots >= 0, grad_out.float()
    rows = y.float()[slots.clamp_min(0).long()]
    dw = torch.where(used, (d[:, None, :] * rows).sum(dim=2), 0.0)
    w = torch.zeros(tokens.numel() + 1, device=DEV)  # by row; the last takes the choices of nobody
    w[torch.where(used, slots, tokens.numel()).long().reshape(-1)] = weights.reshape(-1)
    dy = torch.where(tokens[:, None] >= 0, w[:-1, None] * d[tokens.clamp_min(0).long()], 0.0)
    return dict(weights=dw, y=dy.to(y.dtype))


def _run_plain(s):
    c, op = s["c"], s["c"]["op"]
    if op == "norm":
        return _plain_norm(s["x"], s["residual"], s["gamma"], c["codes"])
    if op == "linear":
        return _plain_linear(s["x"], s["x_scale"], s["w"], s["w_scale"], s["bias"], s["residual"], c["act"], c["w_trans"],
                             FLOAT[c["out"]])
    if op == "route":
        return _plain_route(s["logits"], c["k"], c["renormalize"])
    if op == "route_grad":
        return _plain_route_grad(s["logits"], s["weights"], s["experts"], s["counts"], s["routed"], s["grad_weights"],
                                 s["grad_loss"], c["renormalize"])
    if op == "dispatch":
        return _plain_dispatch(s["q"], s["scale"], s["tokens"])
    if op == "combine":
        return _plain_combine(s["y"], s["slots"], s["weights"], s["residual"])
    return _plain_combine_grad(s["grad_out"], s["y"], s["slots"], s["tokens"], s["weights"])


# ------------------------------------------------------------------------------------------------
# the library's calls
# ------------------------------------------------------------------------------------------------
def _run_own(s):
    a, c, op, buf = _lib(), s["c"], s["c"]["op"], s["buf"]
    if op == "norm":
        q, scale, h = a.add_rms_norm_quant(s["x"], s["gamma"], EPS, a.INT8 if c["codes"] == "int8" else a.FP8_E4M3,
                                           residual=s["residual"], **buf)
        return dict(q=q, scale=scale) if s["residual"] is None else dict(q=q, scale=scale, h=h)
    if op == "linear":
        act = {"none": a.ACT_NONE, "relu": a.ACT_RELU, "gelu": a.ACT_GELU, "silu": a.ACT_SILU,
               "faster_gelu": a.ACT_FASTER_GELU}[c["act"]]
        return a.quant_linear(s["x"], s["x_scale"], s["w"], s["w_scale"], bias=s["bias"], activation=act,
                              residual=s["residual"], w_trans=c["w_trans"], **buf)
    if op == "route":
        r = a.moe_route(s["logits"], c["k"], renormalize=c["renormalize"], out=a.MoeRouting(**buf))
        return r._asdict()
    if op == "route_grad":
        return a.moe_route_grad(s["logits"], s["weights"], s["experts"], s["counts"], s["routed"],
                                grad_weights=s["grad_weights"], grad_loss=s["grad_loss"], renormalize=c["renormalize"],
                                **buf)
    if op == "dispatch":
        q, scale = a.moe_dispatch(s["q"], s["scale"], s["slots"], s["tokens"], **buf)
        return dict(q=q, scale=scale)
    if op == "combine":
        return a.moe_combine(s["y"], s["slots"], s["weights"], residual=s["residual"], **buf)
    dw, dy = a.moe_combine_grad(s["grad_out"], s["y"], s["slots"], s["tokens"], s["weights"], **buf)
    return dict(weights=dw, y=dy)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    c, op = case, case["op"]
    size = {"f16": 2, "bf16": 2, "f32": 4}
    if op == "norm":
        m, n, es = c["m"], c["n"], size[c["dtype"]]
        return dict(bytes=m * n * (es * (3 if c["residual"] else 1) + 1) + n * es + 4 * m, flops=6 * m * n)
    if op == "linear":
        m, n, k, es = c["m"], c["n"], c["k"], size[c["out"]]
        return dict(bytes=m * k + n * k + m * n * es * (2 if c["residual"] else 1) + 4 * m + 4 * n * (2 if c["bias"] else 1),
                    flops=2 * m * n * k)
    t, e, k = c["tokens"], c["experts"], c["k"]
    if op == "route":
        return dict(bytes=t * e * size[c["dtype"]] + 16 * t * k + 8 * e, flops=t * e * 4)
    if op == "route_grad":
        return dict(bytes=2 * t * e * size[c["dtype"]] + 12 * t * k + 8 * e, flops=t * e * 8)
    n, rows = c["n"], t * k
    if op == "dispatch":
        return dict(bytes=(t + rows) * (n + 4) + 8 * rows, flops=0)
    es = size[c["dtype"]]
    if op == "combine":
        return dict(bytes=(rows + t * (2 if c["residual"] else 1)) * n * es + 8 * rows, flops=2 * rows * n)
    return dict(bytes=(2 * rows + t) * n * es + 16 * rows, flops=3 * rows * n)


# ------------------------------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ------------------------------------------------------------------------------------------------
def _exact_softmax(z):
    """rows over their unmasked entries; 0 where masked, and in rows that are masked whole"""
    p = torch.softmax(z, dim=1)
    return torch.where(torch.isfinite(z), p, torch.zeros_like(p)).nan_to_num(nan=0.0)


def _exact_choice(z, k):
    """1 where an expert is chosen: fewer than k come before it (larger, or equal with a lower index)"""
    rank = torch.empty_like(z, dtype=torch.long)
    step = max(1, (1 << 27) // z.shape[1] ** 2)
    lower = torch.ones((z.shape[1], z.shape[1]), device=DEV, dtype=torch.bool).tril(-1)  # [e, other]: other < e
    for at in range(0, z.shape[0], step):
        part = z[at:at + step]
        before = (part[:, None, :] > part[:, :, None]) | ((part[:, None, :] == part[:, :, None]) & lower)
        rank[at:at + step] = before.sum(dim=2)
    return (rank < k) & torch.isfinite(z), rank


def _exact_routing(z, k, renormalize):
    """dense [tokens, experts] weights, the choices and their ranks, and the balance loss"""
    p = _exact_softmax(z)
    chosen, rank = _exact_choice(z.detach(), k)
    w = torch.where(chosen, p, torch.zeros_like(p))
    if renormalize:
        w = w / w.sum(dim=1, keepdim=True).clamp_min(1e-300)
    live = torch.isfinite(z).any(dim=1).sum().clamp_min(1)
    share = chosen.sum(dim=0).double() / chosen.sum().clamp_min(1)
    return w, chosen, rank, z.shape[1] * (share * (p.sum(dim=0) / live)).sum()


def exact(case, seed):
    c, s, op = case, _inputs(case, seed), case["op"]
    if op == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h = (h + s["residual"].double()).to(s["x"].dtype).double()
        normed = h / ((h ** 2).mean(dim=1, keepdim=True) + EPS).sqrt() * s["gamma"].double()
        scale = normed.abs().amax(dim=1) / TOP[c["codes"]]
        q = None
        if c["codes"] == "fp8":
            q = (normed / scale.clamp_min(1e-300)[:, None]).clamp(-448, 448).float().to(torch.float8_e4m3fn).double()
        out = dict(q=q, scale=scale)
        return out if s["residual"] is None else dict(out, h=h)
    if op == "linear":
        w = s["w"].float().double()
        x = s["x"].float().double() * s["x_scale"].double()[:, None]
        v = torch.matmul(x, w.t() if c["w_trans"] else w) * s["w_scale"].double()
        if s["bias"] is not None:
            v = v + s["bias"].double()
        if c["act"] == "relu":
            v = v * (v > 0)
        elif c["act"] == "gelu":
            v = v * torch.special.ndtr(v)
        elif c["act"] in ("silu", "faster_gelu"):
            v = v * torch.sigmoid(v * (1.0 if c["act"] == "silu" else 1.702))
        return v if s["residual"] is None else v + s["residual"].double()
    if op in ("route", "route_grad"):
        z = s["logits"].double()
        if op == "route":
            w, chosen, rank, loss = _exact_routing(z, c["k"], c["renormalize"])
            by_rank = torch.zeros((c["tokens"], c["experts"]), dtype=torch.float64, device=DEV)
            by_rank.scatter_(1, rank, torch.where(chosen, w, 0.0))
            return dict(weights=by_rank[:, :c["k"]], experts=None, slots=None, tokens=None, counts=None, routed=None,
                        loss=loss.reshape(1))
        # differentiated by autograd, from the same definition
        live = torch.isfinite(z)
        v = torch.where(live, z, 0.0).requires_grad_(True)
        w, chosen, rank, loss = _exact_routing(torch.where(live, v, -math.inf), c["k"], c["renormalize"])
        up = torch.zeros_like(w)
        up.scatter_add_(1, s["experts"].clamp_min(0).long(), torch.where(s["experts"] >= 0, s["grad_weights"].double(), 0.0))
        total = (torch.where(chosen, w * up, torch.zeros_like(w))).sum() + s["grad_loss"].double().sum() * loss
        return torch.autograd.grad(total, v)[0].nan_to_num(nan=0.0)
    if op == "dispatch":
        pick = s["tokens"].long()
        zero = torch.zeros(1, dtype=torch.float64, device=DEV)
        q = None
        if c["codes"] == "fp8":
            table = torch.cat([s["q"].float().double(), zero.expand(1, c["n"])])
            q = table[torch.where(pick < 0, c["tokens"], pick)]
        return dict(q=q, scale=torch.cat([s["scale"].double(), zero])[torch.where(pick < 0, c["tokens"], pick)])
    live = (s["slots"] >= 0).double()
    w = s["weights"].double() * live
    if op == "combine":
        v = torch.zeros((c["tokens"], c["n"]), dtype=torch.float64, device=DEV)
        for j in range(c["k"]):
            v += w[:, j, None] * s["y"][s["slots"][:, j].long().clamp(min=0)].double()
        return v if s["residual"] is None else v + s["residual"].double()
    d = s["grad_out"].double()
    dw = torch.zeros_like(w)
    dy = torch.zeros((c["tokens"] * c["k"], c["n"]), dtype=torch.float64, device=DEV)
    for j in range(c["k"]):
        at = s["slots"][:, j].long()
        dw[:, j] = (d * s["y"][at.clamp(min=0)].double()).sum(dim=1) * live[:, j]
        dy[at[at >= 0]] = (w[:, j, None] * d)[at >= 0]
    return dict(weights=dw, y=dy)
