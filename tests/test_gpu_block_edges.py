"""The block operators (ascq_add_rms_norm_quant, ascq_quant_linear, ascq_moe_*) at the edges of their ranges: streams beside each
other, infinities, tiny and empty rows, very many rows.  Each test states its tolerance."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_side_stream_beside_work_on_the_current_one(ascq_gpu):
    """Calls on a stream while the current one still writes to blocks it has given back: the calls' own memory is none of those
    (whole numbers, equal bits)"""
    a = ascq_gpu
    g = torch.Generator(device="cuda").manual_seed(7)
    x = (torch.randn(40, 8192, generator=g, device="cuda") * 30).clamp(-127, 127).to(torch.int8)
    w = (torch.randn(640, 8192, generator=g, device="cuda") * 30).clamp(-127, 127).to(torch.int8)
    xs, ws = torch.rand(40, generator=g, device="cuda"), torch.rand(640, generator=g, device="cuda")
    logits = torch.randn(3000, 64, generator=g, device="cuda")
    linear = lambda st: a.quant_linear(x, xs, w, ws, out_dtype=torch.float32, stream=st)  # noqa: E731
    want, route = linear(None), a.moe_route(logits, 6)
    need = a.quant_linear_workspace_size(x, w, True, torch.float32)
    assert need > 0
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for st in (side, side.cuda_stream):
        for _ in range(5):
            for size in (need, want.numel() * 4, 3000 * 6 * 4, 64 * 47 * 8):
                given_back = torch.empty(size, dtype=torch.uint8, device="cuda")
                for _ in range(30):
                    given_back.fill_(255)
                del given_back
            got, r = linear(st), a.moe_route(logits, 6, stream=st)
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            assert all(torch.equal(p, q) for p, q in zip(r, route))


def test_route_gradient_of_a_large_upstream_gradient(ascq_gpu):
    """grad_loss E counts / (sum counts routed) in an order that does not pass fp32's range while the result is inside it: the
    gradient of 2e38 is 2^100 times that of 2e38 / 2^100, bit for bit (a power of two; nothing here is subnormal)"""
    a = ascq_gpu
    x = torch.randn(40, 16, generator=torch.Generator().manual_seed(3)).cuda()
    r = a.moe_route(x, 2)
    grad = lambda v: a.moe_route_grad(x, r.weights, r.experts, r.counts, r.routed,  # noqa: E731
                                      grad_loss=torch.tensor([v], device="cuda"))
    large, small = grad(2e38), grad(2e38 / 2.0 ** 100)
    assert torch.isfinite(large).all() and torch.equal(large, small * 2.0 ** 100)


def _same(got, want):
    """equal bits, any NaN being as good as another"""
    assert got.dtype == want.dtype
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(torch.where(nan, 0, got), torch.where(nan, 0, want))


@pytest.mark.parametrize("n", [64, 77, 2048, 4099])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_combine_gradient_keeps_infinities(ascq_gpu, dt, n):
    """grad_y is one fp32 product rounded once to its type (so equal bits): infinities and NaN of grad_out arrive, and a
    product past the type's range is infinite -- what a loss scaler looks for"""
    a = ascq_gpu
    t, k = 5, 2
    slots = torch.arange(t * k, dtype=torch.int32, device="cuda").view(t, k)
    tokens = torch.arange(t * k, dtype=torch.int32, device="cuda") // k
    w = torch.full((t, k), 0.5, device="cuda")
    w[3] = 1e20
    g = torch.randn(t, n, generator=torch.Generator().manual_seed(n)).to(dt)
    g[1, 3], g[1, n - 1], g[2, 0], g[2, n // 2] = float("inf"), -float("inf"), float("nan"), torch.finfo(dt).max
    g = g.cuda()
    y = torch.ones(t * k, n, dtype=dt, device="cuda")
    dw, dy = a.moe_combine_grad(g, y, slots, tokens, w)
    _same(dy, (w.view(-1, 1) * g.float()[tokens.long()]).to(dt))
    assert torch.isinf(dy[2, 3]) and torch.isinf(dy[2, n - 1]) and torch.isnan(dy[4, 0])
    if dt is torch.float16:
        assert torch.isinf(dy[6:8]).all()  # 1e20 g
    assert torch.isnan(dw[1]).all() and torch.isnan(dw[2]).all()  # inf - inf, NaN


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("e", [8, 33, 64])
def test_route_gradient_overflows_to_infinity(ascq_gpu, e, dt, renormalize):
    """A gradient past its type's range is infinite (the f32 gradient, which the other tests compare, rounded once: its size
    is at least twice the type's largest, or at most half of it, wherever it is looked at)"""
    a = ascq_gpu
    t, k = 9, 2
    x = torch.randn(t, e, generator=torch.Generator().manual_seed(e)).to(dt).cuda()
    r = a.moe_route(x, k, renormalize)
    for scale in (1.0, 1e6, 1e38):
        up = torch.full((1,), scale, device="cuda")
        dw = torch.randn(t, k, generator=torch.Generator().manual_seed(1)).cuda() * scale
        got = a.moe_route_grad(x, r.weights, r.experts, r.counts, r.routed, grad_weights=dw, grad_loss=up, renormalize=renormalize)
        wide = a.moe_route_grad(x.float(), r.weights, r.experts, r.counts, r.routed, grad_weights=dw, grad_loss=up,
                                renormalize=renormalize)
        top = torch.finfo(dt).max
        over, under = wide.abs() > 2 * top, wide.abs() < top / 2
        assert torch.isinf(got[over]).all() and torch.equal(got[over].sign().float(), wide[over].sign())
        assert torch.isfinite(got[under]).all()
        if dt is torch.float16 and scale > 1e6:
            assert over.any()
    up.fill_(float("inf"))
    got = a.moe_route_grad(x, r.weights, r.experts, r.counts, r.routed, grad_loss=up, renormalize=renormalize)
    assert not torch.isfinite(got).any()


def _rounded(v, dt):
    """an fp32 value in dt: what is finite saturates, infinities and NaN stay"""
    top = torch.finfo(dt).max
    return torch.where(torch.isfinite(v), v.clamp(-top, top), v).to(dt)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [8, 96, 513, 4096, 66000])
def test_norm_of_an_infinite_sum(ascq_gpu, n, dt, codes):
    """an infinity or NaN in x or the residual: h keeps it (equal bits), codes 0, scale and norm NaN; the other rows are those of
    the same call without it"""
    a = ascq_gpu
    g = torch.Generator().manual_seed(n)
    x, r = torch.randn(9, n, generator=g).to(dt), torch.randn(9, n, generator=g).to(dt)
    gamma = (torch.rand(n, generator=g) + 0.5).to(dt).cuda()
    code = a.INT8 if codes == "int8" else a.FP8_E4M3
    plain = a.add_rms_norm_quant(x.cuda(), gamma, 1e-5, code, residual=r.cuda())
    inf, top = float("inf"), torch.finfo(dt).max
    x[1, 2] = inf
    r[2, n - 1] = -inf
    x[3, 0], r[3, 0] = inf, inf
    x[4, n // 2], r[4, n // 2] = inf, -inf
    x[5, 1], r[5, 1] = -inf, top
    r[7, n // 2] = float("nan")
    bad, good = [1, 2, 3, 4, 5, 7], [0, 6, 8]
    norm = torch.empty(9, n, dtype=dt, device="cuda")
    q, s, h = a.add_rms_norm_quant(x.cuda(), gamma, 1e-5, code, residual=r.cuda(), norm_out=norm)
    _same(h.cpu(), _rounded(x.float() + r.float(), dt))
    assert torch.isinf(h.cpu()[[1, 2, 3, 5], [2, n - 1, 0, 1]]).all()
    assert torch.all(q[bad].float() == 0) and torch.isnan(s[bad]).all() and torch.isnan(norm[bad]).all()
    assert torch.equal(q[good].view(torch.uint8), plain[0][good].view(torch.uint8)) and torch.equal(s[good], plain[1][good])
    into = x.cuda()
    again = a.add_rms_norm_quant(into, gamma, 1e-5, code, residual=r.cuda(), residual_out=into)
    _same(into, h)
    assert torch.equal(again[0].view(torch.uint8), q.view(torch.uint8))


@pytest.mark.parametrize("n", [64, 77, 2048])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_combine_keeps_infinities(ascq_gpu, dt, n):
    """infinities and NaN of the rows and the residual stay; a finite sum past a 16-bit type's range saturates.  (weights 1 and
    one choice: the fp32 sum y + residual is rounded once, and the result is equal to that)"""
    a = ascq_gpu
    t = 8
    slots = torch.arange(t, dtype=torch.int32, device="cuda").view(t, 1)
    g = torch.Generator().manual_seed(n)
    y, r = torch.randn(t, n, generator=g).to(dt), torch.randn(t, n, generator=g).to(dt)
    inf, top = float("inf"), torch.finfo(dt).max
    y[1, 3], r[2, n - 1], y[3, 0], r[3, 0] = inf, -inf, inf, -inf
    y[4, 5], r[5, 1] = float("nan"), float("nan")
    y[6], r[6] = top * 0.75, top * 0.5
    y[7], r[7] = -top, -inf
    got = a.moe_combine(y.cuda(), slots, torch.ones(t, 1, device="cuda"), residual=r.cuda()).cpu()
    _same(got, _rounded(y.float() + r.float(), dt))
    assert got[1, 3] == inf and got[2, n - 1] == -inf and torch.isnan(got[3, 0]) and torch.all(got[7] == -inf)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k,w_trans", [(3, 80, 128, True), (40, 77, 8192, True), (300, 260, 128, True), (300, 264, 128, False),
                                           (300, 77, 130, True), (4, 64, 0, True)])
def test_linear_keeps_infinities(ascq_gpu, m, n, k, w_trans, dt):
    """infinities and NaN of the bias and the residual stay; a finite value past a 16-bit type's range saturates.  (x is zero, so
    the result is the fp32 sum bias + residual rounded once, and equal to that.)"""
    a = ascq_gpu
    x = torch.zeros(m, k, dtype=torch.int8, device="cuda")
    w = torch.ones((n, k) if w_trans else (k, n), dtype=torch.int8, device="cuda")
    g = torch.Generator().manual_seed(n)
    bias, r = torch.randn(n, generator=g), torch.randn(m, n, generator=g).to(dt)
    inf, top = float("inf"), torch.finfo(dt).max
    bias[1], bias[n - 1], bias[5], bias[6] = inf, -inf, float("nan"), top / 2
    r[0, 3], r[1, n - 2], r[2, 1], r[2, 4] = inf, -inf, -inf, float("nan")
    r[:, 6] = top
    if dt is torch.float32:
        r[:, 6] = top / 4
    got = a.quant_linear(x, torch.ones(m, device="cuda"), w, torch.ones(n, device="cuda"), bias=bias.cuda(), residual=r.cuda(),
                         w_trans=w_trans, out_dtype=dt).cpu()
    _same(got, _rounded(bias + r.float(), dt))
    assert got[0, 3] == inf and got[1, n - 2] == -inf and torch.isnan(got[2, 1]) and got[0, n - 1] == -inf


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("e", [8, 60, 300])
def test_route_gradient_without_choices_out_of_range(ascq_gpu, e, renormalize):
    """a choice that is no expert counts as none, for the token's other choices too (equal bits)"""
    a = ascq_gpu
    t, k = 12, 3
    g = torch.Generator().manual_seed(e)
    x, dw = torch.randn(t, e, generator=g).cuda(), (torch.randn(t, k, generator=g) * 3).cuda()
    r = a.moe_route(x, k, renormalize)
    odd, none = r.experts.clone(), r.experts.clone()
    for i, (j, bad) in enumerate(((1, e), (0, 2 ** 31 - 1), (2, -7), (1, -(2 ** 31)), (0, e + 5))):
        odd[i, j], none[i, j] = bad, -1
    grad = lambda experts: a.moe_route_grad(x, r.weights, experts, r.counts, r.routed, grad_weights=dw,  # noqa: E731
                                            renormalize=renormalize)
    assert torch.equal(grad(odd), grad(none))
    assert not torch.equal(grad(odd)[:5], grad(r.experts)[:5]) and torch.equal(grad(odd)[5:], grad(r.experts)[5:])


@pytest.mark.parametrize("k,pitch", [(1, 1 << 32), (2, (1 << 31) - 8192), (3, 1 << 24)])
def test_linear_over_rows_far_apart(ascq_gpu, k, pitch):
    """w [k, n] of few rows, gigabytes apart: neither what lies between them nor what follows k in x's rows is multiplied (small
    whole numbers: exact)"""
    a = ascq_gpu
    m, n = 200, 320
    g = torch.Generator(device="cuda").manual_seed(k)
    raw = torch.full(((k - 1) * pitch + n,), 3, dtype=torch.int8, device="cuda")
    w = raw.as_strided((k, n), (pitch, 1))
    w.copy_(torch.randint(-9, 9, (k, n), generator=g, device="cuda", dtype=torch.int8))
    x = torch.full((m, 32), 5, dtype=torch.int8, device="cuda")[:, :k]
    x.copy_(torch.randint(-9, 9, (m, k), generator=g, device="cuda", dtype=torch.int8))
    ones = torch.ones(max(m, n), device="cuda")
    want = x.float() @ w.float()
    assert torch.equal(a.quant_linear(x, ones[:m], w, ones[:n], w_trans=False, out_dtype=torch.float32), want)
    f8 = torch.float8_e4m3fn
    xf, wf = torch.full((m, 32), float("nan"), device="cuda").to(f8)[:, :k], raw.float().to(f8).as_strided((k, n), (pitch, 1))
    xf.copy_(x.float().to(f8))
    assert torch.equal(a.quant_linear(xf, ones[:m], wf, ones[:n], w_trans=False, out_dtype=torch.float32), want)


def test_norm_of_very_many_rows(ascq_gpu):
    """more rows than a grid has room for: each as its like among the first (equal bits)"""
    a = ascq_gpu
    m, n, every = (1 << 26) + 5, 8, 1 << 16
    x = torch.randn(every, n, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").half()
    gamma = torch.linspace(0.5, 1.5, n, device="cuda").half()
    q, s, _ = a.add_rms_norm_quant(x, gamma)
    wide, ws, _ = a.add_rms_norm_quant(x.repeat((m + every - 1) // every, 1)[:m], gamma)
    assert torch.equal(wide[:-5].view(-1, every, n), q.expand(m // every, -1, -1)) and torch.equal(wide[-5:], q[:5])
    assert torch.equal(ws[:-5].view(-1, every), s.expand(m // every, -1)) and torch.equal(ws[-5:], s[:5])


def test_rows_of_very_many_tokens(ascq_gpu):
    """more tokens than a grid has room for: rows moved to the reverse order and back, and their gradients (equal bits: weights 1
    and 2, one choice)"""
    a = ascq_gpu
    t, n = (1 << 26) + 5, 8
    slots = torch.arange(t - 1, -1, -1, dtype=torch.int32, device="cuda").view(t, 1)
    x = torch.randint(-100, 100, (t, n), dtype=torch.int8, device="cuda")
    rows, _ = a.moe_dispatch(x, None, slots, slots.view(t))
    assert torch.equal(rows, x.flip(0))
    y = rows.half()
    del rows
    out = a.moe_combine(y, slots, torch.ones(t, 1, device="cuda"))
    assert torch.equal(out, x.half())
    two = torch.full((t, 1), 2.0, device="cuda")
    dw, dy = a.moe_combine_grad(out, y, slots, slots.view(t), two)
    assert torch.equal(dy, y * 2)
    assert torch.equal(dw.view(t), (x.float() ** 2).sum(dim=1))


def test_route_gradient_of_very_many_tokens(ascq_gpu):
    """more tokens than a grid of 64 lanes each has room for: each token as its like among the first (equal bits)"""
    a = ascq_gpu
    every, e = 1 << 16, 300
    x = torch.randn(every, e, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").half()
    r = a.moe_route(x, 1)
    ones = torch.ones(every, 1, device="cuda")
    args = dict(grad_loss=torch.full((1,), 64.0, device="cuda"), renormalize=False)
    want = a.moe_route_grad(x, r.weights, r.experts, r.counts, r.routed, grad_weights=ones, **args)
    t = (1 << 26) + 5  # (64 lanes a token)
    more = (t + every - 1) // every
    wide = x.repeat(more, 1)[:t]
    got = a.moe_route_grad(wide, r.weights.repeat(more, 1)[:t], r.experts.repeat(more, 1)[:t], r.counts, r.routed,
                           grad_weights=ones.repeat(more, 1)[:t], out=wide, **args)
    assert got is wide
    for at in range(0, t - every, every * 64):
        part = got[at:at + every * 64]
        assert torch.equal(part, want.repeat(64, 1)[:part.shape[0]])
    assert torch.equal(got[-5:], want[:5])


def test_linear_of_very_many_tiles(ascq_gpu):
    """more output tiles than a grid has room for (k = 0: the bias and the residual, exact)"""
    a = ascq_gpu
    m = (1 << 30) + 70
    r = torch.arange(1024, device="cuda").half().repeat(m // 1024 + 1)[:m].view(m, 1)
    got = a.quant_linear(torch.empty(m, 0, dtype=torch.int8, device="cuda"), torch.ones(m, device="cuda"),
                         torch.empty(1, 0, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"),
                         bias=torch.full((1,), 0.5, device="cuda"), residual=r, out_dtype=torch.float16)
    assert torch.equal(got, r + 0.5)


def test_rows_without_elements(ascq_gpu):
    """rows of no elements: the norm's scales are those of a row of zeros, the dispatch moves scales alone, the combine's weight
    gradients are sums of nothing"""
    a = ascq_gpu
    side = torch.cuda.Stream()
    for st in (None, side, side.cuda_stream):
        x = torch.empty(5, 0, dtype=torch.float16, device="cuda")
        full = torch.full((5,), 9.0, device="cuda")
        torch.cuda.synchronize()
        q, s, h = a.add_rms_norm_quant(x, torch.empty(0, dtype=torch.float16, device="cuda"), residual=x, scale_out=full, stream=st)
        torch.cuda.synchronize()
        assert s is full and torch.all(s == 0) and q.shape == (5, 0) and h.shape == (5, 0)
    tokens = torch.tensor([1, 0, 2, 2, -1, -1], dtype=torch.int32, device="cuda")
    slots = torch.tensor([[1, -1], [0, -1], [2, 3]], dtype=torch.int32, device="cuda")
    scale, got = torch.tensor([1.0, 2.0, 3.0], device="cuda"), torch.full((6,), 9.0, device="cuda")
    for dt in (torch.int8, torch.float16):
        rows, got = a.moe_dispatch(torch.empty(3, 0, dtype=dt, device="cuda"), scale, slots, tokens, scale_out=got.fill_(9.0))
        assert got.tolist() == [2.0, 1.0, 3.0, 3.0, 0.0, 0.0] and rows.shape == (6, 0)
    y, w = torch.empty(6, 0, device="cuda"), torch.ones(3, 2, device="cuda")
    dw, dy = a.moe_combine_grad(torch.empty(3, 0, device="cuda"), y, slots, tokens, w, out=torch.full((3, 2), 9.0, device="cuda"))
    assert torch.all(dw == 0) and dy.shape == (6, 0)
    assert a.moe_combine(y, slots, w).shape == (3, 0)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-5])
@pytest.mark.parametrize("dt,n", [("f32", 64), ("f32", 513), ("f32", 4096), ("f32", 16000), ("f32", 20001), ("f32", 70000),
                                  ("bf16", 96), ("bf16", 1000), ("bf16", 4100), ("bf16", 20000), ("bf16", 20001),
                                  ("bf16", 60000), ("bf16", 70000), ("f16", 640)])
def test_norm_of_tiny_rows(ascq_gpu, dt, n, eps, codes):
    """Rows, gammas and products far below 1, down to subnormal numbers: codes times scale is the norm of the definition in 64
    bits, as for ordinary rows, also where the squares or the products' reciprocal leave fp32's range.  Bounds of
    test_gpu_norm.py (the products' powers of two are exact, so the same roundings are taken), and a scale or norm that is
    subnormal itself is off by a unit of it."""
    from test_gpu_norm import DT, ULP, _check

    a = ascq_gpu
    g = torch.Generator().manual_seed(n)
    low = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}[dt]
    size = [1.0, 1e-12, 1e-16, 1e-19, 1e-22, 1e-30, 1e-36, 1e-38, 3e-39, 20 * low]
    if dt == "f16":
        size = [1.0, 1e-3, 1e-5, 1e-6, 20 * low]
    rows = torch.tensor(size, dtype=torch.float64)[:, None]
    x = (torch.randn(len(size), n, generator=g, dtype=torch.float64) * rows).to(DT[dt])
    r = (torch.randn(len(size), n, generator=g, dtype=torch.float64) * rows).to(DT[dt])
    x[0, 1:] = r[0] = 0  # one number, and zeros
    code = a.INT8 if codes == "int8" else a.FP8_E4M3
    for power in (0, -10, -60, -90, -120, 40):
        if dt == "f16" and power not in (0, -10):
            continue
        gamma = ((torch.rand(n, generator=g) + 0.5) * 2.0 ** power).to(DT[dt])
        gamma[3] = 0
        for residual in (None, r):
            norm = torch.empty(x.shape, dtype=DT[dt], device="cuda")
            into = x.cuda()
            q, s, h = a.add_rms_norm_quant(into, gamma.cuda(), eps, code, residual=None if residual is None else r.cuda(),
                                           residual_out=None if residual is None else into, norm_out=norm)
            h, s, norm = h.cpu(), s.cpu(), norm.cpu()
            t = h.double() * gamma.double()
            rstd = 1 / torch.sqrt((h.double() ** 2).mean(dim=1) + eps)
            # (products below half of fp32's smallest number are 0; a scale that rounds to 0 leaves codes of 0)
            none = t.abs().amax(dim=1) < 2.0 ** -150
            keep = (t.abs().amax(dim=1) * rstd / (127 if codes == "int8" else 448) > 2.0 ** -148) & ~none
            assert torch.all(s[none] == 0) and torch.all(q.cpu()[none].float() == 0) and torch.all(norm[none] == 0)
            assert keep.any()
            _check(x[keep], gamma, None if residual is None else r[keep], codes, q.cpu()[keep], s[keep], h[keep], eps=eps)
            assert torch.isfinite(s).all() and torch.all(q.float().abs() <= (127 if codes == "int8" else 448))
            assert torch.all(s[~keep] <= 2.0 ** -147)
            want = torch.where((t == 0) | none[:, None], 0.0, t * rstd[:, None])
            near = want.abs() < torch.finfo(DT[dt]).max / 2
            bound = (ULP[dt] + (n / 256 + 40) * 2.0 ** -24) * want.abs() + low
            assert torch.all(((norm.double() - want).abs() <= bound) | ~near)


@pytest.mark.parametrize("t,e", [(9, 8), (64, 64), (3000, 64), (600, 256), (70, 1000)])
def test_routing_weights_are_quotients(ascq_gpu, t, e):
    """A weight is a quotient rounded once, not a product with a rounded reciprocal: one choice renormalised has the weight 1,
    k equal ones 1 / k each, and of E equal logits any choice has 1 / E (powers of two: equal bits), whatever the logits are"""
    a = ascq_gpu
    x = (torch.randn(t, e, generator=torch.Generator().manual_seed(e)) * 3).cuda()
    assert torch.all(a.moe_route(x, 1).weights == 1.0)
    for k in (2, 4, 8):
        # (the k largest alike, the others anything below: their share of the softmax leaves the renormalised weights)
        y = x.clone()
        y.scatter_(1, x.topk(k).indices, x.amax(dim=1, keepdim=True).expand(-1, k))
        assert torch.all(a.moe_route(y, k).weights == 1.0 / k)
    for n in (2, 3, 7, 8):
        same = torch.randn(t, 1, generator=torch.Generator().manual_seed(n)).expand(t, n).contiguous().cuda()
        one = torch.ones(1, device="cuda")
        assert torch.all(a.moe_route(same, 1, renormalize=False).weights == one / n)


@pytest.mark.parametrize("m,k", [(1, 64), (3, 8192), (300, 64), (2, 0)])
@pytest.mark.parametrize("act", ["gelu", "silu", "faster_gelu"])
def test_activations_of_f32_outputs(ascq_gpu, act, m, k):
    """An f32 output has the activation to a few units of fp32, also where it is small.  x is zero, so the activation's argument is
    the bias, exactly.  GELU: the complementary error function is allowed 16 units, and its argument's two roundings move it by
    at most x^2 units and a few; the others: the exponential 3 units, its argument's rounding |b x|, an addition, a product and a
    division; a result below 2^-126 is off by units of the smallest number."""
    a = ascq_gpu
    v = torch.cat([torch.linspace(-14, 14, 4001), torch.linspace(-100, 100, 401), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e30, -1e30])])
    n = v.numel()
    code = dict(gelu=a.ACT_GELU, silu=a.ACT_SILU, faster_gelu=a.ACT_FASTER_GELU)[act]
    got = a.quant_linear(torch.zeros(m, k, dtype=torch.int8, device="cuda"), torch.ones(m, device="cuda"),
                         torch.zeros(n, k, dtype=torch.int8, device="cuda"), torch.ones(n, device="cuda"), bias=v.cuda(),
                         activation=code, out_dtype=torch.float32).cpu().double()
    z = v.double()
    if act == "gelu":
        want, units = 0.5 * z * torch.special.erfc(-z * 0.5 ** 0.5), 20 + z * z
    else:
        b = 1.0 if act == "silu" else 1.702
        e = torch.exp(-b * z.abs())
        want, units = z * torch.where(z < 0, e, 1.0) / (1 + e), 8 + b * z.abs()
    # (past 2^100 only the side that is the argument itself is left, or nothing)
    units = units.clamp_max(1e5)
    off = (got - want).abs() - (units * 2.0 ** -23 * want.abs() + 200 * 2.0 ** -149)
    assert torch.all(off <= 0), (act, v[off.max(dim=1).indices[0]], off.max())
    special = torch.tensor([float("inf"), -float("inf"), float("nan")])
    got = a.quant_linear(torch.zeros(m, k, dtype=torch.int8, device="cuda"), torch.ones(m, device="cuda"),
                         torch.zeros(3, k, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda"), bias=special.cuda(),
                         activation=code, out_dtype=torch.float32).cpu()
    assert torch.all(torch.isinf(got[:, 0])) and torch.all(got[:, 1] == 0) and torch.all(torch.isnan(got[:, 2]))


@pytest.mark.parametrize("m,n,k", [(1, 4000, 64), (3, 4004, 8192), (300, 4000, 64), (300, 4004, 64)])
@pytest.mark.parametrize("act", ["gelu", "silu", "faster_gelu"])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_activations_of_16_bit_outputs(ascq_gpu, dt, act, m, n, k):
    """A 16-bit output is the activation rounded once, where it is small too: half a unit of the type, and a hundredth of one for
    the activation's own error -- GELU's polynomial 1.3e-6, exponentials of rounded arguments x^2 2^-23 and 4 units, some more
    roundings: below 2e-5 in all where the result is normal.  x is zero, so the activation's argument is the bias, exactly."""
    a = ascq_gpu
    v = torch.cat([torch.linspace(-9, 9, 3000), torch.linspace(-60, 60, n - 3000)])
    code = dict(gelu=a.ACT_GELU, silu=a.ACT_SILU, faster_gelu=a.ACT_FASTER_GELU)[act]
    got = a.quant_linear(torch.zeros(m, k, dtype=torch.int8, device="cuda"), torch.ones(m, device="cuda"),
                         torch.zeros(n, k, dtype=torch.int8, device="cuda"), torch.ones(n, device="cuda"), bias=v.cuda(),
                         activation=code, out_dtype=dt).cpu().double()
    z = v.double()
    if act == "gelu":
        want = 0.5 * z * torch.special.erfc(-z * 0.5 ** 0.5)
    else:
        e = torch.exp(-(1.0 if act == "silu" else 1.702) * z.abs())
        want = z * torch.where(z < 0, e, 1.0) / (1 + e)
    half, low = (2.0 ** -11, 2.0 ** -25) if dt is torch.float16 else (2.0 ** -8, 2.0 ** -126)
    binade = torch.exp2(torch.floor(torch.log2(want.abs().clamp_min(1e-300))))
    off = (got - want).abs() - (half * 1.0001 * binade + 2e-5 * want.abs() + low)
    assert torch.all(off <= 0), (act, v[off.max(dim=1).indices[0]], off.max())


@pytest.mark.parametrize("w_trans", [True, False])
@pytest.mark.parametrize("m,n,k,shift", [(1, 512, 4096, 0), (16, 1024, 1024, 0), (17, 512, 8192, 0), (40, 256, 11008, 0),
                                         (64, 512, 2048, 0), (100, 384, 11008, 0), (300, 516, 4096, 0), (1030, 1100, 1003, 0),
                                         (2048, 2048, 1024, 0), (70, 100, 515, 3), (5, 64, 144, 1)])
def test_fp8_sums_of_f32_outputs(ascq_gpu, m, n, k, shift, w_trans):
    """An f32 output of e4m3 operands has fp32 sums.  Of normal data, against 64 bits, normwise: K / 32 accumulations that each
    round the sum so far (2^-24 of it, in both directions alike: their square root), and eight roundings more for the products
    inside one, the scales and the store."""
    a = ascq_gpu
    g = torch.Generator(device="cuda").manual_seed(m + n)

    def codes(rows, cols):
        pad = torch.zeros(rows * cols + 64, device="cuda").to(torch.float8_e4m3fn)
        v = pad[shift:shift + rows * cols].view(rows, cols)
        v.copy_((torch.randn(rows, cols, generator=g, device="cuda") * 64).clamp(-448, 448).to(torch.float8_e4m3fn))
        return v

    x, w = codes(m, k), codes(n, k) if w_trans else codes(k, n)
    xs, ws = (torch.rand(s, generator=g, device="cuda") + 0.5 for s in (m, n))
    wf = w.float().double()
    want = x.float().double() @ (wf.t().contiguous() if w_trans else wf) * ws.double() * xs.double()[:, None]
    for room in (None, torch.empty(1, dtype=torch.uint8, device="cuda")):
        got = a.quant_linear(x, xs, w, ws, w_trans=w_trans, out_dtype=torch.float32, workspace=room)
        assert (got.double() - want).norm() <= ((k / 32) ** 0.5 + 8) * 2.0 ** -24 * want.norm()
