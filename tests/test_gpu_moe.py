"""Expert routing, its gradients, and the rows' movement (ascq_moe_*) against plain 64-bit implementations.

Tolerances.  Choices, counts and orders are whole numbers and equal.  A softmax probability: exp's argument is an fp32
difference (exact to 2^-24 of |l| + |top| <= 32 here: 4e-6 relative) and exp, sum and quotient take E / 64 + 16 roundings.
The loss adds up to 2^14 probabilities in steps of 64 tokens (1e-6 a step of 64, below 1e-5 in all).  A gradient is a sum of
a few products of such numbers: 1e-5 of the sum of their magnitudes, and half an ulp of its type.  The combine adds k
products in fp32 (2^-24 (k + 1) of their magnitudes) and rounds once; its weight gradient adds n products in n / 256 + 16
steps."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
ULP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def _logits(t, e, dt, seed, masked=0.0, padded=0.0, ties=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, e, generator=g) * 2 + torch.randn(e, generator=g)
    if ties:
        x = x.round()
    x = torch.where(torch.rand(t, e, generator=g) < masked, -math.inf, x)
    x = torch.where(torch.rand(t, 1, generator=g) < padded, -math.inf, x)
    return x.to(DT[dt])


def _reference(logits, k, renormalize):
    """token by token, in 64 bits"""
    x = logits.double()
    x = torch.where(torch.isnan(x), -math.inf, x).clamp_max(3.402823466e38)
    t, e = x.shape
    p = torch.zeros(t, e, dtype=torch.float64)
    experts = torch.full((t, k), -1, dtype=torch.int32)
    weights = torch.zeros(t, k, dtype=torch.float64)
    by_expert = [[] for _ in range(e)]
    routed = 0
    for i in range(t):
        row = x[i].tolist()
        live = [j for j in range(e) if row[j] > -math.inf]
        if not live:
            continue
        routed += 1
        top = max(row[j] for j in live)
        ex = {j: math.exp(row[j] - top) for j in live}
        total = sum(ex.values())
        for j in live:
            p[i, j] = ex[j] / total
        pick = sorted(live, key=lambda j: (-row[j], j))[:k]
        w = [ex[j] / total for j in pick]
        s = sum(w)
        for at, j in enumerate(pick):
            experts[i, at] = j
            weights[i, at] = w[at] / s if renormalize else w[at]
            by_expert[j].append((i, at))
    slots = torch.full((t, k), -1, dtype=torch.int32)
    tokens = torch.full((t * k,), -1, dtype=torch.int32)
    row = 0
    for j in range(e):
        for i, at in by_expert[j]:
            slots[i, at] = row
            tokens[row] = i
            row += 1
    counts = torch.tensor([len(b) for b in by_expert], dtype=torch.int64)
    loss = 0.0
    if routed:
        loss = e * float((counts.double() / row * p.sum(dim=0) / routed).sum())
    return dict(p=p, weights=weights, experts=experts, slots=slots, tokens=tokens, counts=counts, routed=routed, loss=loss)


def _check_route(r, want):
    for key in ("experts", "slots", "tokens", "counts"):
        assert torch.equal(getattr(r, key).cpu(), want[key]), key
    assert r.routed.item() == want["routed"]
    assert torch.all((r.weights.cpu().double() - want["weights"]).abs() <= 1.2e-5 * want["weights"] + 1e-37)
    assert abs(r.loss.item() - want["loss"]) <= 2e-5 * want["loss"]


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 8, 2), (16, 16, 2), (63, 60, 4), (64, 64, 8), (65, 64, 6), (200, 7, 7),
                                   (130, 128, 8), (129, 256, 8), (70, 300, 16), (40, 512, 4), (66, 1024, 16), (1000, 16, 2),
                                   (300, 33, 3), (257, 2, 1)])
def test_route(ascq_gpu, t, e, k, dt, renormalize):
    for masked, padded, ties in ((0.0, 0.0, False), (0.5, 0.2, False), (0.1, 0.0, True)):
        x = _logits(t, e, dt, t * e + k, masked, padded, ties)
        r = ascq_gpu.moe_route(x.cuda(), k, renormalize)
        _check_route(r, _reference(x, k, renormalize))


def test_route_many_tokens(ascq_gpu):
    for t, e, k in ((5000, 64, 6), (16385, 8, 2)):
        x = _logits(t, e, "f32", 3, 0.0, 0.1)
        _check_route(ascq_gpu.moe_route(x.cuda(), k), _reference(x, k, True))


def test_route_is_the_same_every_time(ascq_gpu):
    x = _logits(4096, 64, "bf16", 8, 0.1, 0.1).cuda()
    first = ascq_gpu.moe_route(x, 6)
    for _ in range(5):
        again = ascq_gpu.moe_route(x, 6)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("e,k", [(16, 4), (64, 8), (100, 3)])
def test_route_special_logits(ascq_gpu, e, k):
    """NaN and -inf mask an expert, +inf counts as the largest finite number, the type's lowest value is a number like
    others; rows of one or no expert left; equal logits go to the lowest experts"""
    for dt in ("f32", "bf16", "f16"):
        x = _logits(12, e, dt, 2)
        low = torch.finfo(DT[dt]).min
        x[0] = 0.25
        x[1] = low
        x[2] = low
        x[2, e - 1] = 1.0
        x[3] = math.nan
        x[4] = -math.inf
        x[4, 5] = -3.0
        x[5, 3] = math.nan
        x[6, 1] = math.inf
        x[7, 1] = x[7, e - 2] = math.inf
        x[8] = -math.inf
        x[9] = math.inf
        x[10] = -math.inf
        x[10, 2] = x[10, 7] = low
        want = _reference(x, k, True)
        _check_route(ascq_gpu.moe_route(x.cuda(), k), want)
        assert want["experts"][0].tolist() == list(range(k)) and want["experts"][3].tolist() == [-1] * k


def test_route_all_padding_and_no_tokens(ascq_gpu):
    r = ascq_gpu.moe_route(torch.full((100, 8), -math.inf, device="cuda"), 2)
    assert r.counts.sum() == 0 and r.routed.item() == 0 and r.loss.item() == 0
    assert torch.all(r.experts == -1) and torch.all(r.slots == -1) and torch.all(r.tokens == -1) and torch.all(r.weights == 0)
    r = ascq_gpu.moe_route(torch.empty((0, 8), device="cuda"), 2)
    assert r.counts.sum() == 0 and r.routed.item() == 0 and r.loss.item() == 0


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("e,pad,shift", [(16, 3, 1), (64, 8, 0), (60, 1, 5), (256, 40, 8)])
def test_route_strides(ascq_gpu, e, pad, shift, dt):
    t, k = 75, 3
    x = _logits(t, e, dt, 4, 0.2)
    b = torch.full((t * (e + pad) + shift,), 50.0, dtype=DT[dt], device="cuda")
    v = b[shift:].view(t, e + pad)[:, :e]
    v.copy_(x)
    r = ascq_gpu.moe_route(v, k)
    _check_route(r, _reference(x, k, True))
    g = torch.full_like(b, 7.0)
    gv = g[shift:].view(t, e + pad)[:, :e]
    ascq_gpu.moe_route_grad(v, r.weights, r.experts, r.counts, r.routed, grad_loss=torch.ones(1, device="cuda"), out=gv)
    dense = ascq_gpu.moe_route_grad(x.cuda(), r.weights, r.experts, r.counts, r.routed, grad_loss=torch.ones(1, device="cuda"))
    assert torch.equal(gv, dense)
    assert torch.all(g[shift:].view(t, e + pad)[:, e:] == 7.0)


def _grad_reference(x, want, k, renormalize, dw, dl):
    """the formula, in 64 bits, and the sum of the magnitudes it adds"""
    p, experts = want["p"], want["experts"].long()
    t, e = p.shape
    c = want["counts"].double()
    live = p.sum(dim=1) > 0
    g = torch.zeros(t, e, dtype=torch.float64)
    if dl is not None and want["routed"]:
        g += dl * e * c / (c.sum() * want["routed"])
    d = torch.zeros(t, e, dtype=torch.float64)
    size = torch.zeros(t, e, dtype=torch.float64)
    if dw is not None:
        for i in range(t):
            js = [j for j in range(k) if experts[i, j] >= 0]
            w = want["weights"][i]
            mean = sum(float(dw[i, j] * w[j]) for j in js)
            mag = sum(abs(float(dw[i, j] * w[j])) for j in js)
            for j in js:
                if renormalize:
                    d[i, experts[i, j]] += w[j] * (dw[i, j] - mean)
                    size[i, experts[i, j]] += w[j] * (abs(dw[i, j]) + mag)
                else:
                    g[i, experts[i, j]] += dw[i, j]
    dot = (p * g).sum(dim=1, keepdim=True)
    out = torch.where(live[:, None], p * (g - dot) + d, 0.0)
    return out, size + p * (g.abs() + (p * g.abs()).sum(dim=1, keepdim=True))


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,e,k", [(1, 8, 2), (17, 16, 2), (64, 64, 8), (90, 60, 4), (50, 7, 7), (33, 256, 8), (20, 1024, 16),
                                   (9, 300, 5), (5, 1, 1)])
def test_route_grad(ascq_gpu, t, e, k, dt, renormalize):
    g = torch.Generator().manual_seed(t + e)
    dw = torch.randn(t, k, generator=g)
    dl = torch.tensor([3.0])
    for masked, padded in ((0.0, 0.0), (0.5, 0.3)):
        x = _logits(t, e, dt, e, masked, padded)
        want = _reference(x, k, renormalize)
        r = ascq_gpu.moe_route(x.cuda(), k, renormalize)
        for use_w, use_l in ((True, True), (True, False), (False, True), (False, False)):
            got = ascq_gpu.moe_route_grad(x.cuda(), r.weights, r.experts, r.counts, r.routed,
                                          grad_weights=dw.cuda() if use_w else None, grad_loss=dl.cuda() if use_l else None,
                                          renormalize=renormalize)
            ref, size = _grad_reference(x, want, k, renormalize, dw.double() if use_w else None, 3.0 if use_l else None)
            off = (got.cpu().double() - ref).abs() - (ULP[dt] * ref.abs() + 2e-5 * size + (6e-8 if dt == "f16" else 1e-37))
            assert torch.all(off <= 0), (use_w, use_l, off.max())


@pytest.mark.parametrize("renormalize", [True, False])
def test_route_grad_against_differences(ascq_gpu, renormalize):
    """central differences of the 64-bit forward, the choices and counts held"""
    t, e, k = 6, 12, 3
    x = _logits(t, e, "f32", 21, 0.2)
    want = _reference(x, k, renormalize)
    dw = torch.randn(t, k, generator=torch.Generator().manual_seed(1)).double()
    c = want["counts"].double()

    def value(z):
        p = torch.softmax(z, dim=1)
        w = torch.where(want["experts"] >= 0, p.gather(1, want["experts"].clamp_min(0).long()), 0.0)
        if renormalize:
            w = w / w.sum(dim=1, keepdim=True)
        return float((w * dw).sum() + 2.0 * e * (c / c.sum() * p.sum(dim=0) / want["routed"]).sum())

    r = ascq_gpu.moe_route(x.cuda(), k, renormalize)
    got = ascq_gpu.moe_route_grad(x.cuda(), r.weights, r.experts, r.counts, r.routed, grad_weights=dw.float().cuda(),
                                  grad_loss=torch.tensor([2.0], device="cuda"), renormalize=renormalize).cpu()
    z = x.double()
    for i in range(t):
        for j in range(e):
            if not math.isfinite(z[i, j]):
                assert got[i, j] == 0
                continue
            up, down = z.clone(), z.clone()
            up[i, j] += 1e-5
            down[i, j] -= 1e-5
            # (third derivatives are at most a few units: 1e-10; the forward's rounding over the step 1e-11)
            assert abs((value(up) - value(down)) / 2e-5 - got[i, j].item()) <= 5e-6 * max(1.0, abs(got[i, j].item()))


def _routing(ascq, t, e, k, seed, padded=0.0):
    x = _logits(t, e, "f32", seed, 0.3 if padded else 0.0, padded)
    return ascq.moe_route(x.cuda(), k)


@pytest.mark.parametrize("dt", [torch.int8, torch.float8_e4m3fn, torch.float16, torch.float32])
@pytest.mark.parametrize("t,e,k,n,padded", [(1, 8, 2, 64, 0), (16, 16, 2, 4096, 0), (65, 8, 3, 1000, 0.3), (40, 16, 1, 17, 0.2),
                                            (300, 60, 4, 512, 0.25), (9, 64, 16, 8191, 0)])
def test_dispatch(ascq_gpu, t, e, k, n, padded, dt):
    r = _routing(ascq_gpu, t, e, k, n, padded)
    g = torch.Generator().manual_seed(n)
    bits = {torch.int8: torch.int8, torch.float8_e4m3fn: torch.int8, torch.float16: torch.int16, torch.float32: torch.int32}[dt]
    for pad, shift in ((0, 0), (16, 0), (3, 1)):
        raw = torch.randint(-100, 100, (t * (n + pad) + shift,), generator=g).to(bits).cuda()
        x = raw.view(dt)[shift:].view(t, n + pad)[:, :n]
        s = torch.rand(t, generator=g).cuda()
        rows, scale = ascq_gpu.moe_dispatch(x, s, r.slots, r.tokens)
        at = r.tokens.long()
        xi = x.contiguous().view(bits)
        want = torch.where(at[:, None] >= 0, xi[at.clamp_min(0)], torch.zeros_like(xi[:1]))
        assert torch.equal(rows.view(bits), want)
        assert torch.equal(scale, torch.where(at >= 0, s[at.clamp_min(0)], torch.zeros_like(s[:1])))
        rows, none = ascq_gpu.moe_dispatch(x, None, r.slots, r.tokens)
        assert none is None and torch.equal(rows.view(bits), want)


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("t,e,k,n,padded", [(1, 8, 2, 64, 0), (16, 16, 2, 4096, 0), (65, 8, 3, 1000, 0.3), (40, 16, 1, 17, 0.2),
                                            (200, 60, 4, 512, 0.25), (5, 64, 16, 8191, 0), (3, 16, 2, 20000, 0)])
def test_combine_and_its_gradients(ascq_gpu, t, e, k, n, padded, dt):
    r = _routing(ascq_gpu, t, e, k, n + 1, padded)
    g = torch.Generator().manual_seed(n)
    y, res, dout = (torch.randn(s, generator=g).to(DT[dt]) for s in ((t * k, n), (t, n), (t, n)))
    y[r.tokens.cpu() < 0] = math.nan  # rows of no token are not read
    slots, w = r.slots.cpu().long(), r.weights.cpu().double()
    parts = torch.where(slots[:, :, None] >= 0, w[:, :, None] * y.double()[slots.clamp_min(0)], torch.zeros(1, dtype=torch.float64))
    for residual in (res, None):
        want = parts.sum(dim=1) + (0 if residual is None else residual.double())
        mag = parts.abs().sum(dim=1) + (0 if residual is None else residual.double().abs())
        got = ascq_gpu.moe_combine(y.cuda(), r.slots, r.weights, residual=None if residual is None else residual.cuda())
        assert torch.all((got.cpu().double() - want).abs() <= ULP[dt] * want.abs() + (k + 2) * 2.0 ** -24 * mag + 2.0 ** -25)
    into = res.cuda()
    assert ascq_gpu.moe_combine(y.cuda(), r.slots, r.weights, residual=into, out=into) is into
    assert torch.equal(into, ascq_gpu.moe_combine(y.cuda(), r.slots, r.weights, residual=res.cuda()))
    # gradients
    dw, dy = ascq_gpu.moe_combine_grad(dout.cuda(), y.cuda(), r.slots, r.tokens, r.weights)
    prod = torch.where(slots[:, :, None] >= 0, dout.double()[:, None, :] * y.double()[slots.clamp_min(0)],
                       torch.zeros(1, dtype=torch.float64))
    bound = (n / 256 + 32) * 2.0 ** -24
    assert torch.all((dw.cpu().double() - prod.sum(dim=2)).abs() <= bound * prod.abs().sum(dim=2))
    want = torch.zeros(t * k, n, dtype=torch.float64)
    for i in range(t):
        for j in range(k):
            if slots[i, j] >= 0:
                want[slots[i, j]] = w[i, j] * dout[i].double()
    assert torch.all((dy.cpu().double() - want).abs() <= (ULP[dt] + 2.0 ** -23) * want.abs() + 2.0 ** -25)
    only, none = ascq_gpu.moe_combine_grad(dout.cuda(), y.cuda(), r.slots, r.tokens, r.weights, need_grad_y=False)
    assert none is None and torch.equal(only, dw)


def test_combine_grad_against_differences(ascq_gpu):
    """the combine is linear in its weights and rows: differences of the kernel's own forward in f32"""
    t, e, k, n = 5, 8, 2, 96
    r = _routing(ascq_gpu, t, e, k, 1)
    g = torch.Generator().manual_seed(0)
    y, dout = torch.randn(t * k, n, generator=g).cuda(), torch.randn(t, n, generator=g).cuda()
    dw, dy = ascq_gpu.moe_combine_grad(dout, y, r.slots, r.tokens, r.weights)
    value = lambda yy, ww: (ascq_gpu.moe_combine(yy, r.slots, ww).double() * dout.double()).sum().item()  # noqa: E731
    for i, j in ((0, 0), (2, 1), (4, 1)):
        up, down = r.weights.clone(), r.weights.clone()
        up[i, j] += 0.5
        down[i, j] -= 0.5
        # (n outputs of about 1, each rounded at 2^-24 of its size: 1e-6 in all, over a step of 1)
        assert abs(value(y, up) - value(y, down) - dw[i, j].item()) <= 2e-5 * n ** 0.5
    for row, c in ((0, 0), (7, 50), (9, 95)):
        up, down = y.clone(), y.clone()
        up[row, c] += 0.5
        down[row, c] -= 0.5
        assert abs(value(up, r.weights) - value(down, r.weights) - dy[row, c].item()) <= 1e-5


def test_slots_out_of_range_are_ignored(ascq_gpu):
    """slots that no routing gives (past the rows, negative) count as no choice: nothing is read or written there"""
    t, k, n = 4, 2, 64
    slots = torch.tensor([[0, 8], [100000, 1], [2, -5], [2 ** 31 - 1, 3]], dtype=torch.int32, device="cuda")
    tokens = torch.tensor([0, 1, 2, 3, -1, -1, -1, -1], dtype=torch.int32, device="cuda")
    w = torch.ones(t, k, device="cuda")
    y = torch.randn(t * k, n, device="cuda")
    out = ascq_gpu.moe_combine(y, slots, w)
    assert torch.equal(out, torch.stack([y[0], y[1], y[2], y[3]]))
    x = torch.randn(t, n, device="cuda")
    rows, _ = ascq_gpu.moe_dispatch(x, None, slots, tokens)
    assert torch.equal(rows[:4], x) and torch.all(rows[4:] == 0)
    dw, dy = ascq_gpu.moe_combine_grad(x, y, slots, tokens, w)
    assert torch.equal(dy[:4], x) and torch.all(dy[4:] == 0)
    assert torch.all(dw.flatten()[[1, 2, 5, 6]] == 0)


def test_experts_out_of_range_are_ignored(ascq_gpu):
    x = torch.randn(3, 8, device="cuda")
    r = ascq_gpu.moe_route(x, 2)
    odd = r.experts.clone()
    odd[0, 1] = 8
    odd[1, 0] = 2 ** 31 - 1
    odd[2, 1] = -7
    g = ascq_gpu.moe_route_grad(x, r.weights, odd, r.counts, r.routed, grad_weights=torch.ones(3, 2, device="cuda"))
    assert torch.isfinite(g).all()


def test_on_another_stream(ascq_gpu):
    x = _logits(3000, 64, "f32", 5)
    gx = x.cuda()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    r = ascq_gpu.moe_route(gx, 4, stream=st)
    st.synchronize()
    _check_route(r, _reference(x, 4, True))


@pytest.mark.parametrize("t,e,k", [(64, 256, 8), (40, 1000, 16), (64, 16, 2), (33, 300, 4)])
def test_route_without_workspace(ascq_gpu, t, e, k):
    """Up to 64 tokens the C entry runs without a workspace, also where it would use one."""
    x = _logits(t, e, "f32", 5, 0.1, 0.1).cuda()
    want = ascq_gpu.moe_route(x, k)
    r = ascq_gpu.MoeRouting(*(torch.full_like(v, -7) for v in want))
    p = ascq_gpu._RouteParam(t, e, e, ascq_gpu._FLOAT_CODE[torch.float32], k, 1)
    status = ascq_gpu.lib().ascq_moe_route(*(v.data_ptr() for v in r), x.data_ptr(), ctypes.byref(p), None, 0,
                                           torch.cuda.current_stream().cuda_stream)
    assert status == ascq_gpu.OK
    for name in ("experts", "slots", "tokens", "counts", "routed", "weights"):
        assert torch.equal(getattr(r, name), getattr(want, name)), name
    assert torch.allclose(r.loss, want.loss, rtol=1e-5, atol=0)  # the tokens' sums come in another order


@pytest.mark.parametrize("t,e,k", [(17, 700, 3), (500, 100, 5), (2048, 256, 8), (2049, 65, 2), (33000, 9, 1)])
def test_route_chunks(ascq_gpu, t, e, k):
    """Short chunks of tokens for many experts, long ones, and more of them than blocks."""
    x = _logits(t, e, "bf16", 7, 0.2, 0.1, True)
    _check_route(ascq_gpu.moe_route(x.cuda(), k), _reference(x, k, True))


@pytest.mark.parametrize("t,e,k,n", [(300, 60, 8, 2056), (600, 8, 3, 1000), (1100, 16, 1, 2049), (1025, 4, 2, 5)])
def test_many_rows(ascq_gpu, t, e, k, n):
    test_dispatch(ascq_gpu, t, e, k, n, 0.2, torch.int8)
    test_combine_and_its_gradients(ascq_gpu, t, e, k, n, 0.2, "bf16")
