"""The block operators together: the example's mixture-of-experts block, graph capture, and calls on several streams."""
from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


def _example():
    spec = importlib.util.spec_from_file_location("quantized_moe_block", ROOT / "examples" / "quantized_moe_block.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("tokens,hidden,ffn,experts,top_k", [(1, 512, 256, 8, 2), (70, 512, 320, 16, 4), (600, 1024, 384, 8, 2)])
def test_block_matches_fp32(ascq_gpu, tokens, hidden, ffn, experts, top_k):
    """int8 rows and weights put uniform errors of 1 / 254 of the largest element into each factor; a row's largest of n
    normal elements is about sqrt(2 ln n) <= 4 times its size, so a product of two is off by 4 sqrt(2) / 254 / sqrt(3) = 1.3 %,
    and two products in a row by 2 %; 4 % is twice that"""
    _, _, err, loss, gradient = _example().run(tokens, hidden, ffn, experts, top_k)
    assert err < 0.04
    assert torch.isfinite(gradient).all()
    assert abs(gradient.sum(dim=1)).max() < 1e-4  # a softmax's gradient sums to nothing
    assert 0.9 < loss < experts


def test_capture(ascq_gpu):
    """every operator recorded in a graph and replayed over new inputs equals the eager calls, bit for bit"""
    a = ascq_gpu
    t, hidden, e, k = 40, 1024, 64, 4
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x, res, gamma = rnd(t, hidden).half(), rnd(t, hidden).half(), rnd(hidden).half()
    w = (rnd(e, hidden) * 30).clamp(-127, 127).to(torch.int8)
    wide = (rnd(hidden, 8192) * 30).clamp(-127, 127).to(torch.int8)  # K = 8192: sums of a split K
    act = (rnd(t, 8192) * 30).clamp(-127, 127).to(torch.int8)
    ones = torch.ones(8192, device="cuda") / 1000
    dout = rnd(t, hidden).half()

    def step():
        q, s, h = a.add_rms_norm_quant(x, gamma, residual=res)
        logits = a.quant_linear(q, s, w, ones[:e], out_dtype=torch.float32)
        r = a.moe_route(logits, k)
        rows, rs = a.moe_dispatch(q, s, r.slots, r.tokens)
        y = a.quant_linear(act, ones[:t], wide, ones[:hidden], residual=h, out_dtype=torch.float16)
        z = (rows.float() * rs[:, None]).half()
        out = a.moe_combine(z, r.slots, r.weights, residual=y)
        dw, dz = a.moe_combine_grad(dout, z, r.slots, r.tokens, r.weights)
        dl = a.moe_route_grad(logits, r.weights, r.experts, r.counts, r.routed, grad_weights=dw, grad_loss=ones[:1].clone())
        return [q, s, h, logits, *r, rows, rs, y, out, dw, dz, dl]

    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        step()
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for i in range(4):
        x.copy_(rnd(t, hidden).half())
        res.copy_(rnd(t, hidden).half())
        want = [v.clone() for v in step()]
        torch.cuda.synchronize()
        for v in kept:
            v.view(torch.uint8).fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        for n, (got, ref) in enumerate(zip(kept, want)):
            assert torch.equal(got.view(torch.uint8), ref.view(torch.uint8)), (i, n)


def test_streams_side_by_side(ascq_gpu):
    """calls of several streams at a time, each with workspaces of its own, equal the same calls alone"""
    a = ascq_gpu
    g = torch.Generator(device="cuda").manual_seed(5)
    cases = []
    for n in range(3):
        x = (torch.randn(48 + n, 8192, generator=g, device="cuda") * 30).clamp(-127, 127).to(torch.int8)
        w = (torch.randn(640, 8192, generator=g, device="cuda") * 30).clamp(-127, 127).to(torch.int8)
        logits = torch.randn(3000 + n, 64, generator=g, device="cuda")
        cases.append((x, torch.rand(48 + n, device="cuda"), w, torch.rand(640, device="cuda"), logits))
    run = lambda c: (a.quant_linear(c[0], c[1], c[2], c[3], out_dtype=torch.float32), *a.moe_route(c[4], 6))  # noqa: E731
    alone = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for st, c in zip(streams, cases):
            with torch.cuda.stream(st):
                got.append(run(c))
        torch.cuda.synchronize()
        for one, ref in zip(got, alone):
            assert all(torch.equal(p, q) for p, q in zip(one, ref))


def test_long_offsets(ascq_gpu):
    """rows beyond 2^31 elements, and weights beyond 2^31 bytes"""
    a = ascq_gpu
    m, n = 270000, 8192
    x = torch.zeros(m, n, dtype=torch.int8, device="cuda")
    x[m - 1] = torch.arange(n, device="cuda").remainder(200).sub(100).to(torch.int8)
    s = torch.ones(m, device="cuda")
    slots = torch.arange(m, device="cuda", dtype=torch.int32).flip(0)[:, None].contiguous()
    rows, _ = a.moe_dispatch(x, s, slots, slots.flatten())
    assert torch.equal(rows[0], x[m - 1]) and rows[1:100].abs().sum() == 0
    # a linear over the same rows: more than 2^31 bytes of x
    w = torch.ones(16, n, dtype=torch.int8, device="cuda")
    y = a.quant_linear(x, s, w, torch.ones(16, device="cuda"), out_dtype=torch.float32)
    assert torch.all(y[m - 1] == float(x[m - 1].int().sum())) and torch.all(y[: m - 1] == 0)
    del rows, x
    # more than 2^31 bytes of w: pieces of channels, the last of them one channel
    k = 16384
    piece = ((1 << 31) - 16) // k // 256 * 256
    w = torch.ones(piece + 1, k, dtype=torch.int8, device="cuda")
    w[piece - 1, 0], w[piece, k - 1] = 5, -7
    x = torch.ones(3, k, dtype=torch.int8, device="cuda")
    ones = torch.ones(piece + 1, device="cuda")
    y = a.quant_linear(x, ones[:3], w, ones, bias=ones, out_dtype=torch.float32)
    want = torch.full((piece + 1,), float(k + 1), device="cuda")
    want[piece - 1] += 4
    want[piece] -= 8
    assert torch.equal(y, want.expand(3, -1))
    del w, y
    h = torch.zeros(m, n, dtype=torch.float16, device="cuda")
    h[m - 1] = 2.0
    q, sc, _ = a.add_rms_norm_quant(h, torch.ones(n, dtype=torch.float16, device="cuda"))
    assert torch.all(q[m - 1] == 127) and torch.all(q[: m - 1] == 0)
    assert math.isclose(sc[m - 1].item() * 127, 1.0, rel_tol=1e-5)
