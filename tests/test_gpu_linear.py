"""The quantised linear (ascq_quant_linear) against the definition in 64 bits.

Tolerances.  int8 sums are exact.  z = sum w_scale x_scale + bias takes four fp32 roundings, the activation's slope is at
most 1.13 and its own error at most 1e-6 |z| (fp32 exponential, reciprocal, and the erfc polynomial's 1.5e-7), the
residual's addition one rounding more, and the output type's rounding half an ulp.  fp8: operands of -2, -1.5 .. 2 have
products on a grid of 2^-2 up to 4, whose sums are exact, so they get the same bound (index mistakes show); for
normal data the matrix unit drops what lies 2^-13 below the largest product of 16."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
ULP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
ACTS = ["none", "faster_gelu", "relu", "gelu", "silu"]


def _codes(g, shape, kind):
    if kind == "int8":
        return torch.randint(-127, 128, shape, generator=g, dtype=torch.int8)
    if kind == "fp8":  # exact sums
        return (torch.randint(-4, 5, shape, generator=g).float() / 2).to(torch.float8_e4m3fn)
    return torch.randn(shape, generator=g).to(torch.float8_e4m3fn)  # fp8_normal


def _make(m, n, k, kind, out, seed, bias=True, residual=True, w_trans=True):
    g = torch.Generator().manual_seed(seed)
    unit = {"int8": 73.0, "fp8": 1.3, "fp8_normal": 1.0}[kind]
    d = dict(x=_codes(g, (m, k), kind), w=_codes(g, (n, k) if w_trans else (k, n), kind),
             x_scale=(torch.rand(m, generator=g) + 0.5) / unit,
             w_scale=(torch.rand(n, generator=g) + 0.5) / (unit * math.sqrt(max(k, 1))),
             bias=torch.randn(n, generator=g) if bias else None,
             residual=torch.randn(m, n, generator=g).to(DT[out]) if residual else None)
    return d


def _exact(d, act, w_trans):
    w = d["w"].float().double()
    s = d["x"].float().double() @ (w.t() if w_trans else w) * d["w_scale"].double() * d["x_scale"].double()[:, None]
    z = s if d["bias"] is None else s + d["bias"].double()
    a = z
    if act == "relu":
        a = z.clamp_min(0)
    elif act == "gelu":
        a = z * torch.special.ndtr(z)
    elif act in ("silu", "faster_gelu"):
        a = z * torch.sigmoid(z * (1 if act == "silu" else 1.702))
    y = a if d["residual"] is None else a + d["residual"].double()
    size = s.abs() + (0 if d["bias"] is None else d["bias"].double().abs())
    return y, size


def _sum_slack(d, kind, w_trans):
    """what the fp8 matrix unit may drop: 2^-13 of the largest product of a group of 16, per product; groups lie within
    128 consecutive k"""
    if kind != "fp8_normal":
        return 0.0
    x, w = d["x"].float().abs(), d["w"].float().abs()
    w = w if w_trans else w.t()
    pad = -x.shape[1] % 128
    top = lambda t: torch.nn.functional.pad(t, (0, pad)).view(t.shape[0], -1, 128).amax(dim=2).double()  # noqa: E731
    return (top(x) @ top(w).t()) * 128 * 2.0 ** -13 * d["w_scale"].double() * d["x_scale"].double()[:, None]


def _compare(got, d, act, out, kind, w_trans):
    want, size = _exact(d, act, w_trans)
    r = 0 if d["residual"] is None else d["residual"].double().abs()
    bound = ULP[out] * want.abs() + 1.13 * (6 * 2.0 ** -24 * size + _sum_slack(d, kind, w_trans)) + 1e-6 * size \
        + 2.0 ** -24 * (size + r) + 2.0 ** -25
    off = (got.double() - want).abs() - bound
    assert torch.all(off <= 0), f"worst {off.max().item():.3g} past the bound"


def _gpu(d):
    return {k: None if v is None else v.cuda() for k, v in d.items()}


def _run(a, d, act, out, w_trans, **kw):
    g = _gpu(d)
    code = dict(zip(ACTS, (a.ACT_NONE, a.ACT_FASTER_GELU, a.ACT_RELU, a.ACT_GELU, a.ACT_SILU)))[act]
    return a.quant_linear(g["x"], g["x_scale"], g["w"], g["w_scale"], bias=g["bias"], activation=code,
                          residual=g["residual"], w_trans=w_trans, out_dtype=DT[out], **kw)


SHAPES = [(1, 1, 1), (1, 16, 64), (2, 5, 17), (1, 4096, 256), (16, 512, 1024), (17, 100, 96), (32, 4096, 512), (33, 260, 1024),
          (64, 1000, 2048), (64, 64, 8192), (65, 384, 256), (129, 257, 272), (200, 512, 128), (256, 768, 640), (300, 4100, 144),
          (1000, 520, 1040), (7, 12, 0), (3, 33, 4095), (130, 129, 1001), (1030, 516, 515)]


@pytest.mark.parametrize("w_trans", [True, False])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_shapes(ascq_gpu, m, n, k, kind, w_trans):
    """from one row to large tiles, odd sizes, k = 0"""
    i = SHAPES.index((m, n, k)) + 2 * (kind == "fp8") + w_trans
    act, out = ACTS[i % 5], ("f16", "bf16", "f32")[i % 3]
    d = _make(m, n, k, kind, out, i, w_trans=w_trans, bias=i % 4 != 0, residual=i % 3 != 1)
    _compare(_run(ascq_gpu, d, act, out, w_trans).cpu(), d, act, out, kind, w_trans)


@pytest.mark.parametrize("m,n,k", [(4, 320, 512), (150, 192, 256)])
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("kind", ["int8", "fp8", "fp8_normal"])
def test_epilogues(ascq_gpu, kind, act, out, m, n, k):
    for bias in (True, False):
        for residual in (True, False):
            d = _make(m, n, k, kind, out, 11, bias=bias, residual=residual)
            _compare(_run(ascq_gpu, d, act, out, True).cpu(), d, act, out, kind, True)


@pytest.mark.parametrize("m,n,k", [(256, 256, 256), (512, 768, 512), (1024, 2048, 256), (2048, 1024, 384), (2304, 2304, 128),
                                   (384, 4096, 272), (4096, 1536, 160), (700, 11008, 128), (2048, 8192, 512)])
@pytest.mark.parametrize("w_trans", [True, False])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_every_tile(ascq_gpu, kind, w_trans, m, n, k):
    """sizes that spread over the tile shapes, with a last tile row and column that are not full"""
    m, n = m - 3, n - 4
    out = "bf16" if kind == "fp8" else "f16"
    d = _make(m, n, k, kind, out, m + n, w_trans=w_trans)
    want_gpu = {key: None if v is None else v.cuda() for key, v in d.items()}
    got = _run(ascq_gpu, d, "silu", out, w_trans)
    # (the 64-bit product on the GPU: it only checks)
    w = want_gpu["w"].float().double()
    z = want_gpu["x"].float().double() @ (w.t().contiguous() if w_trans else w)
    z = z * want_gpu["w_scale"].double() * want_gpu["x_scale"].double()[:, None]
    size = z.abs() + want_gpu["bias"].double().abs()
    z = z + want_gpu["bias"].double()
    want = z * torch.sigmoid(z) + want_gpu["residual"].double()
    bound = ULP[out] * want.abs() + 9e-7 * size + 1e-6 * size + 2.0 ** -24 * want_gpu["residual"].double().abs() + 2.0 ** -25
    assert torch.all((got.double() - want).abs() <= bound)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("w_trans", [True, False])
@pytest.mark.parametrize("m,n,k,shift,pad", [(5, 96, 256, 0, 16), (5, 96, 256, 1, 3), (130, 200, 320, 4, 12), (130, 200, 321, 0, 15),
                                             (40, 128, 512, 8, 64), (257, 260, 1000, 3, 1)])
def test_strides_and_alignment(ascq_gpu, m, n, k, shift, pad, w_trans, kind):
    """operands, residual and output inside wider buffers, off 16 bytes; what lies around the output stays"""
    d = _make(m, n, k, kind, "f16", m + shift, w_trans=w_trans)
    g = _gpu(d)
    def wide(t, p, fill):  # noqa: E306
        rows, cols = t.shape
        b = torch.full((rows * (cols + p) + shift + 64,), fill, dtype=torch.float32, device="cuda").to(t.dtype)
        v = b[shift:shift + rows * (cols + p)].view(rows, cols + p)[:, :cols]
        v.copy_(t)
        return b, v
    _, x = wide(g["x"], pad, 3.0)
    _, w = wide(g["w"], pad + 1, 3.0)
    _, r = wide(g["residual"], pad, 9.0)
    by, y = wide(torch.zeros(m, n, dtype=torch.float16, device="cuda"), pad + 2, 5.0)
    before = by.clone()
    got = ascq_gpu.quant_linear(x, g["x_scale"], w, g["w_scale"], bias=g["bias"], residual=r, w_trans=w_trans, out=y)
    assert got is y
    _compare(y.cpu(), d, "none", "f16", kind, w_trans)
    untouched = torch.ones_like(by, dtype=torch.bool)
    untouched[shift:shift + m * (n + pad + 2)].view(m, n + pad + 2)[:, :n] = False
    assert torch.equal(by[untouched], before[untouched])


@pytest.mark.parametrize("m,n,k", [(3, 512, 1024), (64, 4096, 8192), (200, 300, 256), (1025, 768, 512)])
def test_into_the_residual(ascq_gpu, m, n, k):
    d = _make(m, n, k, "int8", "bf16", 3)
    g = _gpu(d)
    got = ascq_gpu.quant_linear(g["x"], g["x_scale"], g["w"], g["w_scale"], bias=g["bias"], residual=g["residual"],
                                out=g["residual"])
    _compare(got.cpu(), d, "none", "bf16", "int8", True)


@pytest.mark.parametrize("w_trans", [True, False])
@pytest.mark.parametrize("m,n,k", [(1, 4096, 8192), (16, 4096, 11008), (64, 2048, 8192), (5, 640, 1001), (130, 320, 777)])
def test_with_and_without_a_workspace(ascq_gpu, m, n, k, w_trans):
    """int8: the same bits with the workspace asked for, with less of it, and with none"""
    d = _make(m, n, k, "int8", "f32", 17, w_trans=w_trans)
    g = _gpu(d)
    need = ascq_gpu.quant_linear_workspace_size(g["x"], g["w"], w_trans, torch.float32)
    call = lambda ws: ascq_gpu.quant_linear(g["x"], g["x_scale"], g["w"], g["w_scale"], bias=g["bias"],  # noqa: E731
                                            residual=g["residual"], w_trans=w_trans, out_dtype=torch.float32, workspace=ws)
    full = call(torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda"))
    _compare(full.cpu(), d, "none", "f32", "int8", w_trans)
    for ws in (torch.empty(max(need - 256, 1), dtype=torch.uint8, device="cuda"), torch.empty(1, dtype=torch.uint8, device="cuda"),
               torch.empty(need + 64, dtype=torch.uint8, device="cuda")[1:]):
        assert torch.equal(call(ws), full)
    assert torch.equal(call(None), full)


def test_extreme_values(ascq_gpu):
    """int8 sums at the edge of int32's half, scales that overflow the output (saturated), NaN and infinite scales"""
    k = 65536
    x = torch.full((2, k), -128, dtype=torch.int8)
    w = torch.full((64, k), -128, dtype=torch.int8)
    one = torch.ones(64)
    y = ascq_gpu.quant_linear(x.cuda(), torch.ones(2).cuda(), w.cuda(), one.cuda(), out_dtype=torch.float32)
    assert torch.all(y == float(k * 128 * 128))
    y = ascq_gpu.quant_linear(x.cuda(), torch.tensor([1.0, math.nan]).cuda(), w.cuda(), one.cuda(), out_dtype=torch.float16)
    assert torch.all(y[0] == 65504) and torch.all(torch.isnan(y[1]))
    y = ascq_gpu.quant_linear(x.cuda(), torch.tensor([1e30, -1e30]).cuda(), w.cuda(), one.cuda(), out_dtype=torch.float32,
                              activation=ascq_gpu.ACT_GELU)
    assert torch.all(y[0] > 1e38) and torch.all(y[1] == 0)
    for act in (ascq_gpu.ACT_SILU, ascq_gpu.ACT_GELU, ascq_gpu.ACT_RELU):
        y = ascq_gpu.quant_linear(x.cuda(), torch.tensor([1e35, -1e35]).cuda(), w.cuda(), one.cuda(), out_dtype=torch.float32,
                                  activation=act)
        assert torch.all(torch.isinf(y[0])) and torch.all(y[1] == 0)


@pytest.mark.parametrize("m", [4, 300])
def test_e4m3_nan(ascq_gpu, m):
    """a NaN code reaches its row (of x) or column (of w) and nothing else; none beyond k reaches anything"""
    n, k = 96, 200
    d = _make(m, n, k, "fp8", "f32", 2, residual=False)
    wide = torch.full((m, 256), 127, dtype=torch.uint8).view(torch.float8_e4m3fn)  # NaN behind k
    xb = wide.clone().view(torch.uint8)
    xb[:, :k] = d["x"].view(torch.uint8)
    xb[1, 7] = 127
    x = xb.cuda().view(torch.float8_e4m3fn)[:, :k]
    y = ascq_gpu.quant_linear(x, d["x_scale"].cuda(), d["w"].cuda(), d["w_scale"].cuda(), bias=d["bias"].cuda(),
                              out_dtype=torch.float32).cpu()
    rows = torch.isnan(y)
    assert torch.all(rows[1]) and not rows[[i for i in range(m) if i != 1]].any()


def test_on_another_stream(ascq_gpu):
    """operands made on the stream of the call; the call's own workspace included"""
    d = _make(16, 4096, 8192, "int8", "f16", 5)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        y = _run(ascq_gpu, d, "none", "f16", True)
    st.synchronize()
    _compare(y.cpu(), d, "none", "f16", "int8", True)
    g = _gpu(d)
    torch.cuda.synchronize()
    y = ascq_gpu.quant_linear(g["x"], g["x_scale"], g["w"], g["w_scale"], bias=g["bias"], residual=g["residual"],
                              out_dtype=torch.float16, stream=st)
    st.synchronize()
    _compare(y.cpu(), d, "none", "f16", "int8", True)


@pytest.mark.parametrize("shape", [(0, 64, 128), (4, 0, 128)])
def test_nothing_to_do(ascq_gpu, shape):
    m, n, k = shape
    y = ascq_gpu.quant_linear(torch.zeros(m, k, dtype=torch.int8, device="cuda"), torch.zeros(m, device="cuda"),
                              torch.zeros(n, k, dtype=torch.int8, device="cuda"), torch.zeros(n, device="cuda"))
    assert y.shape == (m, n)
