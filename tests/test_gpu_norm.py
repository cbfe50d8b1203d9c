"""Residual addition + RMS norm + 8-bit output (ascq_add_rms_norm_quant) against the definition in 64 bits.

Tolerances.  t = h gamma, a, and the code's argument v = t (Q (1 / a)) take five fp32 roundings, so v is within 5 x 2^-24 |v|
of the 64-bit one: a code is the nearest code to some value that close.  The scale a rstd / Q: the sum of n squares is added up in
at most n / 256 + 16 steps (half of its relative error reaches rstd), and five more roundings.  The stored sum h is the
16-bit rounding of an fp32 sum, which is the correctly rounded one (24 bits >= 2 x 11 + 2)."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
ULP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}  # half an ulp, relative
EPS = 1e-5


def _e4m3_distance(v: torch.Tensor) -> torch.Tensor:
    """distance of v (within +-448) from the nearest e4m3 value: the format's step at |v| is 2^(max(e, -6) - 3)"""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -20))).clamp_min(-6)
    step = torch.exp2(e - 3)
    return (v - torch.round(v / step) * step).abs()


def _check(x, gamma, residual, codes, q, scale, h, norm=None, eps=EPS):
    """all on the CPU"""
    name = {v: k for k, v in DT.items()}[x.dtype]
    n = x.shape[1]
    want_h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    assert torch.equal(h, want_h)
    big = 127.0 if codes == "int8" else 448.0
    t = want_h.double() * gamma.double()
    a = t.abs().amax(dim=1)
    # (a row of zeros has scale 0 by definition, with eps 0 too)
    rstd = torch.where(a > 0, 1 / torch.sqrt((want_h.double() ** 2).mean(dim=1) + eps), 0.0)
    want_s = a * rstd / big
    bound = (n / 256 + 32) * 2.0 ** -24
    assert torch.all((scale.double() - want_s).abs() <= bound * want_s + 2.0 ** -149)
    live = a > 0
    v = torch.where(live[:, None], t * (big / a.clamp_min(1e-300))[:, None], torch.zeros_like(t))
    got = q.float().double()
    slack = 5 * 2.0 ** -24 * v.abs()
    if codes == "int8":
        assert torch.all((got - v).abs() <= 0.5 + slack)
    else:
        assert torch.all((got - v).abs() <= _e4m3_distance(v) + 2 * slack)
    if norm is not None:
        want = t * rstd[:, None]
        assert torch.all((norm.double() - want).abs() <= (ULP[name] + bound + 2.0 ** -22) * want.abs() + 2.0 ** -25)


def _data(m, n, dt, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, n + pad, generator=g).to(DT[dt])[:, :n]
    r = (torch.randn(m, n, generator=g) * 3).to(DT[dt])
    gamma = (torch.rand(n, generator=g) + 0.5).to(DT[dt])
    return x, r, gamma


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("m,n", [(1, 1), (3, 7), (2, 8), (5, 63), (1, 64), (65, 512), (4, 1000), (1, 4096), (3, 4097), (2, 5120),
                                 (9, 8192), (2, 11008), (2, 16384), (3, 16392), (2, 20001), (1, 70000)])
def test_matches_64_bits(ascq_gpu, m, n, dt, codes):
    x, r, gamma = _data(m, n, dt, m * 7 + n)
    code = ascq_gpu.INT8 if codes == "int8" else ascq_gpu.FP8_E4M3
    for residual in (r, None):
        norm = torch.empty(m, n, dtype=DT[dt], device="cuda")
        q, s, h = ascq_gpu.add_rms_norm_quant(x.cuda(), gamma.cuda(), EPS, code,
                                              residual=None if residual is None else residual.cuda(), norm_out=norm)
        assert q.dtype == (torch.int8 if codes == "int8" else torch.float8_e4m3fn)
        _check(x, gamma, residual, codes, q.cpu(), s.cpu(), h.cpu(), norm.cpu())


@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("n,pad,shift", [(512, 8, 0), (512, 3, 0), (512, 64, 1), (1000, 24, 8), (129, 7, 1), (4096, 4096, 0)])
def test_strides_and_alignment(ascq_gpu, n, pad, shift, dt):
    """rows inside a wider buffer, at element offsets off 16 bytes, h and residual with other pitches than x"""
    m = 6
    x, r, gamma = _data(m, n, dt, n + pad + shift)
    def wide(t, p):  # noqa: E306
        b = torch.full((m * (n + p) + shift + 16,), 7.0, dtype=DT[dt], device="cuda")
        v = b[shift:shift + m * (n + p)].view(m, n + p)[:, :n]
        v.copy_(t)
        return b, v
    bx, vx = wide(x, pad)
    br, vr = wide(r, pad + 5)
    bh, vh = wide(torch.zeros(m, n), pad + 9)
    before = bh.clone()
    q, s, h = ascq_gpu.add_rms_norm_quant(vx, gamma.cuda(), EPS, residual=vr, residual_out=vh)
    assert h is vh
    _check(x, gamma, r, "int8", q.cpu(), s.cpu(), vh.cpu())
    untouched = torch.ones_like(bh, dtype=torch.bool)
    untouched[shift:shift + m * (n + pad + 9)].view(m, n + pad + 9)[:, :n] = False
    assert torch.equal(bh[untouched], before[untouched])


@pytest.mark.parametrize("n", [8, 72, 257, 1000, 3001, 4096, 5120, 11008, 20000, 30000, 66000])
@pytest.mark.parametrize("into", ["x", "residual"])
def test_in_place(ascq_gpu, n, into):
    """threads whose share of a row is not whole read its last elements too: they must not count once they are stored over"""
    x, r, gamma = _data(40, n, "bf16", n)
    r[:, -8:] *= 30  # (the last elements' second sum would be the largest)
    gx, gr = x.cuda(), r.cuda()
    q, s, h = ascq_gpu.add_rms_norm_quant(gx, gamma.cuda(), EPS, residual=gr, residual_out=gx if into == "x" else gr)
    _check(x, gamma, r, "int8", q.cpu(), s.cpu(), h.cpu())
    assert torch.equal((gr if into == "x" else gx).cpu(), r if into == "x" else x)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("n", [96, 513, 4096])
def test_rows_without_an_answer(ascq_gpu, n, dt, codes):
    """zero rows: codes and scale 0 (eps 0 too); NaN, infinity, or squares past fp32: codes 0, scale and norm NaN; the other
    rows are not touched by them"""
    x, _, gamma = _data(8, n, dt, 5)
    x[0] = 0
    x[1, n // 2] = math.nan
    x[2, n - 1] = math.inf
    x[3, 0] = -math.inf
    if dt != "f16":
        x[4] = 3e19
        x[4, 3] = -1e30
    code = ascq_gpu.INT8 if codes == "int8" else ascq_gpu.FP8_E4M3
    for eps in (EPS, 0.0):
        norm = torch.empty_like(x, device="cuda")
        q, s, _ = ascq_gpu.add_rms_norm_quant(x.cuda(), gamma.cuda(), eps, code, norm_out=norm)
        q, s, norm = q.float().cpu(), s.cpu(), norm.cpu()
        bad = [1, 2, 3] + ([4] if dt != "f16" else [])
        good = [i for i in range(8) if i not in bad]
        assert torch.all(q[bad] == 0) and torch.all(torch.isnan(s[bad])) and torch.all(torch.isnan(norm[bad]))
        assert torch.all(q[0] == 0) and s[0] == 0 and torch.all(norm[0] == 0)
        _check(x[good], gamma, None, codes, q[good], s[good], x[good], norm[good], eps)


def test_saturation_of_the_sum(ascq_gpu):
    """a residual sum past f16 saturates to 65504, as every f16 conversion here does"""
    x = torch.full((2, 64), 60000.0, dtype=torch.float16)
    q, s, h = ascq_gpu.add_rms_norm_quant(x.cuda(), torch.ones(64, dtype=torch.float16, device="cuda"), residual=x.cuda())
    assert torch.all(h == 65504) and torch.all(q == 127)
    assert torch.allclose(s.cpu(), torch.full((2,), 1 / 127), rtol=1e-6)


def test_large_channels_and_tiny_rows(ascq_gpu):
    """gamma with a zero and large channels; rows down to fp32's subnormals keep codes within +-127"""
    x, r, gamma = _data(6, 640, "f32", 3)
    gamma[5] = 0
    gamma[77] = 300.0
    x[1] *= 1e-20
    x[2] *= 1e-36
    r.zero_()
    q, s, h = ascq_gpu.add_rms_norm_quant(x.cuda(), gamma.cuda(), EPS, residual=r.cuda())
    keep = [0, 1, 3, 4, 5]
    _check(x[keep], gamma, r[keep], "int8", q.cpu()[keep], s.cpu()[keep], h.cpu()[keep])
    assert torch.isfinite(s).all() and q.abs().max() <= 127


def test_on_another_stream(ascq_gpu):
    x, r, gamma = _data(33, 4096, "f16", 9)
    gx, gr, gg = x.cuda(), r.cuda(), gamma.cuda()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    q, s, h = ascq_gpu.add_rms_norm_quant(gx, gg, EPS, residual=gr, stream=st)
    st.synchronize()
    _check(x, gamma, r, "int8", q.cpu(), s.cpu(), h.cpu())


def test_no_rows(ascq_gpu):
    x = torch.empty(0, 64, dtype=torch.float16, device="cuda")
    q, s, h = ascq_gpu.add_rms_norm_quant(x, torch.ones(64, dtype=torch.float16, device="cuda"))
    assert q.shape == (0, 64) and s.shape == (0,)
