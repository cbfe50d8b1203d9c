"""Refusals of the block operators (norm, linear, routing, rows): bad arguments give a negative status and a message, and
launch nothing -- no GPU needed.  The Python binding refuses tensors of the wrong shape, type, layout or device."""
from __future__ import annotations

import ctypes

import pytest
import torch

import ascq

D = ctypes.c_void_p(0x1000)
ODD = ctypes.c_void_p(0x1001)


def _err(status, expect, text=""):
    assert status == expect, f"status {status}: {ascq.last_error()}"
    assert text in ascq.last_error()


def test_norm_arguments():
    def call(q=D, s=D, h=None, norm=None, x=D, r=None, g=D, m=4, n=64, ldx=0, ldr=0, ldh=0, src=ascq.F16, dst=ascq.INT8,
             eps=1e-6):
        p = ascq._NormQuantParam(m, n, ldx, ldr, ldh, src, dst, eps)
        return ascq.lib().ascq_add_rms_norm_quant(q, s, h, norm, x, r, g, ctypes.byref(p), None)

    _err(ascq.lib().ascq_add_rms_norm_quant(D, D, None, None, D, None, D, None, None), ascq.E_INVALID_ARG, "null params")
    _err(call(src=ascq.INT8), ascq.E_UNSUPPORTED)
    _err(call(dst=ascq.FP8_E5M2), ascq.E_UNSUPPORTED)
    for bad in (dict(m=-1), dict(n=-1), dict(ldx=63), dict(r=D, ldr=32), dict(r=D, h=D, ldh=1), dict(h=D), dict(q=None),
                dict(s=None), dict(x=None), dict(g=None), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
                dict(x=ODD), dict(g=ODD), dict(r=ODD), dict(norm=ODD), dict(s=ODD), dict(r=D, h=D, ldr=64, ldh=72),
                dict(x=ctypes.c_void_p(0x1002), src=ascq.F32)):
        _err(call(**bad), ascq.E_INVALID_ARG)
    _err(call(m=1 << 31), ascq.E_UNSUPPORTED)
    _err(call(m=1 << 30, ldx=1 << 40), ascq.E_UNSUPPORTED)
    _err(call(m=0, q=None, x=None), ascq.OK)
    _err(call(n=0, q=None, x=None), ascq.OK)


def test_linear_arguments():
    def call(y=D, x=D, xs=D, w=D, ws=D, b=None, r=None, m=4, n=64, k=128, ldx=0, ldw=0, ldr=0, ldy=0, code=ascq.INT8,
             out=ascq.F16, trans=1, act=0, size=False):
        p = ascq._LinearParam(m, n, k, ldx, ldw, ldr, ldy, code, out, trans, act)
        if size:
            need = ctypes.c_size_t(0)
            return ascq.lib().ascq_quant_linear_workspace_size(x, w, ctypes.byref(p), ctypes.byref(need))
        return ascq.lib().ascq_quant_linear(y, x, xs, w, ws, b, r, ctypes.byref(p), None, 0, None)

    _err(ascq.lib().ascq_quant_linear(D, D, D, D, D, None, None, None, None, 0, None), ascq.E_INVALID_ARG, "null params")
    for size in (False, True):
        _err(call(code=ascq.INT4, size=size), ascq.E_UNSUPPORTED)
        _err(call(code=ascq.FP8_E5M2, size=size), ascq.E_UNSUPPORTED)
        _err(call(out=ascq.INT8, size=size), ascq.E_UNSUPPORTED)
        for bad in (dict(trans=2), dict(act=5), dict(act=-1), dict(m=-1), dict(n=-1), dict(k=-1), dict(ldx=127), dict(ldw=127),
                    dict(trans=0, ldw=63), dict(ldr=63), dict(ldy=63)):
            _err(call(size=size, **bad), ascq.E_INVALID_ARG)
        _err(call(k=1 << 17, size=size), ascq.E_UNSUPPORTED, "int32")
        _err(call(m=1 << 31, size=size), ascq.E_UNSUPPORTED)
        _err(call(m=1 << 30, n=1 << 30, size=size), ascq.E_UNSUPPORTED)
    for bad in (dict(y=None), dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(y=ODD), dict(r=ODD), dict(xs=ODD),
                dict(ws=ODD), dict(b=ODD), dict(r=D, ldr=72)):
        _err(call(**bad), ascq.E_INVALID_ARG)
    _err(call(m=0, y=None, x=None), ascq.OK)
    _err(call(n=0, y=None, w=None), ascq.OK)
    _err(ascq.lib().ascq_quant_linear_workspace_size(D, D, None, None), ascq.E_INVALID_ARG)


def test_route_arguments():
    L = ascq.lib()

    def param(t=128, e=16, ld=0, ty=ascq.F32, k=2):
        return ascq._RouteParam(t, e, ld, ty, k, 1)

    def call(*ptrs, ws=D, room=1 << 20, **kw):
        ptrs = list(ptrs) or [D] * 8
        return L.ascq_moe_route(*ptrs, ctypes.byref(param(**kw)), ws, room, None)

    for bad in (dict(t=-1), dict(e=0), dict(k=0), dict(k=17, e=64), dict(k=5, e=4), dict(ld=15)):
        _err(call(**bad), ascq.E_INVALID_ARG)
    _err(call(ty=ascq.INT8), ascq.E_UNSUPPORTED)
    _err(call(e=1025), ascq.E_UNSUPPORTED)
    _err(call(t=1 << 30), ascq.E_UNSUPPORTED)
    for i in range(8):
        _err(call(*[None if j == i else D for j in range(8)]), ascq.E_INVALID_ARG, "null")
        _err(call(*[ODD if j == i else D for j in range(8)]), ascq.E_INVALID_ARG, "aligned")
    need = ctypes.c_size_t(0)
    _err(L.ascq_moe_route_workspace_size(ctypes.byref(param(t=5000)), ctypes.byref(need)), ascq.OK)
    assert need.value > 0
    _err(call(t=5000, room=need.value - 1), ascq.E_INVALID_ARG, "workspace")
    _err(call(t=5000, ws=None), ascq.E_INVALID_ARG, "workspace")
    _err(call(t=5000, ws=ctypes.c_void_p(0x1008)), ascq.E_INVALID_ARG, "workspace")
    _err(L.ascq_moe_route_workspace_size(ctypes.byref(param()), None), ascq.E_INVALID_ARG)

    def grad(g=D, ldg=0, x=D, w=D, e=D, c=D, n=D, dw=D, dl=D, **kw):
        return L.ascq_moe_route_grad(g, ldg, x, w, e, c, n, dw, dl, ctypes.byref(param(**kw)), None)

    for bad in (dict(g=None), dict(x=None), dict(w=None), dict(e=None), dict(c=None), dict(n=None), dict(ldg=15), dict(g=ODD),
                dict(dw=ODD), dict(dl=ODD), dict(k=0), dict(ldg=20)):
        _err(grad(**bad), ascq.E_INVALID_ARG)
    _err(grad(t=0, g=None, x=None), ascq.OK)


def test_rows_arguments():
    L = ascq.lib()

    def param(t=8, n=64, ld=0, ty=ascq.F16, k=2):
        return ctypes.byref(ascq._RowsParam(t, n, ld, ty, k))

    def dispatch(rows=D, rs=D, x=D, xs=D, slots=D, tokens=D, **kw):
        return L.ascq_moe_dispatch(rows, rs, x, xs, slots, tokens, param(**kw), None)

    def combine(out=D, y=D, slots=D, w=D, r=None, **kw):
        return L.ascq_moe_combine(out, y, slots, w, r, param(**kw), None)

    def grad(dw=D, dy=D, g=D, y=D, slots=D, tokens=D, w=D, **kw):
        return L.ascq_moe_combine_grad(dw, dy, g, y, slots, tokens, w, param(**kw), None)

    for f in (dispatch, combine, grad):
        for bad in (dict(t=-1), dict(n=-1), dict(k=0), dict(k=17), dict(slots=None), dict(slots=ODD)):
            _err(f(**bad), ascq.E_INVALID_ARG)
        _err(f(ty=ascq.INT32), ascq.E_UNSUPPORTED)
        _err(f(t=1 << 30), ascq.E_UNSUPPORTED)
        _err(f(t=0), ascq.OK)
    _err(combine(ty=ascq.INT8), ascq.E_UNSUPPORTED)
    _err(grad(ty=ascq.FP8_E4M3), ascq.E_UNSUPPORTED)
    for bad in (dict(rs=None), dict(xs=None), dict(rows=None), dict(x=None), dict(tokens=None), dict(ld=63), dict(x=ODD),
                dict(rows=ODD)):
        _err(dispatch(**bad), ascq.E_INVALID_ARG)
    for bad in (dict(out=None), dict(y=None), dict(w=None), dict(r=ODD), dict(out=ODD)):
        _err(combine(**bad), ascq.E_INVALID_ARG)
    for bad in (dict(g=None), dict(y=None), dict(tokens=None), dict(w=None), dict(dy=ODD), dict(dw=ODD)):
        _err(grad(**bad), ascq.E_INVALID_ARG)
    _err(grad(dw=None, dy=None), ascq.OK)


def _refused(f, *args, status=ascq.E_INVALID_ARG, **kw):
    with pytest.raises(ascq.AscqError) as e:
        f(*args, **kw)
    assert e.value.status == status


def test_binding_refusals():
    h = torch.zeros(4, 64, dtype=torch.float16)
    g = torch.ones(64, dtype=torch.float16)
    norm = ascq.add_rms_norm_quant
    _refused(norm, h, g)  # CPU tensors
    _refused(norm, h, g[:32])
    _refused(norm, h, g.float())
    _refused(norm, h.t(), g[:4])
    _refused(norm, h[:, ::2], g[:32])
    _refused(norm, h, g, residual=h[:3])
    _refused(norm, h, g, residual=h.float())
    _refused(norm, h, g, residual_out=h)
    _refused(norm, h[0], g)
    _refused(norm, h.int(), g, status=ascq.E_UNSUPPORTED)
    _refused(norm, h, g, dst_type=ascq.INT4, status=ascq.E_UNSUPPORTED)
    _refused(norm, h, g, out=torch.zeros(4, 64, dtype=torch.uint8))
    x, w = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(32, 64, dtype=torch.int8)
    xs, ws = torch.ones(4), torch.ones(32)
    lin = ascq.quant_linear
    _refused(lin, x, xs, w, ws)  # CPU tensors
    _refused(lin, x, xs[:3], w, ws)
    _refused(lin, x, xs.half(), w, ws)
    _refused(lin, x, xs, w, ws[:31])
    _refused(lin, x, xs, w, ws, bias=ws.half())
    _refused(lin, x, xs, w, ws, bias=ws[:8])
    _refused(lin, x, xs, w[:, :32], ws)
    _refused(lin, x, xs, w.t(), ws, w_trans=False)
    _refused(lin, x, xs, w, ws, residual=torch.zeros(4, 32))  # out is bf16
    _refused(lin, x, xs, w.view(torch.float8_e4m3fn), ws)
    _refused(lin, x.short(), xs, w, ws, status=ascq.E_UNSUPPORTED)
    _refused(lin, x, xs, w, ws, out_dtype=torch.int32, status=ascq.E_UNSUPPORTED)
    logits = torch.zeros(4, 8)
    _refused(ascq.moe_route, logits, 2)  # CPU tensors
    _refused(ascq.moe_route, logits, 9)
    _refused(ascq.moe_route, logits.t(), 2)
    _refused(ascq.moe_route, logits.int(), 2, status=ascq.E_UNSUPPORTED)
    slots, tokens, wts = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(4, 2)
    _refused(ascq.moe_dispatch, x, xs, slots, tokens)  # CPU tensors
    _refused(ascq.moe_dispatch, x, xs, slots.long(), tokens)
    _refused(ascq.moe_dispatch, x, xs, slots, tokens[:7])
    _refused(ascq.moe_dispatch, x, None, slots, tokens, scale_out=torch.zeros(8))
    y = torch.zeros(8, 64)
    _refused(ascq.moe_combine, y, slots, wts)  # CPU tensors
    _refused(ascq.moe_combine, y[:7], slots, wts)
    _refused(ascq.moe_combine, y, slots, wts.half())
    _refused(ascq.moe_combine, y, slots, wts, residual=torch.zeros(4, 64).half())
    _refused(ascq.moe_combine_grad, torch.zeros(3, 64), y, slots, tokens, wts)
    _refused(ascq.moe_combine_grad, torch.zeros(4, 64), y, slots, tokens, wts, out=torch.zeros(4, 3))
