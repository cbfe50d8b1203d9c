"""Refusals of the paged int4 cache's operators: bad arguments give a negative status and a message, and launch nothing -- no GPU
needed.  The Python binding refuses tensors of the wrong shape, type, layout or device, and takes memory from the right stream."""
from __future__ import annotations

import ctypes

import pytest
import torch

import ascq
from test_block_checks import D, ODD, _err, _refused
from test_block_streams import SIDE, host  # noqa: F401  (a fixture)

OFF8 = ctypes.c_void_p(0x1008)


def _cache(k=D, v=D, ks=D, vs=D, pages=10, ldc=0, lds=0, kv=2, page=16, d=128, group=32):
    return ctypes.byref(ascq._KvCache(k, v, ks, vs, pages, ldc, lds, kv, page, d, group))


def _seq(table=D, lengths=D, starts=None, ld=0, batch=3, columns=4):
    return ctypes.byref(ascq._KvSequences(table, lengths, starts, ld, batch, columns))


BAD_CACHE = [(dict(k=None), ascq.E_INVALID_ARG), (dict(v=None), ascq.E_INVALID_ARG), (dict(ks=None), ascq.E_INVALID_ARG),
             (dict(vs=None), ascq.E_INVALID_ARG), (dict(k=OFF8), ascq.E_INVALID_ARG), (dict(vs=OFF8), ascq.E_INVALID_ARG),
             (dict(pages=0), ascq.E_INVALID_ARG), (dict(pages=-1), ascq.E_INVALID_ARG), (dict(pages=1 << 31), ascq.E_UNSUPPORTED),
             (dict(kv=0), ascq.E_INVALID_ARG), (dict(kv=1025), ascq.E_UNSUPPORTED), (dict(d=96), ascq.E_UNSUPPORTED),
             (dict(d=0), ascq.E_UNSUPPORTED), (dict(d=512), ascq.E_UNSUPPORTED), (dict(group=16), ascq.E_UNSUPPORTED),
             (dict(group=0), ascq.E_UNSUPPORTED), (dict(d=64, group=128), ascq.E_UNSUPPORTED), (dict(page=8), ascq.E_UNSUPPORTED),
             (dict(page=48), ascq.E_UNSUPPORTED), (dict(page=2048), ascq.E_UNSUPPORTED), (dict(page=-16), ascq.E_UNSUPPORTED),
             (dict(ldc=2047), ascq.E_INVALID_ARG), (dict(ldc=2056), ascq.E_INVALID_ARG), (dict(lds=255), ascq.E_INVALID_ARG),
             (dict(lds=260), ascq.E_INVALID_ARG), (dict(ldc=1 << 60), ascq.E_UNSUPPORTED)]
BAD_SEQ = [(dict(table=None), ascq.E_INVALID_ARG), (dict(lengths=None), ascq.E_INVALID_ARG), (dict(table=ODD), ascq.E_INVALID_ARG),
           (dict(lengths=ODD), ascq.E_INVALID_ARG), (dict(batch=-1), ascq.E_INVALID_ARG), (dict(columns=-1), ascq.E_INVALID_ARG),
           (dict(ld=3), ascq.E_INVALID_ARG), (dict(columns=1 << 27), ascq.E_UNSUPPORTED), (dict(ld=1 << 60), ascq.E_UNSUPPORTED)]


def test_append_arguments():
    def call(k=D, v=D, slots=D, t=4, ldk=0, hdk=0, ldv=0, hdv=0, ty=ascq.F16, cache=None):
        p = ascq._KvAppendParam(t, ldk, hdk, ldv, hdv, ty)
        return ascq.lib().ascq_kv_append(cache or _cache(), k, v, slots, ctypes.byref(p), None)

    _err(ascq.lib().ascq_kv_append(_cache(), D, D, D, None, None), ascq.E_INVALID_ARG, "null params")
    _err(ascq.lib().ascq_kv_append(None, D, D, D, ctypes.byref(ascq._KvAppendParam(1, 0, 0, 0, 0, ascq.F16)), None),
         ascq.E_INVALID_ARG, "null cache")
    for bad, status in BAD_CACHE:
        _err(call(cache=_cache(**bad)), status)
    for bad in (dict(k=None), dict(v=None), dict(slots=None), dict(k=ODD), dict(v=ODD), dict(slots=ctypes.c_void_p(0x1004)),
                dict(t=-1), dict(ldk=100), dict(ldv=127), dict(hdk=127), dict(hdv=1),
                dict(k=ctypes.c_void_p(0x1002), ty=ascq.F32)):
        _err(call(**bad), ascq.E_INVALID_ARG)
    _err(call(ty=ascq.INT8), ascq.E_UNSUPPORTED)
    _err(call(t=1 << 31), ascq.E_UNSUPPORTED)
    _err(call(t=1 << 20, ldk=1 << 40), ascq.E_UNSUPPORTED)
    _err(call(t=0, k=None, v=None, slots=None), ascq.OK)


@pytest.mark.parametrize("name", ["attention", "size", "weights"])
def test_attention_arguments(name):
    L = ascq.lib()

    def call(out=D, lse=D, q=D, t=3, most=1, ldq=0, hdq=0, ldo=0, hdo=0, window=0, ty=ascq.F16, heads=4, causal=1, scale=1.0, cap=64,
             decay=1.0, w=None, cache=None, seq=None):
        p = ctypes.byref(ascq._KvAttentionParam(t, most, ldq, hdq, ldo, hdo, window, ty, heads, causal, scale))
        c, s = cache or _cache(), seq or _seq()
        if name == "size":
            return L.ascq_kv_attention_workspace_size(c, s, p, ctypes.byref(ctypes.c_size_t(0)))
        if name == "weights":
            return L.ascq_kv_weights(out, w, cap, decay, q, lse, c, s, p, None)
        return L.ascq_kv_attention(out, lse, q, c, s, p, None, 0, None)

    for bad, status in BAD_CACHE:
        _err(call(cache=_cache(**bad)), status)
    for bad, status in BAD_SEQ:
        _err(call(seq=_seq(**bad)), status)
    _err(call(seq=_seq(starts=ODD)), ascq.E_INVALID_ARG)
    for bad in (dict(t=-1), dict(t=4), dict(window=-1), dict(heads=0), dict(heads=3), dict(heads=-2), dict(causal=2), dict(hdq=127),
                dict(ldq=127), dict(hdo=5), dict(ldo=64), dict(scale=float("nan")), dict(scale=float("inf")),
                dict(most=-1, seq=_seq(starts=D))):
        _err(call(**bad), ascq.E_INVALID_ARG)
    for bad in (dict(ty=ascq.F32), dict(ty=ascq.INT8), dict(heads=1 << 17), dict(ldq=1 << 60),
                dict(t=1 << 31, seq=_seq(starts=D)), dict(t=1 << 30, most=1 << 30, heads=64, seq=_seq(starts=D))):
        _err(call(**bad), ascq.E_UNSUPPORTED)
    none = _seq(table=None, lengths=None, batch=0)
    _err(call(t=0, out=None, lse=None, q=None, seq=none), ascq.OK)
    if name == "size":
        _err(L.ascq_kv_attention_workspace_size(_cache(), _seq(), None, ctypes.byref(ctypes.c_size_t(0))), ascq.E_INVALID_ARG)
        _err(L.ascq_kv_attention_workspace_size(_cache(), _seq(), ctypes.byref(ascq._KvAttentionParam()), None), ascq.E_INVALID_ARG)
        return
    for bad in (dict(out=None), dict(q=None), dict(out=ODD), dict(q=ODD), dict(lse=ODD)):
        _err(call(**bad), ascq.E_INVALID_ARG)
    if name == "weights":
        for bad in (dict(lse=None), dict(cap=63), dict(cap=-1), dict(decay=float("inf")), dict(decay=float("nan")), dict(w=ODD)):
            _err(call(**bad), ascq.E_INVALID_ARG)
        _err(call(cap=1 << 31), ascq.E_UNSUPPORTED)


def test_evict_arguments():
    def call(kept=D, n=ctypes.c_void_p(0x2000), wo=D, w=D, into=None, cap=64, cap_out=64, ldi=0, keep=32, recent=4, pages=2,
             cache=None, seq=None):
        p = ascq._KvEvictParam(cap, cap_out, ldi, keep, recent, pages)
        return ascq.lib().ascq_kv_evict(kept, n, wo, w, into, cache or _cache(), seq or _seq(), ctypes.byref(p), None, 0, None)

    _err(ascq.lib().ascq_kv_evict(D, D, D, D, None, _cache(), _seq(), None, None, 0, None), ascq.E_INVALID_ARG, "null params")
    for bad, status in BAD_CACHE:
        _err(call(cache=_cache(**bad)), status)
    for bad, status in BAD_SEQ:
        _err(call(seq=_seq(**bad)), status)
    other = ctypes.c_void_p(0x3000)
    for bad in (dict(kept=None), dict(n=None), dict(wo=None), dict(w=None), dict(kept=ODD), dict(n=ODD), dict(wo=ODD), dict(w=ODD),
                dict(into=ODD), dict(n=D), dict(keep=0), dict(keep=-1), dict(recent=-1), dict(recent=33), dict(cap=63),
                dict(cap_out=31), dict(cap_out=63), dict(into=D), dict(into=other, pages=1), dict(into=other, ldi=1),
                dict(into=other, pages=-1)):
        _err(call(**bad), ascq.E_INVALID_ARG)
    _err(call(cap=1 << 31, cap_out=1 << 31), ascq.E_UNSUPPORTED)
    _err(call(into=other, ldi=1 << 60), ascq.E_UNSUPPORTED)
    _err(call(seq=_seq(table=None, lengths=None, batch=0), kept=None, n=None), ascq.OK)
    need = ctypes.c_size_t(7)
    size = ascq.lib().ascq_kv_evict_workspace_size
    _err(size(_cache(), _seq(), None), ascq.E_INVALID_ARG)
    for bad, status in BAD_CACHE:
        _err(size(_cache(**bad), _seq(), ctypes.byref(need)), status)
    for bad, status in BAD_SEQ:
        _err(size(_cache(), _seq(**bad), ctypes.byref(need)), status)
    _err(size(_cache(), _seq(), ctypes.byref(need)), ascq.OK)
    assert need.value == 0
    _err(size(_cache(), _seq(columns=1025), ctypes.byref(need)), ascq.OK)
    assert need.value > 0


def test_binding_refusals():
    cache = ascq.kv_cache(4, 2, 16, 128, 32, device="cpu")
    k = torch.zeros(3, 2, 128, dtype=torch.float16)
    slots = torch.zeros(3, dtype=torch.int64)
    _refused(ascq.kv_append, cache, k, k, slots)  # CPU tensors
    _refused(ascq.kv_append, cache, k, k[:2], slots)
    _refused(ascq.kv_append, cache, k, k.float(), slots)
    _refused(ascq.kv_append, cache, k, k, slots.int())
    _refused(ascq.kv_append, cache, k, k, slots[:2])
    _refused(ascq.kv_append, cache, k[:, :1], k[:, :1], slots)
    _refused(ascq.kv_append, cache, k[:, :, :64], k[:, :, :64], slots)
    _refused(ascq.kv_append, cache, k[0], k[0], slots)
    _refused(ascq.kv_append, cache, k.transpose(1, 2), k, slots)
    _refused(ascq.kv_append, cache, torch.zeros(3, 2, 256, dtype=torch.float16)[:, :, ::2], k, slots)
    _refused(ascq.kv_append, cache, k[:, :1].expand(3, 2, 128), k, slots)
    _refused(ascq.kv_append, cache, k.int(), k.int(), slots, status=ascq.E_UNSUPPORTED)
    good = dict(zip(("k", "v", "k_scale", "v_scale"), cache))
    for bad in (dict(k=cache.k.int()), dict(v=cache.v[:3]), dict(k_scale=cache.k_scale.float()),
                dict(v_scale=cache.v_scale[:, :, :, :2]), dict(k=cache.k.transpose(1, 2)),
                dict(k=torch.zeros(8, 2, 16, 64, dtype=torch.uint8)[::2]), dict(k=cache.k[0]),
                dict(k_scale=cache.k_scale[..., :1], v_scale=cache.v_scale[..., :1]),
                dict(k_scale=cache.k_scale[:, :, :, :3], v_scale=cache.v_scale[:, :, :, :3])):
        _refused(lambda **kw: ascq.KvCache(**kw), **{**good, **bad})
    with pytest.raises(AttributeError):
        cache.k = cache.v
    q, table, lengths = torch.zeros(3, 4, 128, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32), torch.ones(3).int()
    att = ascq.kv_attention
    _refused(att, q, cache, table, lengths)  # CPU tensors
    _refused(att, q[0], cache, table, lengths)
    _refused(att, q[:, :, :64], cache, table, lengths)
    _refused(att, q, cache, table.long(), lengths)
    _refused(att, q, cache, table[0], lengths)
    _refused(att, q, cache, table, lengths[:2])
    _refused(att, q, cache, table, lengths.long())
    _refused(att, q, cache, table, lengths, starts=lengths)
    _refused(att, q, cache, table.t(), lengths)
    _refused(att, q, cache, table, lengths, out=q.half())
    _refused(att, q, cache, table, lengths, out=q[:2])
    _refused(att, q, cache, table, lengths, lse=torch.zeros(3, 2))
    _refused(att, q, cache, table, lengths, workspace=torch.zeros(8, 2)[:, ::2])
    _refused(att, q.float(), cache, table, lengths, status=ascq.E_UNSUPPORTED)
    lse, w = torch.zeros(3, 4), torch.zeros(3, 2, 32)
    _refused(ascq.kv_weights, q, lse, cache, table, lengths)  # CPU tensors
    _refused(ascq.kv_weights, q, lse[:2], cache, table, lengths)
    _refused(ascq.kv_weights, q, lse, cache, table, lengths, weights=w[:, :1])
    _refused(ascq.kv_weights, q, lse, cache, table, lengths, weights=w, out=w[:, :, :31].contiguous())
    _refused(ascq.kv_weights, q, lse, cache, table, lengths, out=w.double())
    ev = ascq.kv_evict
    _refused(ev, cache, table, lengths, w, 8)  # CPU tensors
    _refused(ev, cache, table, lengths, w, 0)
    _refused(ev, cache, table, lengths, w[0], 8)
    _refused(ev, cache, table, lengths, w[:, :1], 8)
    _refused(ev, cache, table, lengths, w, 8, into=table.long())
    _refused(ev, cache, table, lengths, w, 8, into=table[:2])
    _refused(ev, cache, table, lengths, w, 8, kept=torch.zeros(3, 2, 7).int())
    _refused(ev, cache, table, lengths, w, 8, lengths_out=lengths.long())
    _refused(ev, cache, table, lengths, w, 8, weights_out=w[:, :, ::2])
    _refused(ev, cache, table, lengths, w, 8, workspace=w[:, :, ::2])


def _calls(v):
    c, kw = v["cache"], dict(stream=v["stream"])
    table, n, q = v["table"], v["n"], v["q"]
    return {
        "attention": lambda: ascq.kv_attention(q, c, table, n, need_lse=True, **kw),
        "weights": lambda: ascq.kv_weights(q, v["lse"], c, table, n, **kw),
        "evict": lambda: ascq.kv_evict(c, table, n, v["w"], 8, **kw)[:2],
    }


@pytest.mark.parametrize("side", [False, True])
@pytest.mark.parametrize("name", ["attention", "weights", "evict"])
def test_memory_of_a_call_comes_from_its_stream(host, name, side):  # noqa: F811
    real = host.args["h"].new_empty
    v = dict(cache=ascq.KvCache(real(4, 2, 16, 64, dtype=torch.uint8), real(4, 2, 16, 64, dtype=torch.uint8),
                                real(4, 2, 16, 4, 2, dtype=torch.float16), real(4, 2, 16, 4, 2, dtype=torch.float16)),
             table=real(3, 2, dtype=torch.int32), n=real(3, dtype=torch.int32), q=real(3, 4, 128), lse=real(3, 4, dtype=torch.float32),
             w=real(3, 2, 32, dtype=torch.float32), stream=host.Stream(SIDE) if side else None)
    host.taken.clear()
    out = _calls(v)[name]()
    results = [t for t in (out if isinstance(out, tuple) else (out,)) if t is not None]
    where = SIDE if side else 0
    assert host.taken and all(st == where for st, _ in host.taken)
    assert len(host.recorded) == (len(results) if side else 0)
    assert {id(t) for t, _ in host.recorded} <= {id(t) for t in results}
