"""Where the binding takes memory for a call on a stream that is not the current one (CPU only: torch's streams, its
allocation and the library are stood in for)."""
from __future__ import annotations

import contextlib
import types

import pytest
import torch

import ascq

SIDE = 0x5EED


@pytest.fixture
def host(monkeypatch):
    """records (stream, shape, dtype) of every torch.empty, and the tensors recorded on a stream; calls launch nothing"""
    log = types.SimpleNamespace(current=[0], taken=[], recorded=[])

    class Stream:
        def __init__(self, handle):
            self.cuda_stream = handle

    @contextlib.contextmanager
    def use(st):
        log.current.append(st.cuda_stream)
        yield
        log.current.pop()

    class Library:
        def __getattr__(self, name):
            if name.endswith("workspace_size"):
                def size(*args):
                    args[-1]._obj.value = 4096
                    return ascq.OK
                return size
            return lambda *args: ascq.OK

    real = torch.empty
    monkeypatch.setattr(torch.cuda, "stream", use)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Stream(log.current[-1]))
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle, *a: Stream(handle))
    monkeypatch.setattr(ascq, "lib", Library)
    monkeypatch.setattr(ascq, "_stream_ready", False)
    monkeypatch.setattr(ascq, "_raw_stream", None)
    monkeypatch.setattr(ascq, "_same_device", lambda *a: None, raising=False)
    x = dict(device="meta")
    log.args = dict(
        h=real(4, 64, dtype=torch.float16, **x), g=real(64, dtype=torch.float16, **x), q=real(4, 64, dtype=torch.int8, **x),
        w=real(32, 64, dtype=torch.int8, **x), s4=real(4, **x), s32=real(32, **x), logits=real(4, 8, **x), k2=real(4, 2, **x),
        i42=real(4, 2, dtype=torch.int32, **x), i8=real(8, dtype=torch.int32, **x), c8=real(8, dtype=torch.int64, **x),
        one=real(1, dtype=torch.int64, **x), y=real(8, 64, dtype=torch.float16, **x))

    def empty(*args, **kw):
        t = real(*args, **kw)
        log.taken.append((log.current[-1], t))
        return t

    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(torch, "empty_like", lambda t: empty(t.shape, dtype=t.dtype, device=t.device))
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, st: log.recorded.append((t, st.cuda_stream)))
    log.Stream = Stream
    return log


CALLS = {
    "norm": lambda a, v, st: a.add_rms_norm_quant(v["h"], v["g"], residual=v["h"], stream=st),
    "linear": lambda a, v, st: a.quant_linear(v["q"], v["s4"], v["w"], v["s32"], stream=st),
    "route": lambda a, v, st: a.moe_route(v["logits"], 2, stream=st),
    "route_grad": lambda a, v, st: a.moe_route_grad(v["logits"], v["k2"], v["i42"], v["c8"], v["one"], stream=st),
    "dispatch": lambda a, v, st: a.moe_dispatch(v["q"], v["s4"], v["i42"], v["i8"], stream=st),
    "combine": lambda a, v, st: a.moe_combine(v["y"], v["i42"], v["k2"], stream=st),
    "combine_grad": lambda a, v, st: a.moe_combine_grad(v["h"], v["y"], v["i42"], v["i8"], v["k2"], stream=st),
    "quant_dynamic": lambda a, v, st: a.quant_dynamic_per_token(v["h"], stream=st),
    "quant_per_token": lambda a, v, st: a.quant_per_token(v["h"], v["s4"], stream=st),
    "quant_policy": lambda a, v, st: a.ascend_quant_policy(v["h"], v["s4"], a.PER_TOKEN, stream=st),
    "quant_policy_fp4": lambda a, v, st: a.ascend_quant_policy(v["h"], v["s4"], a.PER_GROUP, a.FP4_E2M1, stream=st),
    "quant": lambda a, v, st: a.ascend_quant(v["h"], stream=st),
    "dequant": lambda a, v, st: a.ascend_dequant(v["q"], None, scale_type=a.F32, stream=st),
    "dequant_policy": lambda a, v, st: a.ascend_dequant_policy(v["q"], v["s4"], a.PER_TOKEN, stream=st),
    "antiquant": lambda a, v, st: a.ascend_antiquant(v["q"], a.INT8, v["g"], None, 4, 64, stream=st),
    "antiquant_scalar": lambda a, v, st: a.ascend_antiquant_scalar(v["q"], a.INT8, None, 0.5, 256, stream=st),
    "antiquant_policy": lambda a, v, st: a.ascend_antiquant_policy(v["q"], a.INT8, v["s4"], a.F32, a.PER_TOKEN, 4, 64, stream=st),
    "quantize": lambda a, v, st: a.quantize(v["h"], a.PER_TENSOR, stream=st),
    "quantize_fp4": lambda a, v, st: a.quantize(v["h"], a.PER_TENSOR, a.FP4_E2M1, stream=st),
    "dequantize": lambda a, v, st: a.dequantize(v["logits"], a.PER_TENSOR, stream=st),
    "antiquantize": lambda a, v, st: a.antiquantize(v["q"], a.INT8, a.PER_TENSOR, 4, 64, stream=st),
    "weight_pack": lambda a, v, st: a.weight_pack(v["w"], a.INT8, 64, 32, stream=st),
    "antiquant_matmul": lambda a, v, st: a.antiquant_matmul(v["h"], v["w"], a.INT8, v["g"], None, 64, 32, stream=st),
    "group_matmul": lambda a, v, st: a.quant_group_matmul(v["q"], v["s4"], v["w"], v["k2"], v["c8"], stream=st),
    "nz_to_nd": lambda a, v, st: a.nz_to_nd(v["q"], a.INT8, 1, 16, 32, stream=st),
    "nd_to_nz": lambda a, v, st: a.nd_to_nz(v["q"], a.INT8, 1, 16, 32, stream=st),
}


def _tensors(result):
    if isinstance(result, torch.Tensor):
        return [result]
    return [t for t in result if t is not None]


@pytest.mark.parametrize("handle", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_memory_of_a_call_comes_from_its_stream(host, name, handle):
    """Outputs and workspaces are taken from the memory of the stream that writes them -- a block of another stream's may still
    be in use there -- and results, not workspaces, are kept from reuse until the current stream has read them"""
    out = CALLS[name](ascq, host.args, SIDE if handle else host.Stream(SIDE))
    assert host.taken and all(st == SIDE for st, _ in host.taken)
    kept = {id(t) for t, st in host.recorded if st == 0}
    results = [t for t in _tensors(out) if not any(t is v for v in host.args.values())]
    assert results and all(id(t) in kept for t in results)
    assert len(host.recorded) == len(results)


@pytest.mark.parametrize("name", CALLS)
def test_memory_of_a_call_on_the_current_stream(host, name):
    for st in (None, 0, host.Stream(0)):
        host.taken.clear()
        CALLS[name](ascq, host.args, st)
        assert host.taken and all(at == 0 for at, _ in host.taken) and not host.recorded
