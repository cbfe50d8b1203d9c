"""ascq -- Python binding of libascq.so (the gfx950 quantized-inference library).

Thin ctypes layer over the C ABI declared in include/ascq.h.  Tensors are torch tensors on the
GPU (torch is used for device memory and streams only); every compute call goes through the
C ABI into the HIP kernels.  There is no CPU fallback: if libascq.so is missing or a call fails,
an exception is raised.

The operator names and argument meanings mirror the reference's operator surface
(AscendC::Matmul SetTensorA/SetTensorB/SetBias/SetQuantScalar/SetQuantVector/IterateAll/End,
AscendQuant/AscendDequant/AscendAntiQuant, QuantGroupMatmul); see include/ascq.h for the
reference file:line each entry point replaces.
"""
from __future__ import annotations

import ctypes
import os
from pathlib import Path
from typing import NamedTuple

import torch

_PKG_DIR = Path(__file__).resolve().parent.parent
LIB_PATH = Path(os.environ.get("ASCQ_LIB", _PKG_DIR / "libascq.so"))

# ascq_dtype
INT8, UINT8, INT4, INT32, F16, BF16, F32, U64, FP8_E4M3, FP8_E5M2, FP4_E2M1, E8M0, INT64, FP4_E1M2, HIF8 = range(1, 16)
# ascq_round_mode
ROUND_NONE, ROUND_RINT, ROUND_FLOOR, ROUND_CEIL, ROUND_ROUND, ROUND_TRUNC = range(6)
# ascq_policy
ACT_NONE, ACT_FASTER_GELU, ACT_RELU, ACT_GELU, ACT_SILU = range(5)
PER_TENSOR, PER_CHANNEL, PER_TOKEN, PER_GROUP = range(4)
# IterateAll enAtomic (matmul_config_utils.h:53-55)
ATOMIC_NONE, ATOMIC_ADD, ATOMIC_MAX, ATOMIC_MIN = range(4)
# ascq_arith
ARITH_F16, ARITH_F32 = 0, 1
# ascq_dequant_mode (DeQuantMode)
DEQUANT_SINGLE_ROW, DEQUANT_MULTI_ROW = 0, 1
# ascq_format
FORMAT_ND, FORMAT_PACKED, FORMAT_NZ = 0, 1, 2

OK, E_INVALID_ARG, E_UNSUPPORTED, E_HIP, E_STATE = 0, -1, -2, -3, -4

# torch dtype -> ascq_dtype of floating sources, scales and outputs
_FLOAT_CODE = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32}
_SRC_CODE = {torch.int32: INT32, torch.float32: F32, torch.int8: INT8}

_TORCH_OF = {INT8: torch.int8, INT32: torch.int32, F16: torch.float16, BF16: torch.bfloat16, F32: torch.float32}


class AscqError(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"ascq error {status}: {message}")
        self.status = status


class _QuantParam(ctypes.Structure):
    _fields_ = [
        ("m", ctypes.c_uint32),
        ("n", ctypes.c_uint32),
        ("cal_count", ctypes.c_uint32),
        ("group_size", ctypes.c_uint32),
        ("has_offset", ctypes.c_int32),
        ("kdim", ctypes.c_int32),
        ("round_mode", ctypes.c_int32),
    ]


class _DequantParam(ctypes.Structure):
    _fields_ = [("m", ctypes.c_uint32), ("n", ctypes.c_uint32), ("cal_count", ctypes.c_uint32)]


class _DequantPolicyParam(ctypes.Structure):
    _fields_ = [("m", ctypes.c_uint32), ("n", ctypes.c_uint32), ("cal_count", ctypes.c_uint32),
                ("group_size", ctypes.c_uint32), ("has_offset", ctypes.c_int32), ("kdim", ctypes.c_int32)]


class _QuantizeParam(ctypes.Structure):
    """ascq_quantize_param: QuantizeConfig{policy, hasOffset, roundMode, kDim} + QuantizeParams{m, n, groupSize}"""
    _fields_ = [("policy", ctypes.c_int32), ("has_offset", ctypes.c_int32), ("round_mode", ctypes.c_int32),
                ("kdim", ctypes.c_int32), ("m", ctypes.c_uint32), ("n", ctypes.c_uint32),
                ("group_size", ctypes.c_uint32)]


class _NormQuantParam(ctypes.Structure):
    _fields_ = [("m", ctypes.c_int64), ("n", ctypes.c_int64), ("ld_x", ctypes.c_int64),
                ("ld_residual", ctypes.c_int64), ("ld_h", ctypes.c_int64), ("src_type", ctypes.c_int32),
                ("dst_type", ctypes.c_int32), ("eps", ctypes.c_float)]


class _LinearParam(ctypes.Structure):
    _fields_ = [("m", ctypes.c_int64), ("n", ctypes.c_int64), ("k", ctypes.c_int64), ("ld_x", ctypes.c_int64),
                ("ld_w", ctypes.c_int64), ("ld_residual", ctypes.c_int64), ("ld_y", ctypes.c_int64),
                ("operand_type", ctypes.c_int32), ("out_type", ctypes.c_int32), ("w_trans", ctypes.c_int32),
                ("activation", ctypes.c_int32)]


class _RouteParam(ctypes.Structure):
    _fields_ = [("tokens", ctypes.c_int64), ("experts", ctypes.c_int64), ("ld_logits", ctypes.c_int64),
                ("logits_type", ctypes.c_int32), ("top_k", ctypes.c_int32), ("renormalize", ctypes.c_int32)]


class _RowsParam(ctypes.Structure):
    _fields_ = [("tokens", ctypes.c_int64), ("n", ctypes.c_int64), ("ld_x", ctypes.c_int64), ("type", ctypes.c_int32),
                ("top_k", ctypes.c_int32)]


class _KvCache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
                ("pages", ctypes.c_int64), ("ld_codes", ctypes.c_int64), ("ld_scales", ctypes.c_int64),
                ("kv_heads", ctypes.c_int32), ("page_size", ctypes.c_int32), ("d", ctypes.c_int32), ("group", ctypes.c_int32)]


class _KvSequences(ctypes.Structure):
    _fields_ = [("page_table", ctypes.c_void_p), ("lengths", ctypes.c_void_p), ("starts", ctypes.c_void_p),
                ("ld_table", ctypes.c_int64), ("batch", ctypes.c_int32), ("table_pages", ctypes.c_int32)]


class _KvAppendParam(ctypes.Structure):
    _fields_ = [("tokens", ctypes.c_int64), ("ld_k", ctypes.c_int64), ("hd_k", ctypes.c_int64), ("ld_v", ctypes.c_int64),
                ("hd_v", ctypes.c_int64), ("type", ctypes.c_int32)]


class _KvAttentionParam(ctypes.Structure):
    _fields_ = [("tokens", ctypes.c_int64), ("max_queries", ctypes.c_int64), ("ld_q", ctypes.c_int64), ("hd_q", ctypes.c_int64),
                ("ld_out", ctypes.c_int64), ("hd_out", ctypes.c_int64), ("window", ctypes.c_int64), ("type", ctypes.c_int32),
                ("heads", ctypes.c_int32), ("causal", ctypes.c_int32), ("scale", ctypes.c_float)]


class _KvEvictParam(ctypes.Structure):
    _fields_ = [("cap", ctypes.c_int64), ("cap_out", ctypes.c_int64), ("ld_into", ctypes.c_int64), ("keep", ctypes.c_int32),
                ("recent", ctypes.c_int32), ("into_pages", ctypes.c_int32)]


class _MatmulTypes(ctypes.Structure):
    _fields_ = [
        ("a_type", ctypes.c_int32),
        ("b_type", ctypes.c_int32),
        ("c_type", ctypes.c_int32),
        ("bias_type", ctypes.c_int32),
        ("scale_type", ctypes.c_int32),
        ("b_format", ctypes.c_int32),
    ]


CUBE_TILING_FIELDS = (
    "usedCoreNum M N Ka Kb singleCoreM singleCoreN singleCoreK baseM baseN baseK depthA1 depthB1 stepM stepN isBias "
    "transLength iterateOrder shareMode shareL1Size shareL0CSize shareUbSize batchM batchN singleBatchM singleBatchN "
    "stepKa stepKb depthAL1CacheUB depthBL1CacheUB dbL0A dbL0B dbL0C ALayoutInfoB ALayoutInfoS ALayoutInfoN "
    "ALayoutInfoG ALayoutInfoD BLayoutInfoB BLayoutInfoS BLayoutInfoN BLayoutInfoG BLayoutInfoD CLayoutInfoB "
    "CLayoutInfoS1 CLayoutInfoN CLayoutInfoG CLayoutInfoS2 BatchNum mxTypePara").split()


class CubeTiling(ctypes.Structure):
    """ascq_cube_tiling: the reference's TCubeTiling fields in their order (matmul_tilingdata.h:21-72)"""
    _fields_ = [(f, ctypes.c_int32) for f in CUBE_TILING_FIELDS]


_P = ctypes.c_void_p
_I32, _U32, _I64, _U64, _U16, _U8, _F32 = (ctypes.c_int32, ctypes.c_uint32, ctypes.c_int64, ctypes.c_uint64,
                                          ctypes.c_uint16, ctypes.c_uint8, ctypes.c_float)

# name -> (restype, argtypes)
SIGNATURES = {
    "ascq_last_error": (ctypes.c_char_p, []),
    "ascq_version": (ctypes.c_char_p, []),
    "ascq_device_count": (_I32, []),
    "ascq_set_launch_events": (_I32, [_P, _P]),
    "ascq_pack_quant_pre": (_U64, [_F32, _I32, _I32]),
    "ascq_matmul_create": (_I32, [ctypes.POINTER(_MatmulTypes), ctypes.POINTER(_P)]),
    "ascq_matmul_init": (_I32, [_P, ctypes.POINTER(CubeTiling)]),
    "ascq_matmul_set_org_shape": (_I32, [_P, _I64, _I64, _I64]),
    "ascq_matmul_set_single_shape": (_I32, [_P, _I64, _I64, _I64]),
    "ascq_matmul_set_tail": (_I32, [_P, _I64, _I64, _I64]),
    "ascq_matmul_set_tensor_a": (_I32, [_P, _P, _I32]),
    "ascq_matmul_set_tensor_b": (_I32, [_P, _P, _I32]),
    "ascq_matmul_set_bias": (_I32, [_P, _P]),
    "ascq_matmul_disable_bias": (_I32, [_P]),
    "ascq_matmul_set_quant_scalar": (_I32, [_P, _U64]),
    "ascq_matmul_set_quant_vector": (_I32, [_P, _P]),
    "ascq_matmul_set_antiquant_scalar": (_I32, [_P, _U16, _U16]),
    "ascq_matmul_set_antiquant_vector": (_I32, [_P, _P, _P, _I64]),
    "ascq_matmul_set_tensor_scale_a": (_I32, [_P, _P, _I32]),
    "ascq_matmul_set_tensor_scale_b": (_I32, [_P, _P, _I32]),
    "ascq_matmul_workspace_size": (_I32, [_P, ctypes.POINTER(ctypes.c_size_t)]),
    "ascq_matmul_set_workspace": (_I32, [_P, _P, ctypes.c_size_t]),
    "ascq_matmul_iterate_all": (_I32, [_P, _P, _U8, _P]),
    "ascq_matmul_iterate_all_noalloc": (_I32, [_P, _P, _U8, _P]),
    "ascq_matmul_end": (_I32, [_P]),
    "ascq_matmul_destroy": (_I32, [_P]),
    "ascq_ascend_quant_per_token": (_I32, [_P, _P, _I32, _P, _P, ctypes.POINTER(_QuantParam), _P]),
    "ascq_ascend_quant_dynamic_per_token": (_I32, [_P, _P, _P, _I32, _U32, _U32, _I32, _P]),
    "ascq_ascend_quant_policy": (_I32, [_P, _I32, _P, _I32, _P, _P, _F32, _I32, _I32, ctypes.POINTER(_QuantParam), _P]),
    "ascq_ascend_quant": (_I32, [_P, _I32, _P, _I32, _P, _P, _F32, _F32, _U32, _U32, _P]),
    "ascq_ascend_antiquant_scalar": (_I32, [_P, _I32, _P, _I32, _U16, _U16, _I32, _U64, _P]),
    "ascq_ascend_dequant": (_I32, [_P, _I32, _P, _I32, _P, _I32, _F32, _I32, _I32, ctypes.POINTER(_DequantParam),
                                   _P]),
    "ascq_ascend_dequant_dst_shape": (_I32, [_I32, _I32, ctypes.POINTER(_DequantParam), ctypes.POINTER(_U32),
                                             ctypes.POINTER(_U32)]),
    "ascq_ascend_dequant_policy": (_I32, [_P, _I32, _P, _I32, _P, _P, _I32, _I32, ctypes.POINTER(_DequantPolicyParam),
                                          _P]),
    "ascq_ascend_antiquant": (_I32, [_P, _I32, _P, _I32, _P, _P, _U32, _U32, _U32, _I32, _I32, _P]),
    "ascq_quantize": (_I32, [_P, _I32, _P, _I32, _P, _P, _F32, _F32, _I32, ctypes.POINTER(_QuantizeParam), _P]),
    "ascq_dequantize": (_I32, [_P, _I32, _P, _I32, _P, _F32, _I32, ctypes.POINTER(_QuantizeParam), _P]),
    "ascq_antiquantize": (_I32, [_P, _I32, _P, _I32, _P, _P, _F32, _F32, _I32, ctypes.POINTER(_QuantizeParam), _P]),
    "ascq_ascend_antiquant_policy": (_I32, [_P, _I32, _P, _I32, _P, _P, _I32, _I32, ctypes.c_int64, ctypes.c_int64,
                                            ctypes.c_int64, _I32, _I32, _P]),
    "ascq_weight_pack_size": (_I32, [_I32, _I64, _I64, ctypes.POINTER(ctypes.c_size_t)]),
    "ascq_weight_pack": (_I32, [_P, _P, _I32, _I64, _I64, _I32, _P]),
    "ascq_antiquant_matmul": (_I32, [_P, _P, _P, _I32, _P, _P, _I64, _I64, _I64, _I64, _P]),
    "ascq_quant_group_matmul": (_I32, [_P, _I32, _P, _P, _P, _I32, _P, _P, _I32, _I64, _I64, _I64, _I64, _I32, _P]),
    "ascq_add_rms_norm_quant": (_I32, [_P] * 7 + [ctypes.POINTER(_NormQuantParam), _P]),
    "ascq_quant_linear_workspace_size": (_I32, [_P, _P, ctypes.POINTER(_LinearParam), ctypes.POINTER(ctypes.c_size_t)]),
    "ascq_quant_linear": (_I32, [_P] * 7 + [ctypes.POINTER(_LinearParam), _P, ctypes.c_size_t, _P]),
    "ascq_moe_route_workspace_size": (_I32, [ctypes.POINTER(_RouteParam), ctypes.POINTER(ctypes.c_size_t)]),
    "ascq_moe_route": (_I32, [_P] * 8 + [ctypes.POINTER(_RouteParam), _P, ctypes.c_size_t, _P]),
    "ascq_moe_route_grad": (_I32, [_P, _I64] + [_P] * 7 + [ctypes.POINTER(_RouteParam), _P]),
    "ascq_moe_dispatch": (_I32, [_P] * 6 + [ctypes.POINTER(_RowsParam), _P]),
    "ascq_moe_combine": (_I32, [_P] * 5 + [ctypes.POINTER(_RowsParam), _P]),
    "ascq_moe_combine_grad": (_I32, [_P] * 7 + [ctypes.POINTER(_RowsParam), _P]),
    "ascq_kv_append": (_I32, [ctypes.POINTER(_KvCache), _P, _P, _P, ctypes.POINTER(_KvAppendParam), _P]),
    "ascq_kv_attention_workspace_size": (_I32, [ctypes.POINTER(_KvCache), ctypes.POINTER(_KvSequences),
                                                ctypes.POINTER(_KvAttentionParam), ctypes.POINTER(ctypes.c_size_t)]),
    "ascq_kv_attention": (_I32, [_P] * 3 + [ctypes.POINTER(_KvCache), ctypes.POINTER(_KvSequences),
                                            ctypes.POINTER(_KvAttentionParam), _P, ctypes.c_size_t, _P]),
    "ascq_kv_weights": (_I32, [_P, _P, _I64, _F32, _P, _P, ctypes.POINTER(_KvCache), ctypes.POINTER(_KvSequences),
                               ctypes.POINTER(_KvAttentionParam), _P]),
    "ascq_kv_evict": (_I32, [_P] * 5 + [ctypes.POINTER(_KvCache), ctypes.POINTER(_KvSequences), ctypes.POINTER(_KvEvictParam),
                                        _P, ctypes.c_size_t, _P]),
    "ascq_kv_evict_workspace_size": (_I32, [ctypes.POINTER(_KvCache), ctypes.POINTER(_KvSequences),
                                            ctypes.POINTER(ctypes.c_size_t)]),
    "ascq_nz_size": (ctypes.c_size_t, [_I32, _I64, _I64, _I64]),
    "ascq_nz_to_nd": (_I32, [_P, _P, _I32, _I64, _I64, _I64, _I32, _P]),
    "ascq_nd_to_nz": (_I32, [_P, _P, _I32, _I64, _I64, _I64, _P]),
}

_lib = None


def lib() -> ctypes.CDLL:
    """Load libascq.so (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise AscqError(E_STATE, f"{LIB_PATH} not found: build it with python asc-devkit_clone_amd/build.py")
        handle = ctypes.CDLL(str(LIB_PATH))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def last_error() -> str:
    return lib().ascq_last_error().decode()


def check(status: int, what: str) -> None:
    if status != OK:
        raise AscqError(status, f"{what}: {last_error()}")


def _ptr(t) -> int | None:
    if t is None or isinstance(t, int):
        return t
    return t.data_ptr()


# The current stream's handle.  torch.cuda.current_stream() builds a Stream object around it, 2.5 us of the 6.7 us that a
# small call took; the binding it is built from returns the handle itself in 0.14 us.  The first call goes the public
# way (which also initialises the device).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_stream_ready = False


def _forked() -> None:
    """A forked child goes the public way again, which refuses a device that the parent initialised"""
    global _stream_ready
    _stream_ready = False


os.register_at_fork(after_in_child=_forked)


def _stream(stream) -> int | None:
    global _stream_ready
    if stream is None:
        if _stream_ready:
            return _raw_stream(_current_device())
        handle = torch.cuda.current_stream().cuda_stream
        _stream_ready = _raw_stream is not None and _current_device is not None
        return handle
    return stream if isinstance(stream, int) else stream.cuda_stream


def _new(stream, shape, dtype, device, private: bool = False) -> torch.Tensor:
    """An uninitialised tensor for kernels on `stream` (None: the current one), taken from that stream's memory: a block of
    the current stream's may still be in use by work queued there, which `stream` does not wait for.  The caller reads a
    result on the current stream as a rule, so a block given back is not reused before that stream's work is done either;
    `private`: the call's own, which only `stream` uses."""
    if stream is None or device.type == "cpu":
        return torch.empty(shape, dtype=dtype, device=device)
    current = torch.cuda.current_stream(device)
    if current.cuda_stream == _stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(torch.cuda.ExternalStream(stream, device) if isinstance(stream, int) else stream):
        t = torch.empty(shape, dtype=dtype, device=device)
    if not private:
        t.record_stream(current)
    return t


def _half_bits(v: float) -> int:
    return int(torch.tensor([v], dtype=torch.float16).view(torch.int16).item()) & 0xFFFF


def pack_quant_pre(m1: float, offset9: int = 0, sign: int = 0) -> int:
    return int(lib().ascq_pack_quant_pre(float(m1), offset9, sign))


# ------------------------------------------------------------------------------------------
# AscendQuant / AscendDequant / AscendAntiQuant
# ------------------------------------------------------------------------------------------
def quant_dynamic_per_token(x: torch.Tensor, round_mode: int = ROUND_RINT, out=None, scale_out=None, stream=None):
    """Per-row absmax -> int8 q and fp32 scale (= absmax/127).  x: [m, n] f16 / bf16 / f32."""
    m, n = x.shape
    src_type = _FLOAT_CODE[x.dtype]
    q = out if out is not None else _new(stream, (m, n), torch.int8, x.device)
    s = scale_out if scale_out is not None else _new(stream, (m,), torch.float32, x.device)
    check(lib().ascq_ascend_quant_dynamic_per_token(_ptr(q), _ptr(s), _ptr(x), src_type, m, n, round_mode,
                                                    _stream(stream)), "quant_dynamic_per_token")
    return q, s


def quant_per_token(x: torch.Tensor, scale: torch.Tensor, offset=None, round_mode: int = ROUND_RINT, out=None,
                    stream=None):
    """AscendQuant PER_TOKEN: q = sat_s8(round(f32(x) * scale[row] (+ offset[row])))."""
    m, n = x.shape
    src_type = _FLOAT_CODE[x.dtype]
    q = out if out is not None else _new(stream, (m, n), torch.int8, x.device)
    p = _QuantParam(m, n, m * n, 0, 1 if offset is not None else 0, 1, round_mode)
    check(lib().ascq_ascend_quant_per_token(_ptr(q), _ptr(x), src_type, _ptr(scale), _ptr(offset), ctypes.byref(p),
                                            _stream(stream)), "quant_per_token")
    return q


def ascend_quant_policy(x: torch.Tensor, scale: torch.Tensor, policy: int, dst_type: int = INT8,
                        group_size: int = 0, offset=None, offset_scalar=None, k_dim: int = 1,
                        round_mode: int = ROUND_RINT, scale_type: int | None = None, out=None, stream=None):
    """AscendQuant policy form (PER_TOKEN / PER_GROUP) of x [m, n] (f16 / bf16 / f32) to int8, fp8 (e4m3 / e5m2;
    returned as uint8 codes) or fp4 E2M1 / E1M2 (two codes a byte, [m, n/2] uint8).  scale / offset f16 / bf16 / f32; a
    scalar offset_scalar applies when no offset tensor is given."""
    m, n = x.shape
    src_type = _FLOAT_CODE[x.dtype]
    if scale_type is None:
        scale_type = _FLOAT_CODE[scale.dtype]
    if out is not None:
        q = out
    elif dst_type in (FP4_E2M1, FP4_E1M2):
        q = _new(stream, (m, n // 2), torch.uint8, x.device)
    else:
        q = _new(stream, (m, n), torch.int8 if dst_type == INT8 else torch.uint8, x.device)
    has_off = offset is not None or offset_scalar is not None
    p = _QuantParam(m, n, m * n, group_size, int(has_off), k_dim, round_mode)
    check(lib().ascq_ascend_quant_policy(_ptr(q), dst_type, _ptr(x), src_type, _ptr(scale), _ptr(offset),
                                         float(offset_scalar or 0.0), scale_type, policy, ctypes.byref(p),
                                         _stream(stream)), "ascend_quant_policy")
    return q


def ascend_quant(x: torch.Tensor, dst_type: int = INT8, scale=None, offset=None, scale_scalar: float = 1.0,
                 offset_scalar: float = 0.0, scale_count: int = 0, out=None, stream=None):
    """Legacy AscendQuant (arch-3510 form): per tensor (float scalars) or per channel (scale / offset tensors of the
    source's type; offset None takes offset_scalar as a source-typed value).  dst INT8 / HIF8 (half arithmetic) or
    FP8_E4M3 / FP8_E5M2 (fp32 arithmetic); returns int8 (INT8) or uint8 codes of x's shape."""
    src_type = _FLOAT_CODE[x.dtype]
    q = out if out is not None else _new(stream, x.shape, torch.int8 if dst_type == INT8 else torch.uint8, x.device)
    if scale is not None:
        scale_count = scale_count or scale.numel()
    check(lib().ascq_ascend_quant(_ptr(q), dst_type, _ptr(x), src_type, _ptr(scale), _ptr(offset), float(scale_scalar),
                                  float(offset_scalar), x.numel(), scale_count, _stream(stream)), "ascend_quant")
    return q


def _dtype_code(t) -> int:
    return _FLOAT_CODE[t]


def dequant_dst_shape(dst_dtype, m: int, n: int, cal_count: int, mode: int = DEQUANT_SINGLE_ROW):
    """(rows, row stride) of the legacy AscendDequant's dst after the DEQUANT_WITH_SINGLE_ROW rule"""
    rows, ldd = _U32(), _U32()
    p = _DequantParam(m, n, cal_count)
    check(lib().ascq_ascend_dequant_dst_shape(_dtype_code(dst_dtype), mode, ctypes.byref(p), ctypes.byref(rows),
                                              ctypes.byref(ldd)), "ascend_dequant_dst_shape")
    return rows.value, ldd.value


def ascend_dequant(src: torch.Tensor, scale, dst_dtype=torch.float16, cal_count=None, scale_scalar: float = 1.0,
                   scale_type: int | None = None, mode: int = DEQUANT_SINGLE_ROW, m: int | None = None,
                   n: int | None = None, out=None, stream=None):
    """Legacy AscendDequant<dstT, scaleT, mode>(dst, src, deqScale, {m, n, calCount}): `scale` a deqScale tensor
    (f32 / bf16, or int64 holding uint64 words) or None for the scalar `scale_scalar` (scale_type F32 or BF16).
    Returns dst as [rows, row stride] (rows of n padded to 32 bytes; unwritten elements keep `out`'s values)."""
    if m is None:
        m, n = src.shape
    cal = n if cal_count is None else cal_count
    src_type = {torch.int32: INT32, torch.int8: INT8}[src.dtype]
    dst_type = _dtype_code(dst_dtype)
    if scale_type is None:
        scale_type = F32 if scale is None else {torch.float32: F32, torch.bfloat16: BF16, torch.int64: U64}[scale.dtype]
    rows, ldd = dequant_dst_shape(dst_dtype, m, n, cal, mode)
    y = out if out is not None else _new(stream, (rows, ldd), dst_dtype, src.device)
    p = _DequantParam(m, n, cal)
    check(lib().ascq_ascend_dequant(_ptr(y), dst_type, _ptr(src), src_type, _ptr(scale), scale_type,
                                    float(scale_scalar), PER_TENSOR if scale is None else PER_CHANNEL, mode,
                                    ctypes.byref(p), _stream(stream)), "ascend_dequant")
    return y


def ascend_dequant_policy(src: torch.Tensor, scale: torch.Tensor, policy: int, dst_dtype=torch.float16,
                          group_size: int = 0, kdim: int = 1, cal_count=None, offset=None, out=None, stream=None):
    """AscendDequant<dstT, srcT, scaleT, {hasOffset, kDim}, policy>(dst, src, scale, offset, {m, n, calCount,
    groupSize}): PER_TOKEN (scale[row]) or PER_GROUP (kdim 1: scale[row][col / g]; kdim 0: scale[row / g][col])
    on src [rows, n] int32 / f32 (or int8); scale f32 / f16 / bf16."""
    m, n = src.shape
    src_type = _SRC_CODE[src.dtype]
    scale_type = _FLOAT_CODE[scale.dtype]
    y = out if out is not None else _new(stream, (m, n), dst_dtype, src.device)
    p = _DequantPolicyParam(m, n, m * n if cal_count is None else cal_count, group_size, int(offset is not None), kdim)
    check(lib().ascq_ascend_dequant_policy(_ptr(y), _dtype_code(dst_dtype), _ptr(src), src_type, _ptr(scale),
                                           _ptr(offset), scale_type, policy, ctypes.byref(p), _stream(stream)),
          "ascend_dequant_policy")
    return y


def ascend_antiquant(src: torch.Tensor, src_type: int, scale: torch.Tensor, offset, k: int, n: int,
                     group_size: int = 0, is_transpose: bool = False, dst_dtype=torch.float16,
                     arith: int = ARITH_F16, out=None, stream=None):
    """AscendAntiQuant: dst = (src + offset) * scale.  Returns [K, N] (or [N, K] when is_transpose)."""
    dst_type = {torch.float16: F16, torch.bfloat16: BF16}[dst_dtype]
    shape = (n, k) if is_transpose else (k, n)
    y = out if out is not None else _new(stream, shape, dst_dtype, src.device)
    check(lib().ascq_ascend_antiquant(_ptr(y), dst_type, _ptr(src), src_type, _ptr(offset), _ptr(scale), k, n,
                                      group_size, int(is_transpose), arith, _stream(stream)), "ascend_antiquant")
    return y


def ascend_antiquant_scalar(src: torch.Tensor, src_type: int, offset: float | None, scale: float, count: int,
                            dst_dtype=torch.float16, out=None, stream=None):
    """AscendAntiQuant per tensor: dst[i] = (src[i] + offset) * scale with offset / scale of dst_dtype (offset None:
    scale only); count elements (int4 two per byte)."""
    dst_type = {torch.float16: F16, torch.bfloat16: BF16}[dst_dtype]
    bits = lambda v: int(torch.tensor([v], dtype=dst_dtype).view(torch.int16).item()) & 0xFFFF
    y = out if out is not None else _new(stream, count, dst_dtype, src.device)
    check(lib().ascq_ascend_antiquant_scalar(_ptr(y), dst_type, _ptr(src), src_type, bits(offset or 0.0), bits(scale),
                                             int(offset is not None), count, _stream(stream)), "ascend_antiquant_scalar")
    return y


def ascend_antiquant_policy(src: torch.Tensor, src_type: int, scale: torch.Tensor, scale_type: int, policy: int,
                            m: int, n: int, group_size: int = 0, offset=None, k_dim: int = 0,
                            is_transpose: bool = False, dst_dtype=torch.float16, out=None, stream=None):
    """AscendAntiQuant policy form (PER_TOKEN / PER_GROUP) over [m, n]: int8 / fp8 sources with f16 / bf16 / f32
    scales, fp4 E2M1 / E1M2 sources with E8M0 group scales.  Returns [m, n] of dst_dtype."""
    dst_type = _FLOAT_CODE[dst_dtype]
    y = out if out is not None else _new(stream, (m, n), dst_dtype, src.device)
    check(lib().ascq_ascend_antiquant_policy(_ptr(y), dst_type, _ptr(src), src_type, _ptr(scale), _ptr(offset),
                                             scale_type, policy, m, n, group_size, k_dim, int(is_transpose),
                                             _stream(stream)), "ascend_antiquant_policy")
    return y


# ------------------------------------------------------------------------------------------
# Quantize / Dequantize / AntiQuantize (quantize.h / dequantize.h / antiquantize.h)
# ------------------------------------------------------------------------------------------
def quantize(x: torch.Tensor, policy: int, dst_type: int = INT8, scale=None, offset=None, scale_scalar: float = 1.0,
             offset_scalar=None, scale_type: int | None = None, group_size: int = 0, kdim: int = 1,
             round_mode: int = ROUND_RINT, out=None, stream=None):
    """Quantize<{policy, hasOffset, roundMode, kDim}>(dst, x, scale, offset, {m, n, groupSize}) of x [m, n] in fp32
    arithmetic.  PER_TENSOR: scale_scalar / offset_scalar (values of scale_type); the other policies: `scale` (and
    `offset`, or offset_scalar) tensors.  Returns int8 (INT8) or uint8 codes [m, n] ([m, n / 2] for fp4)."""
    m, n = x.shape
    if scale_type is None:
        scale_type = _FLOAT_CODE[scale.dtype] if scale is not None else F32
    if out is not None:
        q = out
    elif dst_type in (FP4_E2M1, FP4_E1M2):
        q = _new(stream, (m, n // 2), torch.uint8, x.device)
    else:
        q = _new(stream, (m, n), torch.int8 if dst_type == INT8 else torch.uint8, x.device)
    has_off = offset is not None or offset_scalar is not None
    p = _QuantizeParam(policy, int(has_off), round_mode, kdim, m, n, group_size)
    check(lib().ascq_quantize(_ptr(q), dst_type, _ptr(x), _FLOAT_CODE[x.dtype], _ptr(scale), _ptr(offset),
                              float(scale_scalar), float(offset_scalar or 0.0), scale_type, ctypes.byref(p),
                              _stream(stream)), "quantize")
    return q


def dequantize(src: torch.Tensor, policy: int, dst_dtype=torch.float32, scale=None, scale_scalar: float = 1.0,
               scale_type: int | None = None, group_size: int = 0, kdim: int = 1, out=None, stream=None):
    """Dequantize<{policy, false, kDim}>(dst, src, scale, {m, n, groupSize}): dst = cast(f32(src) * scale) over src
    [m, n] int32 (PER_TOKEN / PER_GROUP: int32 or f32).  PER_TENSOR: scale_scalar; PER_CHANNEL: scale [n] (f32, bf16,
    or int64 holding uint64 words)."""
    m, n = src.shape
    src_type = {torch.int32: INT32, torch.float32: F32}[src.dtype]
    if scale_type is None:
        scale_type = F32 if scale is None else {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16,
                                                torch.int64: U64}[scale.dtype]
    y = out if out is not None else _new(stream, (m, n), dst_dtype, src.device)
    p = _QuantizeParam(policy, 0, ROUND_RINT, kdim, m, n, group_size)
    check(lib().ascq_dequantize(_ptr(y), _FLOAT_CODE[dst_dtype], _ptr(src), src_type, _ptr(scale), float(scale_scalar),
                                scale_type, ctypes.byref(p), _stream(stream)), "dequantize")
    return y


def antiquantize(src: torch.Tensor, src_type: int, policy: int, m: int, n: int, dst_dtype=torch.float16, scale=None,
                 offset=None, scale_scalar: float = 1.0, offset_scalar=None, scale_type: int | None = None,
                 group_size: int = 0, kdim: int = 1, out=None, stream=None):
    """AntiQuantize<{policy, hasOffset, kDim}>(dst, src, scale, offset, {m, n, groupSize}): dst = (src + offset) *
    scale in fp32, one cast, over [m, n] (int8 / hifloat8 / fp8 codes; fp4 [m, n / 2] bytes with E8M0 scales).
    PER_TENSOR: scale_scalar / offset_scalar (values of dst_dtype); the other policies: `scale` / `offset` tensors."""
    if scale_type is None:
        scale_type = _FLOAT_CODE[dst_dtype] if scale is None else {torch.float32: F32, torch.float16: F16,
                                                                   torch.bfloat16: BF16, torch.uint8: E8M0}[scale.dtype]
    y = out if out is not None else _new(stream, (m, n), dst_dtype, src.device)
    has_off = offset is not None or offset_scalar is not None
    p = _QuantizeParam(policy, int(has_off), ROUND_RINT, kdim, m, n, group_size)
    check(lib().ascq_antiquantize(_ptr(y), _FLOAT_CODE[dst_dtype], _ptr(src), src_type, _ptr(scale), _ptr(offset),
                                  float(scale_scalar), float(offset_scalar or 0.0), scale_type, ctypes.byref(p),
                                  _stream(stream)), "antiquantize")
    return y


# ------------------------------------------------------------------------------------------
# weight-only antiquant matmul
# ------------------------------------------------------------------------------------------
def weight_pack_size(w_type: int, k: int, n: int) -> int:
    sz = ctypes.c_size_t(0)
    check(lib().ascq_weight_pack_size(w_type, k, n, ctypes.byref(sz)), "weight_pack_size")
    return sz.value


def weight_pack(w: torch.Tensor, w_type: int, k: int, n: int, is_transpose: bool = False, out=None, stream=None):
    nbytes = weight_pack_size(w_type, k, n)
    wp = out if out is not None else _new(stream, (nbytes,), torch.uint8, w.device)
    check(lib().ascq_weight_pack(_ptr(wp), _ptr(w), w_type, k, n, int(is_transpose), _stream(stream)), "weight_pack")
    return wp


def antiquant_matmul(x: torch.Tensor, w_packed: torch.Tensor, w_type: int, scale: torch.Tensor, offset, group_size: int,
                     n: int, out=None, stream=None):
    m, k = x.shape
    y = out if out is not None else _new(stream, (m, n), torch.float16, x.device)
    check(lib().ascq_antiquant_matmul(_ptr(y), _ptr(x), _ptr(w_packed), w_type, _ptr(scale), _ptr(offset), group_size,
                                      m, n, k, _stream(stream)), "antiquant_matmul")
    return y


# ------------------------------------------------------------------------------------------
# quantized group matmul (MoE)
# ------------------------------------------------------------------------------------------
def quant_group_matmul(x: torch.Tensor, per_token_scale: torch.Tensor, w: torch.Tensor, scale: torch.Tensor,
                       group_list: torch.Tensor, list_type: int = 0, w_trans: bool = False,
                       out_dtype=torch.bfloat16, out=None, stream=None, activation: int = 0):
    """activation: ACT_NONE or ACT_FASTER_GELU (the reference sample's epilogue)"""
    m, k = x.shape
    g = scale.shape[0]
    n = scale.shape[1]
    out_type = {torch.bfloat16: BF16, torch.float16: F16}[out_dtype]
    y = out if out is not None else _new(stream, (m, n), out_dtype, x.device)
    check(lib().ascq_quant_group_matmul(_ptr(y), out_type, _ptr(x), _ptr(per_token_scale), _ptr(w), int(w_trans),
                                        _ptr(scale), _ptr(group_list), list_type, g, m, k, n, int(activation),
                                        _stream(stream)),
          "quant_group_matmul")
    return y


# ------------------------------------------------------------------------------------------
# a transformer block's operators around its products: norm, linear, routing, rows by expert
# ------------------------------------------------------------------------------------------
_CODE_TYPE = {torch.int8: INT8, torch.float8_e4m3fn: FP8_E4M3}
_CODE_DTYPE = {INT8: torch.int8, FP8_E4M3: torch.float8_e4m3fn}


def _refuse(what: str, message: str):
    raise AscqError(E_INVALID_ARG, f"{what}: {message}")


def _typed(what: str, name: str, t: torch.Tensor, table: dict) -> int:
    """the ascq_dtype of t; a type outside the table is refused"""
    code = table.get(t.dtype)
    if code is None:
        raise AscqError(E_UNSUPPORTED, f"{what}: {name} of type {t.dtype}")
    return code


def _pitch(what: str, name: str, t: torch.Tensor, shape: tuple, dtype) -> int:
    """The row pitch of t [rows, n], whose rows are contiguous (pitch at least n)."""
    if t.shape != shape or t.dtype is not dtype:
        _refuse(what, f"{name} must be {tuple(shape)} of {dtype}, not {tuple(t.shape)} of {t.dtype}")
    rows, n = shape
    ld, unit = t.stride()
    if (unit != 1 and n > 1) or (ld < n and rows > 1):
        _refuse(what, f"{name}: the elements of a row must be contiguous")
    return max(ld, n)  # (torch gives rows of a single one any stride)


def _dense(what: str, name: str, t: torch.Tensor, shape: tuple, dtype) -> None:
    if t.shape != shape or t.dtype is not dtype or not t.is_contiguous():
        _refuse(what, f"{name} must be a contiguous {tuple(shape)} tensor of {dtype}, not {tuple(t.shape)} of {t.dtype}")


def _same_device(what: str, *tensors) -> None:
    device = tensors[0].get_device()
    if device < 0:
        _refuse(what, "tensors on the CPU: there is no CPU path")
    for t in tensors:
        if t is not None and t.get_device() != device:
            _refuse(what, f"tensors on {tensors[0].device} and {t.device}")


def _at(t) -> int | None:
    return None if t is None else t.data_ptr()


def add_rms_norm_quant(x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-6, dst_type: int = INT8, residual=None,
                       residual_out=None, norm_out=None, out=None, scale_out=None, stream=None):
    """h = x + residual, RMS norm of h by gamma, 8-bit codes with one fp32 scale per row: returns (codes, scale, h), the
    codes int8 (INT8) or float8_e4m3fn (FP8_E4M3).  x [m, n] and residual f16 / bf16 / f32, rows contiguous at any pitch;
    residual_out may be x or residual (in place; without it h is a new tensor, and without a residual h is x);
    norm_out takes the unquantised norm."""
    what = "add_rms_norm_quant"
    if x.dim() != 2:
        _refuse(what, "x must be [m, n]")
    shape, dt = x.shape, x.dtype
    m, n = shape
    src_type = _typed(what, "x", x, _FLOAT_CODE)
    if dst_type not in _CODE_DTYPE:
        raise AscqError(E_UNSUPPORTED, f"{what}: dst_type {dst_type}")
    ldx, ldr, ldh = _pitch(what, "x", x, shape, dt), 0, 0
    _dense(what, "gamma", gamma, (n,), dt)
    h = x
    if residual is not None:
        ldr = _pitch(what, "residual", residual, shape, dt)
        h = residual_out if residual_out is not None else _new(stream, (m, n), dt, x.device)
        ldh = _pitch(what, "residual_out", h, shape, dt)
    elif residual_out is not None:
        _refuse(what, "residual_out needs a residual")
    if norm_out is not None:
        _dense(what, "norm_out", norm_out, shape, dt)
    q = out if out is not None else _new(stream, (m, n), _CODE_DTYPE[dst_type], x.device)
    _dense(what, "out", q, shape, _CODE_DTYPE[dst_type])
    s = scale_out if scale_out is not None else _new(stream, (m,), torch.float32, x.device)
    _dense(what, "scale_out", s, (m,), torch.float32)
    _same_device(what, x, gamma, residual, h, norm_out, q, s)
    if n == 0 and m > 0:  # (the library writes nothing; a row without elements is a row of zeros)
        with torch.cuda.stream(torch.cuda.ExternalStream(_stream(stream), x.device)):
            s.zero_()
        return q, s, h
    p = _NormQuantParam(m, n, ldx, ldr, ldh, src_type, dst_type, eps)
    check(lib().ascq_add_rms_norm_quant(_at(q), _at(s), _at(h) if residual is not None else None, _at(norm_out), _at(x),
                                        _at(residual), _at(gamma), ctypes.byref(p), _stream(stream)), what)
    return q, s, h


def quant_linear(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias=None,
                 activation: int = ACT_NONE, residual=None, w_trans: bool = True, out_dtype=torch.bfloat16, out=None,
                 workspace=None, stream=None):
    """y = cast(act((x @ W) * w_scale * x_scale[:, None] + bias) + residual) of int8 or float8_e4m3fn codes: x [m, k] with a
    scale per token (fp32 [m]), w [n, k] (w_trans) or [k, n] with a scale per channel (fp32 [n]), bias fp32 [n]; y f16,
    bf16 or f32 and residual of its type; rows at any pitch.  out may be the residual.  workspace: a uint8 tensor of
    quant_linear_workspace_size bytes; without one the call takes what it needs from torch's allocator."""
    what = "quant_linear"
    if x.dim() != 2 or w.dim() != 2:
        _refuse(what, "x and w must be matrices")
    m, k = x.shape
    n = w.shape[0] if w_trans else w.shape[1]
    code = _typed(what, "x", x, _CODE_TYPE)
    ldx, ldr = _pitch(what, "x", x, (m, k), x.dtype), 0
    ldw = _pitch(what, "w", w, (n, k) if w_trans else (k, n), x.dtype)
    y = out if out is not None else _new(stream, (m, n), out_dtype, x.device)
    out_type = _typed(what, "out", y, _FLOAT_CODE)
    ldy = _pitch(what, "out", y, (m, n), y.dtype)
    _dense(what, "x_scale", x_scale, (m,), torch.float32)
    _dense(what, "w_scale", w_scale, (n,), torch.float32)
    if bias is not None:
        _dense(what, "bias", bias, (n,), torch.float32)
    if residual is not None:
        ldr = _pitch(what, "residual", residual, (m, n), y.dtype)
    room = _room(what, workspace)
    _same_device(what, x, x_scale, w, w_scale, bias, residual, y, workspace)
    p = _LinearParam(m, n, k, ldx, ldw, ldr, ldy, code, out_type, int(w_trans), activation)
    if workspace is None:
        need = ctypes.c_size_t(0)
        check(lib().ascq_quant_linear_workspace_size(_at(x), _at(w), ctypes.byref(p), ctypes.byref(need)), what)
        if need.value:
            workspace, room = _new(stream, (need.value,), torch.uint8, x.device, private=True), need.value
    check(lib().ascq_quant_linear(_at(y), _at(x), _at(x_scale), _at(w), _at(w_scale), _at(bias), _at(residual),
                                  ctypes.byref(p), _at(workspace), room, _stream(stream)), what)
    return y


def _room(what: str, workspace) -> int:
    """The bytes of a workspace, which is one run of memory: what lies in a view's gaps is not the call's to write"""
    if workspace is None:
        return 0
    if not workspace.is_contiguous():
        _refuse(what, "the workspace must be contiguous")
    return workspace.numel() * workspace.element_size()


def quant_linear_workspace_size(x: torch.Tensor, w: torch.Tensor, w_trans: bool = True, out_dtype=torch.bfloat16) -> int:
    """Bytes of the workspace that quant_linear uses for these operands (0: none)"""
    what = "quant_linear_workspace_size"
    m, k = x.shape
    n = w.shape[0] if w_trans else w.shape[1]
    p = _LinearParam(m, n, k, _pitch(what, "x", x, (m, k), x.dtype),
                     _pitch(what, "w", w, (n, k) if w_trans else (k, n), x.dtype), 0, 0, _typed(what, "x", x, _CODE_TYPE),
                     _FLOAT_CODE[out_dtype], int(w_trans), ACT_NONE)
    need = ctypes.c_size_t(0)
    check(lib().ascq_quant_linear_workspace_size(_at(x), _at(w), ctypes.byref(p), ctypes.byref(need)), what)
    return need.value


class MoeRouting(NamedTuple):
    """What moe_route gives for tokens [T] of k choices among E experts."""
    weights: torch.Tensor  # f32 [T, k]
    experts: torch.Tensor  # int32 [T, k], -1: no choice
    slots: torch.Tensor    # int32 [T, k]: the choice's row, ordered by expert, then token; -1: none
    tokens: torch.Tensor   # int32 [T * k]: the token of each row; -1 behind the last
    counts: torch.Tensor   # int64 [E]: rows per expert, quant_group_matmul's group_list of list_type 1
    routed: torch.Tensor   # int64 [1]: tokens with a choice
    loss: torch.Tensor     # f32 [1]: the balance loss


def _check_routing(what: str, r: MoeRouting, t: int, e: int, k: int) -> None:
    _dense(what, "weights", r.weights, (t, k), torch.float32)
    _dense(what, "experts", r.experts, (t, k), torch.int32)
    _dense(what, "slots", r.slots, (t, k), torch.int32)
    _dense(what, "tokens", r.tokens, (t * k,), torch.int32)
    _dense(what, "counts", r.counts, (e,), torch.int64)
    _dense(what, "routed", r.routed, (1,), torch.int64)
    _dense(what, "loss", r.loss, (1,), torch.float32)


def moe_route(logits: torch.Tensor, top_k: int, renormalize: bool = True, out=None, workspace=None,
              stream=None) -> MoeRouting:
    """The top_k experts of each token by its logits [T, E] (f16 / bf16 / f32; -inf or NaN: masked), their softmax weights,
    the rows' order by expert, the rows per expert and the balance loss (see ascq_moe_route)."""
    what = "moe_route"
    if logits.dim() != 2:
        _refuse(what, "logits must be [tokens, experts]")
    t, e = logits.shape
    p = _RouteParam(t, e, _pitch(what, "logits", logits, (t, e), logits.dtype), _typed(what, "logits", logits, _FLOAT_CODE),
                    top_k, int(renormalize))
    need = ctypes.c_size_t(0)
    check(lib().ascq_moe_route_workspace_size(ctypes.byref(p), ctypes.byref(need)), what)
    r = out
    if r is None:
        new = lambda shape, dt: _new(stream, shape, dt, logits.device)  # noqa: E731
        r = MoeRouting(new((t, top_k), torch.float32), new((t, top_k), torch.int32), new((t, top_k), torch.int32),
                       new((t * top_k,), torch.int32), new((e,), torch.int64), new((1,), torch.int64),
                       new((1,), torch.float32))
    _check_routing(what, r, t, e, top_k)
    room = _room(what, workspace)
    _same_device(what, logits, *r, workspace)
    if workspace is None and need.value:
        workspace, room = _new(stream, (need.value,), torch.uint8, logits.device, private=True), need.value
    check(lib().ascq_moe_route(*map(_at, r), _at(logits), ctypes.byref(p), _at(workspace), room,
                               _stream(stream)), what)
    return r


def moe_route_grad(logits: torch.Tensor, weights: torch.Tensor, experts: torch.Tensor, counts: torch.Tensor,
                   routed: torch.Tensor, grad_weights=None, grad_loss=None, renormalize: bool = True, out=None, stream=None):
    """d / d logits of grad_loss * loss + (grad_weights * weights).sum(), with moe_route's outputs of the same logits;
    grad_weights f32 [T, k], grad_loss f32 [1].  Returns a tensor of the logits' type."""
    what = "moe_route_grad"
    if logits.dim() != 2 or weights.dim() != 2:
        _refuse(what, "logits must be [tokens, experts], weights [tokens, top_k]")
    t, e = logits.shape
    k = weights.shape[1]
    ld = _pitch(what, "logits", logits, (t, e), logits.dtype)
    _dense(what, "weights", weights, (t, k), torch.float32)
    _dense(what, "experts", experts, (t, k), torch.int32)
    _dense(what, "counts", counts, (e,), torch.int64)
    _dense(what, "routed", routed, (1,), torch.int64)
    if grad_weights is not None:
        _dense(what, "grad_weights", grad_weights, (t, k), torch.float32)
    if grad_loss is not None:
        _dense(what, "grad_loss", grad_loss, (1,), torch.float32)
    g = out if out is not None else _new(stream, (t, e), logits.dtype, logits.device)
    ldg = _pitch(what, "out", g, (t, e), logits.dtype)
    _same_device(what, logits, weights, experts, counts, routed, grad_weights, grad_loss, g)
    p = _RouteParam(t, e, ld, _typed(what, "logits", logits, _FLOAT_CODE), k, int(renormalize))
    check(lib().ascq_moe_route_grad(_at(g), ldg, _at(logits), _at(weights), _at(experts), _at(counts), _at(routed),
                                    _at(grad_weights), _at(grad_loss), ctypes.byref(p), _stream(stream)), what)
    return g


def moe_dispatch(x: torch.Tensor, x_scale, slots: torch.Tensor, tokens: torch.Tensor, out=None, scale_out=None,
                 stream=None):
    """Rows of x [T, n] (int8, float8_e4m3fn, f16, bf16 or f32) and their scales (fp32 [T] or None) in the experts' order of
    a MoeRouting's slots and tokens: returns (rows [T * k, n], scales [T * k] or None); rows of no token are 0."""
    what = "moe_dispatch"
    if x.dim() != 2 or slots.dim() != 2:
        _refuse(what, "x must be [tokens, n], slots [tokens, top_k]")
    t, n = x.shape
    k = slots.shape[1]
    code = _typed(what, "x", x, {**_CODE_TYPE, **_FLOAT_CODE})
    ldx = _pitch(what, "x", x, (t, n), x.dtype)
    _dense(what, "slots", slots, (t, k), torch.int32)
    _dense(what, "tokens", tokens, (t * k,), torch.int32)
    rows = out if out is not None else _new(stream, (t * k, n), x.dtype, x.device)
    _dense(what, "out", rows, (t * k, n), x.dtype)
    s = None
    if x_scale is not None:
        _dense(what, "x_scale", x_scale, (t,), torch.float32)
        s = scale_out if scale_out is not None else _new(stream, (t * k,), torch.float32, x.device)
        _dense(what, "scale_out", s, (t * k,), torch.float32)
    elif scale_out is not None:
        _refuse(what, "scale_out needs x_scale")
    _same_device(what, x, x_scale, slots, tokens, rows, s)
    p = _RowsParam(t, n, ldx, code, k)
    check(lib().ascq_moe_dispatch(_at(rows), _at(s), _at(x), _at(x_scale), _at(slots), _at(tokens), ctypes.byref(p),
                                  _stream(stream)), what)
    return rows, s


def moe_combine(y: torch.Tensor, slots: torch.Tensor, weights: torch.Tensor, residual=None, out=None, stream=None):
    """out[t] = sum_j weights[t, j] y[slots[t, j]] + residual[t], of y [T * k, n] f16 / bf16 / f32; out may be the residual"""
    what = "moe_combine"
    if y.dim() != 2 or slots.dim() != 2:
        _refuse(what, "y must be [tokens * top_k, n], slots [tokens, top_k]")
    t, k = slots.shape
    n = y.shape[1]
    code = _typed(what, "y", y, _FLOAT_CODE)
    _dense(what, "y", y, (t * k, n), y.dtype)
    _dense(what, "slots", slots, (t, k), torch.int32)
    _dense(what, "weights", weights, (t, k), torch.float32)
    if residual is not None:
        _dense(what, "residual", residual, (t, n), y.dtype)
    r = out if out is not None else _new(stream, (t, n), y.dtype, y.device)
    _dense(what, "out", r, (t, n), y.dtype)
    _same_device(what, y, slots, weights, residual, r)
    p = _RowsParam(t, n, 0, code, k)
    check(lib().ascq_moe_combine(_at(r), _at(y), _at(slots), _at(weights), _at(residual), ctypes.byref(p),
                                 _stream(stream)), what)
    return r


def moe_combine_grad(grad_out: torch.Tensor, y: torch.Tensor, slots: torch.Tensor, tokens: torch.Tensor,
                     weights: torch.Tensor, need_grad_y: bool = True, out=None, grad_y_out=None, stream=None):
    """moe_combine's gradients: (grad_weights f32 [T, k], grad_y [T * k, n] of y's type, or None without need_grad_y)"""
    what = "moe_combine_grad"
    if y.dim() != 2 or slots.dim() != 2:
        _refuse(what, "y must be [tokens * top_k, n], slots [tokens, top_k]")
    t, k = slots.shape
    n = y.shape[1]
    code = _typed(what, "y", y, _FLOAT_CODE)
    _dense(what, "y", y, (t * k, n), y.dtype)
    _dense(what, "grad_out", grad_out, (t, n), y.dtype)
    _dense(what, "slots", slots, (t, k), torch.int32)
    _dense(what, "tokens", tokens, (t * k,), torch.int32)
    _dense(what, "weights", weights, (t, k), torch.float32)
    dw = out if out is not None else _new(stream, (t, k), torch.float32, y.device)
    _dense(what, "out", dw, (t, k), torch.float32)
    dy = None
    if need_grad_y:
        dy = grad_y_out if grad_y_out is not None else _new(stream, (t * k, n), y.dtype, y.device)
        _dense(what, "grad_y_out", dy, (t * k, n), y.dtype)
    _same_device(what, y, grad_out, slots, tokens, weights, dw, dy)
    p = _RowsParam(t, n, 0, code, k)
    check(lib().ascq_moe_combine_grad(_at(dw), _at(dy), _at(grad_out), _at(y), _at(slots), _at(tokens), _at(weights),
                                      ctypes.byref(p), _stream(stream)), what)
    return dw, dy


# ------------------------------------------------------------------------------------------
# attention over the paged int4 key / value cache
# ------------------------------------------------------------------------------------------
class KvCache:
    """A paged key / value cache: int4 codes k, v (uint8 [pages, kv_heads, page_size, d / 2]) and f16 (scale, offset) pairs k_scale,
    v_scale ([pages, kv_heads, page_size, d / group, 2]); a page's elements are contiguous, pages at any pitch of 16 bytes.  A code
    stands for f16(code * scale + offset).  The tensors are checked here, once, and stay the cache's; iterating gives the four."""
    __slots__ = ("_tensors", "_c", "_ref", "_device")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        what = "KvCache"
        if k.dim() != 4 or k_scale.dim() != 5:
            _refuse(what, "codes must be [pages, kv_heads, page_size, d / 2], scales [pages, kv_heads, page_size, d / group, 2]")
        shape, pairs = k.shape, k_scale.shape
        groups = pairs[3]
        if pairs[:3] != shape[:3] or pairs[4] != 2 or groups < 1 or 2 * shape[3] % groups:
            _refuse(what, f"k_scale {tuple(pairs)} does not fit codes {tuple(shape)}")
        ld = _page_pitch(what, "k", k, shape, torch.uint8)
        ld_scale = _page_pitch(what, "k_scale", k_scale, pairs, torch.float16)
        if ld != _page_pitch(what, "v", v, shape, torch.uint8) or \
                ld_scale != _page_pitch(what, "v_scale", v_scale, pairs, torch.float16):
            _refuse(what, "keys and values must have one page pitch")
        self._device = k.get_device()
        for t in (v, k_scale, v_scale):
            if t.get_device() != self._device:
                _refuse(what, f"tensors on {k.device} and {t.device}")
        self._tensors = (k, v, k_scale, v_scale)
        self._c = _KvCache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), shape[0], ld, ld_scale, shape[1],
                           shape[2], 2 * shape[3], 2 * shape[3] // groups)
        self._ref = ctypes.byref(self._c)

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scale = property(lambda self: self._tensors[2])
    v_scale = property(lambda self: self._tensors[3])

    def __iter__(self):
        return iter(self._tensors)


def kv_cache(pages: int, kv_heads: int, page_size: int, d: int, group: int = 32, device="cuda") -> KvCache:
    """An empty cache (its memory is not set: what no query sees reaches no result)"""
    new = lambda shape, dt: torch.empty(shape, dtype=dt, device=device)  # noqa: E731
    code, scale = (pages, kv_heads, page_size, d // 2), (pages, kv_heads, page_size, d // group, 2)
    return KvCache(new(code, torch.uint8), new(code, torch.uint8), new(scale, torch.float16), new(scale, torch.float16))


def _page_pitch(what: str, name: str, t: torch.Tensor, shape, dtype) -> int:
    """elements from page to page of a pool whose pages are contiguous"""
    if t.shape != shape or t.dtype is not dtype:
        _refuse(what, f"{name} must be {tuple(shape)} of {dtype}, not {tuple(t.shape)} of {t.dtype}")
    if not t.is_contiguous() and not (t.shape[0] > 0 and t[0].is_contiguous()):
        _refuse(what, f"{name}: the elements of a page must be contiguous")
    if t.shape[0] > 1 and t.stride(0) == 0:
        _refuse(what, f"{name}: pages must lie apart")  # (to the library a pitch of 0 is a dense pool's)
    return t.stride(0) if t.shape[0] > 1 else 0


def _cache_arg(what: str, cache: KvCache, on: torch.Tensor) -> _KvCache:
    if cache._device != on.get_device():
        _refuse(what, f"the cache on {cache.k.device}, other tensors on {on.device}")
    return cache._c


def _heads_pitch(what: str, name: str, t: torch.Tensor, shape, dtype):
    """pitches of tokens and heads of t [tokens, heads, d], whose rows of d are contiguous"""
    if t.shape != shape or t.dtype is not dtype:
        _refuse(what, f"{name} must be {tuple(shape)} of {dtype}, not {tuple(t.shape)} of {t.dtype}")
    tokens, heads, d = shape
    ld, hd, unit = t.stride()
    if heads <= 1:
        hd = d  # (torch gives a single one any stride)
    if tokens <= 1:
        ld = max(heads, 1) * hd
    if unit != 1 or hd < d or ld < d:
        _refuse(what, f"{name}: the channels of a head must be contiguous, and rows apart")
    return ld, hd


def _sequences_arg(what: str, page_table: torch.Tensor, lengths: torch.Tensor, starts) -> _KvSequences:
    if page_table.dim() != 2:
        _refuse(what, "page_table must be [batch, pages]")
    batch, columns = page_table.shape
    ld = _pitch(what, "page_table", page_table, page_table.shape, torch.int32)
    _dense(what, "lengths", lengths, (batch,), torch.int32)
    if starts is not None:
        _dense(what, "starts", starts, (batch + 1,), torch.int32)
    return _KvSequences(page_table.data_ptr(), lengths.data_ptr(), _at(starts), ld, batch, columns)


_QUERY_CODE = {torch.float16: F16, torch.bfloat16: BF16}


def _queries_arg(what: str, q: torch.Tensor, c: _KvCache, starts, max_queries, scale, causal, window) -> _KvAttentionParam:
    if q.dim() != 3 or q.shape[2] != c.d:
        _refuse(what, f"q must be [tokens, heads, {c.d}]")
    code = _typed(what, "q", q, _QUERY_CODE)
    ld, hd = _heads_pitch(what, "q", q, q.shape, q.dtype)
    tokens, heads, d = q.shape
    if starts is None:
        max_queries = 1
    elif max_queries is None:
        max_queries = tokens
    return _KvAttentionParam(tokens, max_queries, ld, hd, 0, 0, window, code, heads, int(causal),
                             d ** -0.5 if scale is None else scale)


def kv_append(cache: KvCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, stream=None) -> None:
    """Quantises rows k, v [tokens, kv_heads, d] (f16 / bf16 / f32; tokens and heads at any pitch, so slices of a fused projection
    too) into the cache: token t to row slots[t] % page_size of page slots[t] // page_size (int64; a slot outside the cache, -1 for
    padding, is not written; slots are distinct)."""
    what = "kv_append"
    c = _cache_arg(what, cache, k)
    if k.dim() != 3:
        _refuse(what, "k must be [tokens, kv_heads, d]")
    t = k.shape[0]
    shape = (t, c.kv_heads, c.d)
    code = _typed(what, "k", k, _FLOAT_CODE)
    ldk, hdk = _heads_pitch(what, "k", k, shape, k.dtype)
    ldv, hdv = _heads_pitch(what, "v", v, shape, k.dtype)
    _dense(what, "slots", slots, (t,), torch.int64)
    _same_device(what, k, v, slots)
    p = _KvAppendParam(t, ldk, hdk, ldv, hdv, code)
    check(lib().ascq_kv_append(cache._ref, _at(k), _at(v), _at(slots), ctypes.byref(p), _stream(stream)), what)


def kv_attention(q: torch.Tensor, cache: KvCache, page_table: torch.Tensor, lengths: torch.Tensor, starts=None, max_queries=None,
                 scale=None, causal: bool = True, window: int = 0, need_lse: bool = False, out=None, lse=None, workspace=None,
                 stream=None):
    """softmax(scale q k^T) v over the cached tokens of each sequence: q [tokens, heads, d] (f16 / bf16, tokens and heads at any
    pitch), page_table int32 [batch, pages], lengths int32 [batch] (tokens cached, the queries' own among them).  starts int32
    [batch + 1]: sequence b has the queries starts[b] .. starts[b + 1] - 1 (max_queries at most; give it, the launch is sized by it);
    None: one each.  A query sees the tokens up to its own (causal) and, with window, no more than that many.  scale: 1 / sqrt(d)
    if None.  Returns (out, lse): lse f32 [tokens, heads] when need_lse or a tensor for it is given, else None; rows of no sequence
    are left as they were.  A table narrowed to the longest sequence's pages (page_table[:, :n]) makes the launch smaller.
    workspace: a uint8 tensor of kv_attention_workspace_size bytes; without one the call takes it from torch's allocator."""
    what = "kv_attention"
    c = _cache_arg(what, cache, q)
    s = _sequences_arg(what, page_table, lengths, starts)
    p = _queries_arg(what, q, c, starts, max_queries, scale, causal, window)
    o = out if out is not None else _new(stream, q.shape, q.dtype, q.device)
    p.ld_out, p.hd_out = _heads_pitch(what, "out", o, q.shape, q.dtype)
    if lse is None and need_lse:
        lse = _new(stream, q.shape[:2], torch.float32, q.device)
    if lse is not None:
        _dense(what, "lse", lse, q.shape[:2], torch.float32)
    room = _room(what, workspace)
    _same_device(what, q, page_table, lengths, starts, o, lse, workspace)
    if workspace is None:
        need = ctypes.c_size_t(0)
        check(lib().ascq_kv_attention_workspace_size(cache._ref, ctypes.byref(s), ctypes.byref(p), ctypes.byref(need)), what)
        if need.value:
            workspace, room = _new(stream, (need.value,), torch.uint8, q.device, private=True), need.value
    check(lib().ascq_kv_attention(_at(o), _at(lse), _at(q), cache._ref, ctypes.byref(s), ctypes.byref(p), _at(workspace), room,
                                  _stream(stream)), what)
    return o, lse


def kv_attention_workspace_size(q: torch.Tensor, cache: KvCache, page_table: torch.Tensor, starts=None, max_queries=None,
                                causal: bool = True, window: int = 0) -> int:
    """Bytes of the workspace that kv_attention uses for such a call (0: none)"""
    what = "kv_attention_workspace_size"
    c = _cache_arg(what, cache, q)
    if page_table.dim() != 2:
        _refuse(what, "page_table must be [batch, pages]")
    # (sizes alone are read: any address does for the lengths, and a table without columns has none)
    s = _KvSequences(page_table.data_ptr(), c.k, _at(starts), 0, *page_table.shape)
    p = _queries_arg(what, q, c, starts, max_queries, None, causal, window)
    need = ctypes.c_size_t(0)
    check(lib().ascq_kv_attention_workspace_size(cache._ref, ctypes.byref(s), ctypes.byref(p), ctypes.byref(need)), what)
    return need.value


def kv_weights(q: torch.Tensor, lse: torch.Tensor, cache: KvCache, page_table: torch.Tensor, lengths: torch.Tensor, weights=None,
               decay: float = 1.0, starts=None, max_queries=None, scale=None, causal: bool = True, window: int = 0, out=None,
               stream=None) -> torch.Tensor:
    """The attention each cached token received from these queries, summed over them and over the heads of its key head, on top of
    decay * weights: f32 [batch, kv_heads, cap], cap at least the page table's tokens.  lse as kv_attention returns it for the same
    arguments.  out may be weights; positions from a sequence's length on stay as they were, or, without weights, are zeros."""
    what = "kv_weights"
    c = _cache_arg(what, cache, q)
    s = _sequences_arg(what, page_table, lengths, starts)
    p = _queries_arg(what, q, c, starts, max_queries, scale, causal, window)
    _dense(what, "lse", lse, q.shape[:2], torch.float32)
    cap = s.table_pages * c.page_size
    for t in (weights, out):
        if t is not None and t.dim() == 3:
            cap = t.shape[2]
    shape = (s.batch, c.kv_heads, cap)
    if weights is not None:
        _dense(what, "weights", weights, shape, torch.float32)
    if out is not None:
        _dense(what, "out", out, shape, torch.float32)
    _same_device(what, q, lse, page_table, lengths, starts, weights, out)
    w = out
    if w is None:
        # (positions that the call leaves as they were hold what they held)
        w = _new(stream, shape, torch.float32, q.device)
        if weights is not None:
            with torch.cuda.stream(torch.cuda.ExternalStream(_stream(stream), q.device)):
                w.copy_(weights)
    check(lib().ascq_kv_weights(_at(w), _at(weights), cap, decay, _at(q), _at(lse), cache._ref, ctypes.byref(s), ctypes.byref(p),
                                _stream(stream)), what)
    return w


def kv_evict(cache: KvCache, page_table: torch.Tensor, lengths: torch.Tensor, weights: torch.Tensor, keep: int, recent: int = 0,
             into=None, kept=None, lengths_out=None, weights_out=None, workspace=None, stream=None):
    """Cuts every sequence to its `keep` tokens of most weight (f32 [batch, kv_heads, cap], see kv_weights), the last `recent` always
    among them, per key head.  They move in order to the sequence's first places: in its own pages, which no other sequence shares
    then, or in the pages into (int32 [batch, n], none of page_table's), the old ones staying as they are.  Returns (kept, lengths,
    weights): kept int32 [batch, kv_heads, keep], the tokens' former positions, -1 behind the last; the new lengths, a tensor of their
    own; the kept tokens' weights, zeros behind them, in weights itself unless weights_out [batch, kv_heads, n] is given.
    workspace: a uint8 tensor of kv_evict_workspace_size bytes; without one the call takes it from torch's allocator."""
    what = "kv_evict"
    c = _cache_arg(what, cache, weights)
    s = _sequences_arg(what, page_table, lengths, None)
    if weights.dim() != 3:
        _refuse(what, "weights must be [batch, kv_heads, cap]")
    if not 0 <= recent <= keep or not 1 <= keep < 1 << 31:  # (here: the library's fields would hold the low 32 bits)
        _refuse(what, "0 <= recent <= keep, and keep at least 1 and below 2^31")
    heads = (s.batch, c.kv_heads)
    _dense(what, "weights", weights, (*heads, weights.shape[2]), torch.float32)
    w = weights if weights_out is None else weights_out
    if w.dim() != 3:
        _refuse(what, "weights_out must be [batch, kv_heads, n]")
    _dense(what, "weights_out", w, (*heads, w.shape[2]), torch.float32)
    ld_into = columns = 0
    if into is not None:
        if into.dim() != 2:
            _refuse(what, "into must be [batch, pages]")
        columns = into.shape[1]
        ld_into = _pitch(what, "into", into, (s.batch, columns), torch.int32)
    at = kept if kept is not None else _new(stream, (*heads, keep), torch.int32, weights.device)
    _dense(what, "kept", at, (*heads, keep), torch.int32)
    n = lengths_out if lengths_out is not None else _new(stream, (s.batch,), torch.int32, weights.device)
    _dense(what, "lengths_out", n, (s.batch,), torch.int32)
    room = _room(what, workspace)
    _same_device(what, weights, page_table, lengths, into, at, n, w, workspace)
    p = _KvEvictParam(weights.shape[2], w.shape[2], ld_into, keep, recent, columns)
    if workspace is None:
        need = ctypes.c_size_t(0)
        check(lib().ascq_kv_evict_workspace_size(cache._ref, ctypes.byref(s), ctypes.byref(need)), what)
        if need.value:
            workspace, room = _new(stream, (need.value,), torch.uint8, weights.device, private=True), need.value
    check(lib().ascq_kv_evict(_at(at), _at(n), _at(w), _at(weights), _at(into), cache._ref, ctypes.byref(s), ctypes.byref(p),
                              _at(workspace), room, _stream(stream)), what)
    return at, n, w


def kv_evict_workspace_size(cache: KvCache, page_table: torch.Tensor) -> int:
    """Bytes of the workspace that kv_evict uses for such a call (0: none)"""
    what = "kv_evict_workspace_size"
    c = _cache_arg(what, cache, page_table)
    if page_table.dim() != 2:
        _refuse(what, "page_table must be [batch, pages]")
    s = _KvSequences(page_table.data_ptr(), c.k, None, 0, *page_table.shape)  # (any address, as above)
    need = ctypes.c_size_t(0)
    check(lib().ascq_kv_evict_workspace_size(cache._ref, ctypes.byref(s), ctypes.byref(need)), what)
    return need.value


# ------------------------------------------------------------------------------------------
# NZ fractal <-> ND
# ------------------------------------------------------------------------------------------
def nz_size(dtype: int, batch: int, rows: int, cols: int) -> int:
    return int(lib().ascq_nz_size(dtype, batch, rows, cols))


def nz_to_nd(src: torch.Tensor, dtype: int, batch: int, rows: int, cols: int, transpose_out: bool = False, out=None,
             stream=None):
    """NZ bytes -> ND [batch, rows, cols] (transpose_out: [batch, cols, rows]) as a uint8 tensor of that shape
    times the element size"""
    esize = {INT8: 1, UINT8: 1, FP8_E4M3: 1, FP8_E5M2: 1, F16: 2, BF16: 2, INT32: 4, F32: 4}[dtype]
    shape = (batch, cols, rows * esize) if transpose_out else (batch, rows, cols * esize)
    y = out if out is not None else _new(stream, shape, torch.uint8, src.device)
    check(lib().ascq_nz_to_nd(_ptr(y), _ptr(src), dtype, batch, rows, cols, int(transpose_out), _stream(stream)),
          "nz_to_nd")
    return y


def nd_to_nz(src: torch.Tensor, dtype: int, batch: int, rows: int, cols: int, out=None, stream=None):
    y = out if out is not None else _new(stream, nz_size(dtype, batch, rows, cols), torch.uint8, src.device)
    check(lib().ascq_nd_to_nz(_ptr(y), _ptr(src), dtype, batch, rows, cols, _stream(stream)), "nd_to_nz")
    return y


# ------------------------------------------------------------------------------------------
# Matmul handle (mirrors AscendC::Matmul's call sequence)
# ------------------------------------------------------------------------------------------
class Matmul:
    """Matmul<A, B, C, Bias> handle: SetOrgShape / SetTensorA / SetTensorB / SetBias / SetQuant* /
    SetAntiQuant* / SetTensorScaleA/B / IterateAll / End, each a call into the C ABI."""

    def __init__(self, a_type: int, b_type: int, c_type: int, bias_type: int = 0, scale_type: int = 0,
                 b_format: int = FORMAT_ND):
        self._h = ctypes.c_void_p()
        t = _MatmulTypes(a_type, b_type, c_type, bias_type, scale_type, b_format)
        check(lib().ascq_matmul_create(ctypes.byref(t), ctypes.byref(self._h)), "matmul_create")
        self._keep = []

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value and _lib is not None:
            _lib.ascq_matmul_destroy(h)
            self._h = None

    def Init(self, tiling: CubeTiling):
        check(lib().ascq_matmul_init(self._h, ctypes.byref(tiling)), "Init")

    def SetOrgShape(self, m: int, n: int, k: int):
        check(lib().ascq_matmul_set_org_shape(self._h, m, n, k), "SetOrgShape")

    def SetSingleShape(self, m: int, n: int, k: int):
        check(lib().ascq_matmul_set_single_shape(self._h, m, n, k), "SetSingleShape")

    def SetTail(self, m: int = -1, n: int = -1, k: int = -1):
        check(lib().ascq_matmul_set_tail(self._h, m, n, k), "SetTail")

    def SetTensorA(self, a, is_transpose_a: bool = False):
        self._keep.append(a)
        check(lib().ascq_matmul_set_tensor_a(self._h, _ptr(a), int(is_transpose_a)), "SetTensorA")

    def SetTensorB(self, b, is_transpose_b: bool = False):
        self._keep.append(b)
        check(lib().ascq_matmul_set_tensor_b(self._h, _ptr(b), int(is_transpose_b)), "SetTensorB")

    def SetBias(self, bias):
        self._keep.append(bias)
        check(lib().ascq_matmul_set_bias(self._h, _ptr(bias)), "SetBias")

    def DisableBias(self):
        check(lib().ascq_matmul_disable_bias(self._h), "DisableBias")

    def SetQuantScalar(self, word: int):
        check(lib().ascq_matmul_set_quant_scalar(self._h, word & 0xFFFFFFFFFFFFFFFF), "SetQuantScalar")

    def SetQuantVector(self, words: torch.Tensor):
        self._keep.append(words)
        check(lib().ascq_matmul_set_quant_vector(self._h, _ptr(words)), "SetQuantVector")

    def SetAntiQuantScalar(self, offset: float, scale: float):
        check(lib().ascq_matmul_set_antiquant_scalar(self._h, _half_bits(offset), _half_bits(scale)),
              "SetAntiQuantScalar")

    def SetAntiQuantVector(self, offset, scale, group_size: int = 0):
        self._keep += [offset, scale]
        check(lib().ascq_matmul_set_antiquant_vector(self._h, _ptr(offset), _ptr(scale), group_size),
              "SetAntiQuantVector")

    def SetTensorScaleA(self, s, is_transpose_scale_a: bool = False):
        self._keep.append(s)
        check(lib().ascq_matmul_set_tensor_scale_a(self._h, _ptr(s), int(is_transpose_scale_a)), "SetTensorScaleA")

    def SetTensorScaleB(self, s, is_transpose_scale_b: bool = True):
        self._keep.append(s)
        check(lib().ascq_matmul_set_tensor_scale_b(self._h, _ptr(s), int(is_transpose_scale_b)), "SetTensorScaleB")

    def WorkspaceSize(self) -> int:
        sz = ctypes.c_size_t(0)
        check(lib().ascq_matmul_workspace_size(self._h, ctypes.byref(sz)), "WorkspaceSize")
        return sz.value

    def SetWorkspace(self, ws, nbytes: int):
        self._keep.append(ws)
        check(lib().ascq_matmul_set_workspace(self._h, _ptr(ws), nbytes), "SetWorkspace")

    def IterateAll(self, c, en_atomic: int = 0, stream=None):
        check(lib().ascq_matmul_iterate_all(self._h, _ptr(c), en_atomic, _stream(stream)), "IterateAll")

    def IterateAllNoAlloc(self, c, en_atomic: int = 0, stream=None):
        """IterateAll with the workspace taken from the library's static per-device scratch (allocates nothing)"""
        check(lib().ascq_matmul_iterate_all_noalloc(self._h, _ptr(c), en_atomic, _stream(stream)), "IterateAllNoAlloc")

    def End(self):
        check(lib().ascq_matmul_end(self._h), "End")
        self._keep = []
