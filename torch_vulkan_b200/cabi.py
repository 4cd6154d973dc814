"""ctypes bindings of the C ABI in include/tvb200.h (lib/libtvb200.so).

This is the same boundary the C++ ATen layer binds; tests and the benchmark
call through it directly with device pointers (for example those of
torch.cuda tensors). There is no fallback: if the library was not built, or
no B200 is present, the calls raise.
"""

import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libtvb200.so")

F32, F16, BF16, E4M3, E5M2, I8, U8, I32, I64, F64, BOOL, I16, E4M3FNUZ, E5M2FNUZ = range(14)

_c = ctypes
_vp, _i, _i64, _u64, _u32 = _c.c_void_p, _c.c_int, _c.c_int64, _c.c_uint64, _c.c_uint32


class TvbAlloc(ctypes.Structure):
    _fields_ = [("handle", _vp), ("ptr", _vp), ("size", _u64), ("device", _c.c_int32), ("pad", _c.c_int32)]


class TvbChainItem(ctypes.Structure):
    _fields_ = [("a", _vp), ("a_sm", _i64), ("b", _vp), ("scales", _vp), ("c_ranks", _c.POINTER(_vp)), ("m", _i64),
                ("n_local", _i64), ("k", _i64), ("independent", _c.c_int32), ("reserved", _c.c_int32)]


class TvbGroupItem(ctypes.Structure):
    _fields_ = [("a", _vp), ("a_sm", _i64), ("b", _vp), ("scales", _vp), ("c_ranks", _c.POINTER(_vp)), ("m", _i64), ("c_host", _vp)]


# name -> (restype, argtypes): every entry point include/tvb200.h declares
SIGNATURES = {
    "tvb_last_error": (_c.c_char_p, []),
    "tvb_device_count": (_i, []),
    "tvb_set_device": (_i, [_i]),
    "tvb_current_device": (_i, []),
    "tvb_device_name": (_i, [_i, _c.c_char_p, _c.c_size_t]),
    "tvb_capabilities": (_u32, [_i]),
    "tvb_alloc": (_i, [_i, _u64, _c.POINTER(TvbAlloc)]),
    "tvb_free": (None, [_vp]),
    "tvb_synchronize": (_i, [_i]),
    "tvb_empty_cache": (_i, [_i]),
    "tvb_memory_stats": (None, [_i, _c.POINTER(_u64), _c.POINTER(_u64), _c.POINTER(_u64)]),
    "tvb_stream": (_vp, [_i]),
    "tvb_set_stream": (_i, [_i, _vp]),
    "tvb_dispatch_count": (_u64, []),
    "tvb_shutdown": (None, []),
    "tvb_host_alloc": (_i, [_u64, _c.POINTER(_vp)]),
    "tvb_host_free": (None, [_vp]),
    "tvb_host_is_pinned": (_i, [_vp]),
    "tvb_host_register": (_i, [_vp, _u64, _c.POINTER(_vp)]),
    "tvb_host_unregister": (_i, [_vp]),
    "tvb_memcpy_h2d": (_i, [_i, _vp, _vp, _u64]),
    "tvb_memcpy_d2h": (_i, [_i, _vp, _vp, _u64]),
    "tvb_memcpy_d2d": (_i, [_i, _vp, _vp, _u64]),
    "tvb_memcpy_d2h_async": (_i, [_i, _vp, _vp, _u64]),
    "tvb_memcpy_d2h_overlapped": (_i, [_i, _vp, _vp, _u64]),
    "tvb_join_copies": (_i, [_i]),
    "tvb_copy_strided": (_i, [_i, _vp, _i, _c.POINTER(_i64), _vp, _i, _c.POINTER(_i64), _c.POINTER(_i64), _i]),
    "tvb_fill_strided": (_i, [_i, _vp, _i, _u64, _c.POINTER(_i64), _c.POINTER(_i64), _i]),
    "tvb_add_rowvec": (_i, [_i, _vp, _i, _i64, _vp, _i, _i64, _i64]),
    "tvb_qmm8_widened_bytes": (_u64, [_i64, _i64]),
    "tvb_qmm8_widen": (_i, [_i, _vp, _vp, _i, _i64, _i64, _vp, _u64]),
    "tvb_qmm8_widened": (_i, [_i, _vp, _i, _i64, _vp, _vp, _i64, _i64, _i64]),
    "tvb_mm": (_i, [_i, _vp, _i, _i64, _i64, _vp, _i64, _i64, _vp, _i, _vp, _i, _i64, _i64, _i64, _i]),
    "tvb_addmm": (_i, [_i, _vp, _i, _i64, _i64, _vp, _i64, _i64, _vp, _i, _vp, _i, _i64, _vp, _i, _i64, _i64, _i64, _i]),
    "tvb_qmm8": (_i, [_i, _vp, _i, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _i]),
    "tvb_qmm8_linear": (_i, [_i, _vp, _i, _i64, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64]),
    "tvb_qmm8_gather": (_i, [_i, _vp, _i, _i64, _vp, _vp, _c.POINTER(_vp), _c.POINTER(_vp), _i, _i, _vp, _i, _i64, _i64, _i64]),
    "tvb_wait_flags": (_i, [_i, _vp, _i, _vp]),
    "tvb_set_wait_limit_ms": (_i, [_i]),
    "tvb_qmm8_group": (_i, [_i, _i, _c.POINTER(TvbGroupItem), _i, _i64, _i64]),
    "tvb_qmm8_group_gather": (_i, [_i, _i, _c.POINTER(TvbGroupItem), _i, _c.POINTER(_vp), _i, _i, _vp, _i, _i64, _i64]),
    "tvb_qmm8_chain_create": (_i, [_i, _i, _c.POINTER(TvbChainItem), _i, _c.POINTER(_vp), _i, _i, _vp, _i, _c.POINTER(_vp)]),
    "tvb_qmm8_chain_run": (_i, [_i, _vp]),
    "tvb_qmm8_chain_destroy": (None, [_vp]),
    "tvb_comm_unique_id": (_i, [_c.c_char_p]),
    "tvb_comm_init_rank": (_i, [_i, _c.c_char_p, _i, _i, _i, _c.POINTER(_vp)]),
    "tvb_comm_init_all": (_i, [_c.POINTER(_i), _i, _c.POINTER(_vp)]),
    "tvb_all_gather": (_i, [_vp, _vp, _vp, _u64]),
    "tvb_all_gather_columns": (_i, [_vp, _vp, _vp, _i, _i64, _i64]),
    "tvb_comm_wait": (_i, [_vp, _i]),
    "tvb_comm_abort": (_i, [_vp]),
    "tvb_comm_destroy": (_i, [_vp]),
    "tvb_graph_begin": (_i, [_i]),
    "tvb_graph_end": (_i, [_i, _c.POINTER(_vp)]),
    "tvb_graph_launch": (_i, [_i, _vp]),
    "tvb_graph_destroy": (None, [_vp]),
    "tvb_ipc_export": (_i, [_i, _vp, _c.c_char_p, _c.POINTER(_u64)]),
    "tvb_ipc_import": (_i, [_i, _c.c_char_p, _u64, _c.POINTER(_vp)]),
    "tvb_qmm8_static_scratch": (_i, [_i, _vp, _i, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _vp]),
    "tvb_qmm8_static_scratch_status": (_i, [_i, _vp, _c.POINTER(_i)]),
    "tvb_qmm4_pack": (_i, [_i, _vp, _i64, _vp, _i, _i64, _vp, _i, _i64, _vp]),
    "tvb_qmm4_quantize": (_i, [_i, _vp, _i, _i64, _i64, _i, _vp, _vp, _vp]),
    "tvb_qmm4_matmul": (_i, [_i, _vp, _vp, _vp, _vp, _i, _vp, _i, _i64, _i64, _i64, _i64, _vp]),
    "tvb_qmm4_workspace_bytes": (_u64, [_i64, _i64]),
    "tvb_qmm4": (_i, [_i, _vp, _i, _vp, _i, _vp, _i64, _i64, _i64, _i64, _vp, _u64]),
    "tvb_qmm4_prepared_bytes": (_u64, [_i64, _i64]),
    "tvb_qmm4_prepare": (_i, [_i, _vp, _i64, _i64, _i64, _vp, _u64]),
    "tvb_qmm4_tc_workspace_bytes": (_u64, [_i64, _i64]),
    "tvb_qmm4_decode_usable": (_i, [_i64, _i64, _i64, _i64]),
    "tvb_qmm4_decode_prepared_bytes": (_u64, [_i64, _i64, _i64]),
    "tvb_qmm4_decode_prepare": (_i, [_i, _vp, _i64, _i64, _i64, _vp, _u64]),
    "tvb_qmm4_decode_workspace_bytes": (_u64, [_i64, _i64]),
    "tvb_qmm4_decode": (_i, [_i, _vp, _i, _vp, _i, _vp, _vp, _i64, _i64, _i64, _i64, _vp, _u64]),
    "tvb_qmm4_tc": (_i, [_i, _vp, _i, _vp, _i, _vp, _vp, _i64, _i64, _i64, _i64, _vp, _u64]),
    "tvb_qmm4_prepared16_bytes": (_u64, [_i64, _i64]),
    "tvb_qmm4_prepare16": (_i, [_i, _vp, _i64, _i64, _i64, _vp, _u64]),
    "tvb_qmm4_tc16_workspace_bytes": (_u64, [_i64, _i64]),
    "tvb_qmm4_tc16": (_i, [_i, _vp, _i, _vp, _i, _vp, _vp, _i64, _i64, _i64, _i64, _vp, _u64]),
    "tvb_qmm4_fast_prepared_bytes": (_u64, [_i64, _i64]),
    "tvb_qmm4_fast_prepare": (_i, [_i, _vp, _i64, _i64, _i64, _vp, _u64, _c.POINTER(_i)]),
    "tvb_qmm4_fast_workspace_bytes": (_u64, [_i64, _i64]),
    "tvb_qmm4_fast": (_i, [_i, _vp, _i, _vp, _i, _vp, _vp, _i64, _i64, _i64, _i64, _vp, _u64]),
    "tvb_scaled_mm_gather": (_i, [_i, _vp, _i, _i64, _i64, _vp, _i, _i64, _i64, _vp, _vp, _i, _vp, _i, _vp, _c.POINTER(_vp), _i,
                                  _c.POINTER(_vp), _i, _i, _vp, _i, _i64, _i64, _i64]),
    "tvb_scaled_mm": (_i, [_i, _vp, _i, _i64, _i64, _vp, _i, _i64, _i64, _vp, _vp, _i, _vp, _i, _vp, _vp, _i, _i64, _i64,
                           _i64, _i]),
    "tvb_linear_workspace_bytes": (_u64, [_i, _vp, _i64, _vp, _i64, _i64, _i64, _i64]),
    "tvb_linear": (_i, [_i, _vp, _i, _i64, _vp, _i64, _vp, _i, _vp, _i64, _vp, _vp, _i64, _i64, _i64, _vp, _u64]),
    "tvb_linear_backward_workspace_bytes": (_u64, [_i, _vp, _i64, _vp, _i64, _vp, _i64, _i, _i, _i64, _i64, _i64]),
    "tvb_linear_backward": (_i, [_i, _vp, _i, _i64, _vp, _vp, _i64, _vp, _i64, _i, _vp, _vp, _vp, _i64, _i64, _i64, _vp, _u64]),
    "tvb_layer_norm": (_i, [_i, _vp, _i, _i64, _vp, _vp, _i, _c.c_float, _vp, _vp, _vp, _i64, _i64]),
    "tvb_layer_norm_backward_workspace_bytes": (_u64, [_i64, _i64]),
    "tvb_layer_norm_backward": (_i, [_i, _vp, _i, _i64, _vp, _i64, _vp, _vp, _vp, _i, _vp, _vp, _vp, _i64, _i64, _vp, _u64]),
}

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}  # TvbActivation
WANT_DX, WANT_DW, WANT_DB = 1, 2, 4  # TvbWant

_lib = None


def lib():
    """The loaded library; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with `python -m torch_vulkan_b200._build` "
                               "(there is no fallback without the CUDA library)")
        _lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(_lib, name)
            fn.restype = res
            fn.argtypes = args
    return _lib


class TvbError(RuntimeError):
    pass


def check(rc):
    if rc != 0:
        raise TvbError(lib().tvb_last_error().decode("utf-8", "replace"))


def _dtype_code(dtype):
    import torch

    return {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16, torch.float8_e4m3fn: E4M3, torch.float8_e5m2: E5M2,
            torch.int8: I8, torch.uint8: U8, torch.int32: I32, torch.int64: I64, torch.float64: F64, torch.bool: BOOL,
            torch.int16: I16, torch.float8_e4m3fnuz: E4M3FNUZ, torch.float8_e5m2fnuz: E5M2FNUZ}[dtype]


def _ptr(t):
    return _vp(t.data_ptr()) if t is not None else _vp(0)


def _dev(t):
    return t.device.index if t.device.index is not None else 0


def synchronize(device=0):
    check(lib().tvb_synchronize(device))


# ---- op-level wrappers over device tensors (torch.cuda tensors or any tensor whose data_ptr is a device pointer)

def qmm8(a, b, scales, variant=0):
    """tvb_qmm8 on device tensors: A [m, k] (last dim contiguous), int8 B [n, k], scales [n] in A's dtype."""
    import torch

    m, k = a.shape
    n = b.shape[0]
    assert scales.dtype == a.dtype and b.dtype == torch.int8 and b.is_contiguous()
    c = torch.empty((m, n), dtype=a.dtype, device=a.device)
    check(lib().tvb_qmm8(_dev(a), _ptr(a), _dtype_code(a.dtype), a.stride(0), _ptr(b), _ptr(scales), _ptr(c), m, n, k, variant))
    return c


def qmm8_linear(a, b, scales, bias=None, residual=None, out=None):
    """tvb_qmm8_linear on device tensors: the product of `qmm8`, + bias [n], + residual [m, n] (A's dtype; either may be None).
    `out` may be the residual itself where the decode kernel runs (at most 32 rows)."""
    import torch

    m, k = a.shape
    n = b.shape[0]
    assert scales.dtype == a.dtype and b.dtype == torch.int8 and b.is_contiguous()
    assert bias is None or (bias.dtype == a.dtype and bias.shape == (n,) and bias.is_contiguous())
    assert residual is None or (residual.dtype == a.dtype and residual.shape == (m, n) and residual.is_contiguous())
    c = torch.empty((m, n), dtype=a.dtype, device=a.device) if out is None else out
    check(lib().tvb_qmm8_linear(_dev(a), _ptr(a), _dtype_code(a.dtype), a.stride(0), _ptr(b), _ptr(scales), _ptr(bias),
                                _ptr(residual), _ptr(c), m, n, k))
    return c


def qmm4_pack(weights, scales, bias):
    import torch

    w = weights.contiguous().reshape(-1)
    s = scales.contiguous().reshape(-1)
    nb = 0 if bias is None else bias.numel()
    bvec = None if bias is None else bias.contiguous().reshape(-1)
    packed = torch.empty(w.numel() + s.numel() + nb, dtype=torch.float32, device=w.device)
    check(lib().tvb_qmm4_pack(_dev(w), _ptr(w), w.numel(), _ptr(s), _dtype_code(s.dtype), s.numel(), _ptr(bvec),
                              _dtype_code(bvec.dtype) if bvec is not None else F32, nb, _ptr(packed)))
    return packed


def qmm4_quantize(x, groupwise):
    import torch

    m, k = x.shape
    q = torch.empty((m, k), dtype=torch.int8, device=x.device)
    recip = torch.empty(m, dtype=torch.float32, device=x.device)
    neg_zp = torch.empty(m, dtype=torch.int32, device=x.device)
    check(lib().tvb_qmm4_quantize(_dev(x), _ptr(x), _dtype_code(x.dtype), m, k, 1 if groupwise else 0, _ptr(q), _ptr(recip),
                                  _ptr(neg_zp)))
    return q, recip, neg_zp


def qmm4_matmul(q, recip, neg_zp, packed, n, k, bs, out_dtype, return_iacc=False):
    import torch

    m = q.shape[0]
    nblocks = (k + bs - 1) // bs
    has_bias = 1 if packed.numel() - (n * k // 2 + n * nblocks) else 0
    out = torch.empty((m, n), dtype=out_dtype, device=q.device)
    iacc = torch.empty((m, n, nblocks), dtype=torch.int32, device=q.device) if return_iacc else None
    check(lib().tvb_qmm4_matmul(_dev(q), _ptr(q), _ptr(recip), _ptr(neg_zp), _ptr(packed), has_bias, _ptr(out),
                                _dtype_code(out_dtype), m, n, k, bs, _ptr(iacc)))
    return (out, iacc) if return_iacc else out


def qmm4(x, packed, bs, k, n):
    import torch

    m = x.shape[0]
    nblocks = (k + bs - 1) // bs
    has_bias = 1 if packed.numel() - (n * k // 2 + n * nblocks) else 0
    out = torch.empty((m, n), dtype=x.dtype, device=x.device)
    nbytes = lib().tvb_qmm4_workspace_bytes(m, k)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=x.device)
    check(lib().tvb_qmm4(_dev(x), _ptr(x), _dtype_code(x.dtype), _ptr(packed), has_bias, _ptr(out), m, n, k, bs, _ptr(ws),
                         nbytes))
    return out


def qmm4_prepare(packed, n, k, bs):
    import torch

    nbytes = lib().tvb_qmm4_prepared_bytes(n, k)
    prepared = torch.empty(nbytes, dtype=torch.uint8, device=packed.device)
    check(lib().tvb_qmm4_prepare(_dev(packed), _ptr(packed), n, k, bs, _ptr(prepared), nbytes))
    return prepared


def qmm4_tc(x, packed, prepared, bs, k, n):
    import torch

    m = x.shape[0]
    nblocks = (k + bs - 1) // bs
    has_bias = 1 if packed.numel() - (n * k // 2 + n * nblocks) else 0
    out = torch.empty((m, n), dtype=x.dtype, device=x.device)
    nbytes = lib().tvb_qmm4_tc_workspace_bytes(m, k)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=x.device)
    check(lib().tvb_qmm4_tc(_dev(x), _ptr(x), _dtype_code(x.dtype), _ptr(packed), has_bias, _ptr(prepared), _ptr(out), m, n, k,
                            bs, _ptr(ws), nbytes))
    return out


def qmm4_prepare16(packed, n, k, bs):
    import torch

    nbytes = lib().tvb_qmm4_prepared16_bytes(n, k)
    prepared = torch.empty(nbytes, dtype=torch.uint8, device=packed.device)
    check(lib().tvb_qmm4_prepare16(_dev(packed), _ptr(packed), n, k, bs, _ptr(prepared), nbytes))
    return prepared


def qmm4_tc16(x, packed, prepared, bs, k, n):
    import torch

    m = x.shape[0]
    nblocks = (k + bs - 1) // bs
    has_bias = 1 if packed.numel() - (n * k // 2 + n * nblocks) else 0
    out = torch.empty((m, n), dtype=x.dtype, device=x.device)
    nbytes = lib().tvb_qmm4_tc16_workspace_bytes(m, k)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=x.device)
    check(lib().tvb_qmm4_tc16(_dev(x), _ptr(x), _dtype_code(x.dtype), _ptr(packed), has_bias, _ptr(prepared), _ptr(out), m, n, k,
                              bs, _ptr(ws), nbytes))
    return out


def qmm4_decode_prepare(packed, n, k, bs):
    import torch

    nbytes = lib().tvb_qmm4_decode_prepared_bytes(n, k, bs)
    prepared = torch.empty(nbytes, dtype=torch.uint8, device=packed.device)
    check(lib().tvb_qmm4_decode_prepare(_dev(packed), _ptr(packed), n, k, bs, _ptr(prepared), nbytes))
    return prepared


def qmm4_decode(x, packed, prepared, bs, k, n):
    import torch

    m = x.shape[0]
    has_bias = 1 if packed.numel() - (n * k // 2 + n * (k // bs)) else 0
    out = torch.empty((m, n), dtype=x.dtype, device=x.device)
    nbytes = lib().tvb_qmm4_decode_workspace_bytes(m, k)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=x.device)
    check(lib().tvb_qmm4_decode(_dev(x), _ptr(x), _dtype_code(x.dtype), _ptr(packed), has_bias, _ptr(prepared), _ptr(out), m, n,
                                k, bs, _ptr(ws), nbytes))
    return out


def qmm4_fast_prepare(packed, n, k, bs):
    """(prepared float16 weights, inexact flag)"""
    import torch

    nbytes = lib().tvb_qmm4_fast_prepared_bytes(n, k)
    prepared = torch.empty(nbytes, dtype=torch.uint8, device=packed.device)
    flag = _i(0)
    check(lib().tvb_qmm4_fast_prepare(_dev(packed), _ptr(packed), n, k, bs, _ptr(prepared), nbytes, _c.byref(flag)))
    return prepared, flag.value


def qmm4_fast(x, packed, prepared, bs, k, n):
    import torch

    m = x.shape[0]
    nblocks = (k + bs - 1) // bs
    has_bias = 1 if packed.numel() - (n * k // 2 + n * nblocks) else 0
    out = torch.empty((m, n), dtype=x.dtype, device=x.device)
    nbytes = lib().tvb_qmm4_fast_workspace_bytes(m, k)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=x.device)
    check(lib().tvb_qmm4_fast(_dev(x), _ptr(x), _dtype_code(x.dtype), _ptr(packed), has_bias, _ptr(prepared), _ptr(out), m, n, k,
                              bs, _ptr(ws), nbytes))
    return out


def scaled_mm(a, b, scale_a, scale_b, bias=None, scale_result=None, out_dtype=None, variant=0):
    import torch

    m, k = a.shape
    n = b.shape[1]
    out_dtype = out_dtype or a.dtype
    rowwise = 0 if (scale_a.numel() == 1 and scale_b.numel() == 1) else 1
    sa = scale_a.contiguous().reshape(-1)
    sb = scale_b.contiguous().reshape(-1)
    out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    check(lib().tvb_scaled_mm(_dev(a), _ptr(a), _dtype_code(a.dtype), a.stride(0), a.stride(1), _ptr(b), _dtype_code(b.dtype),
                              b.stride(0), b.stride(1), _ptr(sa), _ptr(sb), rowwise, _ptr(bias),
                              _dtype_code(bias.dtype) if bias is not None else F32, _ptr(scale_result), _ptr(out),
                              _dtype_code(out_dtype), m, n, k, variant))
    return out


# ---- the fused Linear layer and layer norm. Like the wrappers above they take tensors in device memory (torch.cuda tensors, or
# "vk" tensors), queue on the backend's stream (tvb_stream) and allocate their outputs on the operands' device: whoever mixes
# them with other work on the same tensors orders that stream and theirs (tvb_set_stream, or a synchronize between).

_FLOATS = None


def _float_code(t):
    global _FLOATS
    if _FLOATS is None:
        import torch

        _FLOATS = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
    code = _FLOATS.get(t.dtype)
    if code is None:
        raise TypeError(f"float32, float16 or bfloat16 expected, got {t.dtype}")
    return code


def _matrix(fn, name, t, rows, cols, like):
    """Checks a [rows, cols] operand with contiguous columns; returns its row stride in elements."""
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != cols or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{fn}: {name} must be a {like.dtype} matrix [{rows}, {cols}] on {like.device}, got {t.dtype} "
                         f"{list(t.shape)} on {t.device}")
    s0, s1 = t.stride()
    if (cols > 1 and s1 != 1) or (rows > 1 and s0 < cols):
        raise ValueError(f"{fn}: {name} needs contiguous columns and rows that do not overlap (strides {(s0, s1)})")
    return s0 if rows > 1 else cols


def _vector(fn, name, t, n, like, dtypes=None):
    if t.dim() != 1 or t.shape[0] != n or t.device != like.device or not t.is_contiguous() or t.dtype not in (dtypes or (like.dtype,)):
        raise ValueError(f"{fn}: {name} must be a contiguous vector of {n} values on {like.device} of "
                         f"{' or '.join(str(d) for d in (dtypes or (like.dtype,)))}, got {t.dtype} {list(t.shape)} on {t.device}")


def _activation(fn, activation):
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"{fn}: activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    return code


def _workspace(nbytes, like):
    """(tensor to keep, its address or None)"""
    if nbytes == 0:
        return None, None
    import torch

    ws = torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    return ws, ws.data_ptr()


def _out(t):
    return t.data_ptr() if t is not None else None


def linear(x, w, bias=None, residual=None, activation="none", save_preactivation=False):
    """tvb_linear on device tensors: act(x @ w.t() + bias) + residual for x [m, k], w [n, k], bias [n], residual [m, n].
    With save_preactivation returns (y, z), z being x @ w.t() + bias: what linear_backward takes for an activation."""
    import torch

    code, act = _float_code(x), _activation("linear", activation)
    if x.dim() != 2 or w.dim() != 2:
        raise ValueError("linear: x [m, k] and w [n, k] expected")
    (m, k), n = x.shape, w.shape[0]
    x_sm, w_sn = _matrix("linear", "x", x, m, k, x), _matrix("linear", "w", w, n, k, x)
    if bias is not None:
        _vector("linear", "bias", bias, n, x)
    r_sm = _matrix("linear", "residual", residual, m, n, x) if residual is not None else 0
    y = torch.empty((m, n), dtype=x.dtype, device=x.device)
    z = torch.empty((m, n), dtype=x.dtype, device=x.device) if save_preactivation else None
    so, xp, wp = lib(), x.data_ptr(), w.data_ptr()
    nbytes = so.tvb_linear_workspace_bytes(code, xp, x_sm, wp, w_sn, m, n, k)
    ws, ws_ptr = _workspace(nbytes, x)
    check(so.tvb_linear(_dev(x), xp, code, x_sm, wp, w_sn, _out(bias), act, _out(residual), r_sm, y.data_ptr(), _out(z), m, n, k,
                        ws_ptr, nbytes))
    return (y, z) if save_preactivation else y


def linear_backward(dy, x, w, z=None, activation="none", need=(True, True, True)):
    """tvb_linear_backward on device tensors: (dx, dw, db), None where `need` is false. z: what linear saved (not needed
    without an activation)."""
    import torch

    code, act = _float_code(x), _activation("linear_backward", activation)
    if x.dim() != 2 or w.dim() != 2:
        raise ValueError("linear_backward: x [m, k] and w [n, k] expected")
    (m, k), n = x.shape, w.shape[0]
    x_sm, w_sn = _matrix("linear_backward", "x", x, m, k, x), _matrix("linear_backward", "w", w, n, k, x)
    dy_sm = _matrix("linear_backward", "dy", dy, m, n, x)
    if z is not None:
        _matrix("linear_backward", "z", z, m, n, x)
        if not z.is_contiguous():
            raise ValueError("linear_backward: z must be contiguous")
    elif act != 0:
        raise ValueError("linear_backward: an activation's gradient needs z, the values before it")
    dx = torch.empty((m, k), dtype=x.dtype, device=x.device) if need[0] else None
    dw = torch.empty((n, k), dtype=x.dtype, device=x.device) if need[1] else None
    db = torch.empty((n,), dtype=x.dtype, device=x.device) if need[2] else None
    so, dyp, xp, wp = lib(), dy.data_ptr(), x.data_ptr(), w.data_ptr()
    want = (WANT_DX if need[0] else 0) | (WANT_DW if need[1] else 0) | (WANT_DB if need[2] else 0)
    nbytes = so.tvb_linear_backward_workspace_bytes(code, dyp, dy_sm, xp, x_sm, wp, w_sn, act, want, m, n, k)
    ws, ws_ptr = _workspace(nbytes, x)
    check(so.tvb_linear_backward(_dev(x), dyp, code, dy_sm, _out(z), xp, x_sm, wp, w_sn, act, _out(dx), _out(dw), _out(db), m, n, k,
                                 ws_ptr, nbytes))
    return dx, dw, db


def _norm_params(fn, x, d, *params):
    """The common dtype code of weight and bias (each may be None)."""
    import torch

    given = [(name, t) for name, t in params if t is not None]
    for name, t in given:
        _vector(fn, name, t, d, x, (x.dtype, torch.float32))
    if len({t.dtype for _, t in given}) > 1:
        raise ValueError(f"{fn}: weight and bias must have one dtype")
    return _float_code(given[0][1]) if given else _float_code(x)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """tvb_layer_norm on device tensors: (y, mean, rstd) for x [rows, d], weight and bias [d] (of x's dtype or float32)."""
    import torch

    code = _float_code(x)
    if x.dim() != 2:
        raise ValueError("layer_norm: x [rows, d] expected")
    rows, d = x.shape
    x_sm = _matrix("layer_norm", "x", x, rows, d, x)
    pcode = _norm_params("layer_norm", x, d, ("weight", weight), ("bias", bias))
    y = torch.empty((rows, d), dtype=x.dtype, device=x.device)
    mean = torch.empty((rows,), dtype=torch.float32, device=x.device)
    rstd = torch.empty((rows,), dtype=torch.float32, device=x.device)
    check(lib().tvb_layer_norm(_dev(x), x.data_ptr(), code, x_sm, _out(weight), _out(bias), pcode, eps, y.data_ptr(),
                               mean.data_ptr(), rstd.data_ptr(), rows, d))
    return y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight=None, need=(True, True, True)):
    """tvb_layer_norm_backward on device tensors: (dx, dweight, dbias), None where `need` is false; mean and rstd [rows] as
    layer_norm returned them. dweight and dbias have weight's dtype (x's without a weight)."""
    import torch

    code = _float_code(x)
    if x.dim() != 2:
        raise ValueError("layer_norm_backward: x [rows, d] expected")
    rows, d = x.shape
    x_sm, dy_sm = _matrix("layer_norm_backward", "x", x, rows, d, x), _matrix("layer_norm_backward", "dy", dy, rows, d, x)
    pcode = _norm_params("layer_norm_backward", x, d, ("weight", weight))
    for name, t in (("mean", mean), ("rstd", rstd)):
        _vector("layer_norm_backward", name, t, rows, x, (torch.float32,))
    pdtype = weight.dtype if weight is not None else x.dtype
    dx = torch.empty((rows, d), dtype=x.dtype, device=x.device) if need[0] else None
    dg = torch.empty((d,), dtype=pdtype, device=x.device) if need[1] else None
    db = torch.empty((d,), dtype=pdtype, device=x.device) if need[2] else None
    so = lib()
    nbytes = so.tvb_layer_norm_backward_workspace_bytes(rows, d) if need[1] or need[2] else 0
    ws, ws_ptr = _workspace(nbytes, x)
    check(so.tvb_layer_norm_backward(_dev(x), dy.data_ptr(), code, dy_sm, x.data_ptr(), x_sm, mean.data_ptr(), rstd.data_ptr(),
                                     _out(weight), pcode, _out(dx), _out(dg), _out(db), rows, d, ws_ptr, nbytes))
    return dx, dg, db
