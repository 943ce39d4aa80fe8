"""ctypes binding of libstepquant_b200.so (the C ABI in include/stepquant_b200.h).

The library is built in-tree by ``stepquant_b200._build``.  There is no
fallback: if the library is missing every device operation raises.
"""
import ctypes
import os
import struct

import torch

from ._build import LIBRARY

SQ_OK, SQ_ERR_ARGUMENT, SQ_ERR_SHAPE, SQ_ERR_UNSUPPORTED, SQ_ERR_CUDA, SQ_ERR_CAPACITY = range(6)
SQ_STATUS_SLOT_RANGE = 1
SQ_STATUS_TIMEOUT = 2
SQ_F32, SQ_BF16, SQ_F16 = 0, 1, 2
SQ_GDN, SQ_KDA = 0, 1

_DTYPES = {torch.float32: SQ_F32, torch.bfloat16: SQ_BF16, torch.float16: SQ_F16}

_p = ctypes.c_void_p
_i32 = ctypes.c_int32
_i64 = ctypes.c_int64


class SqPlan(ctypes.Structure):
    _fields_ = [("architecture", _i32), ("heads", _i32), ("keys", _i32), ("values", _i32),
                ("value_group_size", _i32), ("storage", _i32), ("page_bytes", _i64),
                ("bits", _p), ("impact", _p), ("offsets", _p), ("rows", _p), ("columns", _p),
                ("bits_host", _p)]


class SqStepArgs(ctypes.Structure):
    _fields_ = [("q", _p), ("k", _p), ("v", _p), ("q_stride", _i64), ("k_stride", _i64), ("v_stride", _i64),
                ("qk_heads", _i32), ("io_dtype", _i32), ("g", _p), ("beta", _p), ("gate_dtype", _i32),
                ("normalize", _i32), ("a_log", _p), ("dt_bias", _p), ("scale", ctypes.c_float),
                ("reserved", _i32), ("out", _p)]


class SqPrefillArgs(ctypes.Structure):
    _fields_ = [("q", _p), ("k", _p), ("v", _p), ("q_stride", _i64), ("k_stride", _i64), ("v_stride", _i64),
                ("io_dtype", _i32), ("qk_heads", _i32), ("heads", _i32), ("keys", _i32), ("values", _i32),
                ("normalize", _i32), ("scale", ctypes.c_float), ("num_seqs", _i32), ("tokens", _i32), ("cu_seqlens", _p),
                ("g", _p), ("beta", _p), ("initial_state", _p), ("final_state", _p), ("out", _p),
                ("workspace", _p), ("workspace_bytes", _i64), ("status", _p)]


class SqNormArgs(ctypes.Structure):
    _fields_ = [("x", _p), ("residual", _p), ("weight", _p), ("residual_out", _p), ("out", _p), ("scale", _p),
                ("x_stride", _i64), ("residual_stride", _i64), ("rows", _i32), ("hidden", _i32), ("dtype", _i32),
                ("weight_dtype", _i32), ("normalize", _i32), ("eps", ctypes.c_float)]


class SqMatmulArgs(ctypes.Structure):
    _fields_ = [("x", _p), ("x_scale", _p), ("w", _p), ("w_scale", _p), ("residual", _p), ("out", _p), ("status", _p),
                ("x_stride", _i64), ("w_stride", _i64), ("residual_stride", _i64), ("rows", _i32), ("width", _i32),
                ("hidden", _i32), ("dtype", _i32), ("wait_clocks", _i64)]


class SqConvArgs(ctypes.Structure):
    _fields_ = [("x", _p), ("weight", _p), ("bias", _p), ("y", _p), ("initial_state", _p), ("final_state", _p),
                ("slots", _p), ("cu_seqlens", _p), ("status", _p), ("x_stride", _i64), ("num_slots", _i64),
                ("tokens", _i32), ("num_seqs", _i32), ("channels", _i32), ("taps", _i32), ("dtype", _i32),
                ("silu", _i32)]


class SqScanArgs(ctypes.Structure):
    _fields_ = [("u", _p), ("dt", _p), ("z", _p), ("b", _p), ("c", _p), ("a", _p), ("d", _p), ("dt_bias", _p),
                ("y", _p), ("initial_state", _p), ("final_state", _p), ("slots", _p), ("cu_seqlens", _p),
                ("status", _p), ("workspace", _p), ("workspace_bytes", _i64), ("u_stride", _i64), ("dt_stride", _i64),
                ("z_stride", _i64), ("b_stride", _i64), ("c_stride", _i64), ("num_slots", _i64), ("tokens", _i32),
                ("num_seqs", _i32), ("channels", _i32), ("states", _i32), ("groups", _i32), ("dtype", _i32),
                ("softplus", _i32)]


class SqRotaryArgs(ctypes.Structure):
    _fields_ = [("x", _p), ("out", _p), ("positions", _p), ("frequencies", _p), ("x_stride", _i64), ("x_head_stride", _i64),
                ("out_stride", _i64), ("out_head_stride", _i64), ("tokens", _i32), ("heads", _i32), ("dim", _i32),
                ("turned", _i32), ("dtype", _i32), ("position_dtype", _i32), ("interleaved", _i32), ("inverse", _i32),
                ("magnitude", ctypes.c_float)]


class SqKvArgs(ctypes.Structure):
    _fields_ = [("k", _p), ("v", _p), ("data", _p), ("page_table", _p), ("lengths", _p), ("cu_seqlens", _p),
                ("positions", _p), ("frequencies", _p), ("status", _p), ("k_stride", _i64), ("k_head_stride", _i64),
                ("v_stride", _i64), ("v_head_stride", _i64), ("table_stride", _i64), ("num_pages", _i64), ("tokens", _i32),
                ("num_seqs", _i32), ("table_width", _i32), ("heads", _i32), ("dim", _i32), ("page_size", _i32),
                ("dtype", _i32), ("turned", _i32), ("position_dtype", _i32), ("interleaved", _i32),
                ("magnitude", ctypes.c_float)]


class SqKvAttentionArgs(ctypes.Structure):
    _fields_ = [("q", _p), ("data", _p), ("out", _p), ("page_table", _p), ("lengths", _p), ("cu_seqlens", _p),
                ("status", _p), ("workspace", _p), ("workspace_bytes", _i64), ("q_stride", _i64), ("q_head_stride", _i64),
                ("table_stride", _i64), ("num_pages", _i64), ("tokens", _i32), ("num_seqs", _i32), ("table_width", _i32),
                ("q_heads", _i32), ("heads", _i32), ("dim", _i32), ("page_size", _i32), ("dtype", _i32), ("window", _i32),
                ("scale", ctypes.c_float), ("wait_clocks", _i64)]


_SIGNATURES = {
    "sq_version": (_i32, []),
    "sq_error_string": (ctypes.c_char_p, [_i32]),
    "sq_packed_layout": (_i32, [_i32, _i32, _i32, _i32, _i32, _p, _i32, _p, _p, _p, _p]),
    "sq_encode": (_i32, [_p, _p, _p, _i32, _p, _i64, _p, _p]),
    "sq_decode": (_i32, [_p, _p, _i64, _p, _i32, _p, _p, _p]),
    "sq_step": (_i32, [_p, _p, _i64, _p, _i32, _p, _p, _p, _p]),
    "sq_scratch_floats": (_i64, [_p]),
    "sq_readout": (_i32, [_p, _p, _i64, _p, _i32, _p, _p, _p, _p, _p]),
    "sq_writeback": (_i32, [_p, _p, _i64, _p, _i32, _p, _p, _p, _p]),
    "sq_fit_state": (_i32, [_p, _p, _i32, _p, _p, _p, _p, _p, _p]),
    "sq_pack": (_i32, [_p, _i64, _i32, _p, _p]),
    "sq_packed_bytes": (_i64, [_i64, _i32]),
    "sq_unpack": (_i32, [_p, _i64, _i32, _p, _p]),
    "sq_fp32_step": (_i32, [_p, _i64, _i32, _i32, _i32, _i32, _p, _i32, _p, _p, _p]),
    "sq_step_async_noalloc": (_i32, [_p, _p, _i64, _p, _i32, _p, _p, _p]),
    "sq_noalloc_scratch_bytes": (_i64, []),
    "sq_budget_stream": (_i32, [_i32, _i32, ctypes.POINTER(_p), ctypes.POINTER(_i32), ctypes.POINTER(_i32)]),
    "sq_selftest_fp16_division": (_i32, [_p, _p, _p, _i64, _p]),
    "sq_gdn_prefill": (_i32, [_p, _p]),
    "sq_gdn_prefill_workspace_bytes": (_i64, [_i32, _i32, _i32]),
    "sq_kda_prefill": (_i32, [_p, _p]),
    "sq_rms_norm": (_i32, [_p, _p]),
    "sq_matmul_fp8": (_i32, [_p, _p]),
    "sq_causal_conv": (_i32, [_p, _p]),
    "sq_causal_conv_step": (_i32, [_p, _p]),
    "sq_selective_scan": (_i32, [_p, _p]),
    "sq_selective_scan_step": (_i32, [_p, _p]),
    "sq_selective_scan_workspace_bytes": (_i64, [_i32] * 5),
    "sq_rotary": (_i32, [_p, _p]),
    "sq_kv_append": (_i32, [_p, _p]),
    "sq_kv_read": (_i32, [_p, _p]),
    "sq_kv_attention": (_i32, [_p, _p]),
    "sq_kv_attention_workspace_bytes": (_i64, [_i32] * 5),
}

EXPORTED = tuple(_SIGNATURES)
_lib = None


def library_path():
    return LIBRARY


def lib():
    """The loaded library; raises RuntimeError when it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIBRARY):
            raise RuntimeError(
                f"stepquant_b200 native library not found at {LIBRARY}; build it with "
                "`python -m stepquant_b200._build` (there is no CPU fallback)")
        handle = ctypes.CDLL(LIBRARY)
        for name, (restype, argtypes) in _SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = restype
            fn.argtypes = argtypes
        _lib = handle
    return _lib


class NativeError(RuntimeError):
    pass


def check(code):
    """Map an sq_error code to the reference's exception types."""
    if code == SQ_OK:
        return
    text = lib().sq_error_string(code).decode()
    if code in (SQ_ERR_ARGUMENT, SQ_ERR_SHAPE, SQ_ERR_CAPACITY):
        raise ValueError(f"stepquant_b200: {text}")
    if code == SQ_ERR_UNSUPPORTED:
        raise NotImplementedError(f"stepquant_b200: {text}")
    raise NativeError(f"stepquant_b200: {text} ({torch.cuda.get_device_name() if torch.cuda.is_available() else 'no device'})")


def dtype_code(dtype):
    try:
        return _DTYPES[dtype]
    except KeyError:
        raise ValueError(f"unsupported dtype {dtype}; use float32, bfloat16 or float16") from None


def ptr(tensor):
    return None if tensor is None else ctypes.c_void_p(tensor.data_ptr())


def stream_handle(stream=None):
    stream = torch.cuda.current_stream() if stream is None else stream
    return ctypes.c_void_p(stream.cuda_stream)


def require_cuda(*tensors):
    for t in tensors:
        if t is not None and t.device.type != "cuda":
            raise ValueError("stepquant_b200 operates on CUDA tensors only (no CPU fallback)")


# ---------------------------------------------------------------------------
# the layer operators' calls (kernels/norm.py, matmul.py, conv.py, scan.py,
# rotary.py, kv_cache.py)
# ---------------------------------------------------------------------------
_FORMATS = {_p: "P", _i64: "q", _i32: "i", ctypes.c_float: "f"}


def packer(arguments):
    """Function of a ctypes Structure's fields, in order, that returns its
    bytes: a few microseconds less than building the Structure, on calls whose
    kernels take about as long."""
    fmt = struct.Struct("@" + "".join(_FORMATS[kind] for _, kind in arguments._fields_) + "0P")
    assert fmt.size == ctypes.sizeof(arguments)

    def pack(*values):
        try:
            return fmt.pack(*values)
        except struct.error:
            raise ValueError(f"a size or a stride is out of the C structure's range: {values}") from None

    return pack


def launch(entry, packed, index):
    """Run a C entry point of (arguments, stream) on the current stream of device ``index``."""
    if index == torch._C._cuda_getDevice():
        code = entry(packed, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            code = entry(packed, torch._C._cuda_getCurrentRawStream(index))
    if code:
        check(code)


def device_index(first, *others):
    """Index of the CUDA device that ``first`` and the others (or None) lie on."""
    index = first.get_device()
    if index < 0:
        require_cuda(first)
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError(f"expected every tensor on {first.device}, got one on {t.device}")
    return index


def status_word(status):
    """``status`` (or None): four bytes that a kernel sets bits in."""
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
        raise ValueError(f"status: expected an int32 word, got {status.dtype} {list(status.shape)}")
    return status


def address(tensor):
    return 0 if tensor is None else tensor.data_ptr()


def aligned(x):
    """x contiguous with a 16-byte aligned base (copied when it is not)."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def rows_of(x, name):
    """[..., dim] -> [rows, dim] with a contiguous last axis and one row stride (copied when it has none)."""
    if x.dtype not in _DTYPES:
        raise ValueError(f"{name}: unsupported dtype {x.dtype}; use float32, bfloat16 or float16")
    if x.dim() != 2:
        if x.dim() < 1:
            raise ValueError(f"{name}: expected [..., dim]")
        x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1 and x.shape[1] != 1:
        x = x.contiguous()
    return x
