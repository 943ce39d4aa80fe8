"""Residual norm and e4m3 activations of the layers around the recurrent state.

``rms_norm``       root-mean-square norm, with the residual's addition.
``rms_norm_fp8``   the same with an e4m3 output and one fp32 scale per token and
                   128 channels: the operand that ``matmul.matmul_fp8`` reads.
``quantize_fp8``   that output for rows that need no norm.

All run ``sq_rms_norm`` (csrc/sq_norm.cu), statistics in fp32, asynchronously on
the current stream.
"""
import torch

from .. import _native as N

FP8 = torch.float8_e4m3fn
BLOCK = 128  # channels of a scale
E4M3_MAX, SCALE_FLOOR = 448.0, 1e-30  # as in csrc/sq_norm.cu


_pack = N.packer(N.SqNormArgs)


def _run(x, weight, residual, eps, fp8):
    shape = x.shape
    hidden = shape[-1] if shape else 0
    if not hidden:
        raise ValueError("x: expected [..., hidden] with hidden >= 1")
    dtype = N.dtype_code(x.dtype)
    rows, total, res_address, res_stride, weight_dtype, weight_address = N.rows_of(x, "x"), None, 0, 0, N.SQ_F32, 0
    if weight is not None:
        if weight.shape != (hidden,):
            raise ValueError(f"weight: expected [{hidden}], got {list(weight.shape)}")
        weight_dtype = N.dtype_code(weight.dtype)
        weight = weight.contiguous()
        weight_address = weight.data_ptr()
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    if residual is not None and (residual.shape != shape or residual.dtype != x.dtype):
        raise ValueError("residual: expected x's shape and dtype")
    index = N.device_index(x, weight, residual)
    count = rows.shape[0]
    # empty_like is the quicker allocation, of the right layout only for contiguous rows.
    like = x if x.is_contiguous() else None
    if residual is not None:
        res = N.rows_of(residual, "residual")
        res_address, res_stride = res.data_ptr(), res.stride(0)
        total = x.new_empty(shape) if like is None else torch.empty_like(x)
    if fp8:
        out = x.new_empty(shape, dtype=FP8) if like is None else torch.empty_like(x, dtype=FP8)
        scale = x.new_empty((*shape[:-1], (hidden + BLOCK - 1) // BLOCK), dtype=torch.float32)
        scale_address = scale.data_ptr()
    else:
        out, scale, scale_address = x.new_empty(shape) if like is None else torch.empty_like(x), None, 0
    N.launch(N.lib().sq_rms_norm, _pack(rows.data_ptr(), res_address, weight_address, 0 if total is None else total.data_ptr(),
                                        out.data_ptr(), scale_address, rows.stride(0), res_stride, count, hidden, dtype,
                                        weight_dtype, weight is not None, eps), index)
    return out, scale, total


def rms_norm(x, weight, residual=None, *, eps=1e-6):
    """y = h / sqrt(mean(h^2) + eps) * weight with h = x (+ residual).

    x, residual: [..., hidden] float32, bfloat16 or float16, alike, rows any
    stride apart; weight: [hidden] in any of the three.  Returns y in x's
    dtype, or (y, h rounded to x's dtype) with a residual; the norm itself
    takes h unrounded.
    """
    if weight is None:
        raise ValueError("weight is required")
    out, _, total = _run(x, weight, residual, eps, False)
    return out if residual is None else (out, total)


def rms_norm_fp8(x, weight, residual=None, *, eps=1e-6):
    """``rms_norm`` with an 8-bit output: (q, scale) or (q, scale, h).

    q: [..., hidden] float8_e4m3fn; scale: [..., ceil(hidden / 128)] float32,
    max(max |y|, 1e-30) / 448 of each 128 channels; y is q times its scale.
    """
    if weight is None:
        raise ValueError("weight is required")
    out, scale, total = _run(x, weight, residual, eps, True)
    return (out, scale) if residual is None else (out, scale, total)


def quantize_fp8(x):
    """(q, scale) of x itself, as ``rms_norm_fp8`` gives them of the normed rows."""
    return _run(x, None, None, 0.0, True)[:2]
