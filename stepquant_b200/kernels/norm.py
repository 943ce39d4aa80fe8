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


def _run(x, weight, residual, eps, fp8):
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x: expected [..., hidden] with hidden >= 1")
    shape, hidden = x.shape, x.shape[-1]
    rows = N.rows_of(x, "x")
    if weight is not None and (weight.dim() != 1 or weight.shape[0] != hidden):
        raise ValueError(f"weight: expected [{hidden}], got {tuple(weight.shape)}")
    res = None
    if residual is not None:
        if residual.shape != shape or residual.dtype != x.dtype:
            raise ValueError("residual: expected x's shape and dtype")
        res = N.rows_of(residual, "residual")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    device = x.device
    N.same_device(device, weight=weight, residual=residual)
    if weight is not None:
        weight_dtype = N.dtype_code(weight.dtype)
        weight = weight.contiguous()
    else:
        weight_dtype = N.SQ_F32
    count = rows.shape[0]
    out = torch.empty(shape, device=device, dtype=FP8 if fp8 else x.dtype)
    scale = torch.empty(*shape[:-1], -(-hidden // BLOCK), device=device, dtype=torch.float32) if fp8 else None
    total = torch.empty(shape, device=device, dtype=x.dtype) if res is not None else None
    args = N.SqNormArgs(rows.data_ptr(), None if res is None else res.data_ptr(), None if weight is None else weight.data_ptr(),
                        None if total is None else total.data_ptr(), out.data_ptr(),
                        None if scale is None else scale.data_ptr(), rows.stride(0), 0 if res is None else res.stride(0),
                        count, hidden, N.dtype_code(x.dtype), weight_dtype, 0 if weight is None else 1, eps)
    N.launch(N.lib().sq_rms_norm, args, device)
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
