"""Product of e4m3 matrices with an fp32 scale per block of 128 (csrc/sq_matmul.cu).

``matmul_fp8``           out = x w^T of scaled e4m3 operands, + residual.
``quantize_weight_fp8``  the e4m3 weight and its 128 x 128 block scales, once at loading.

Activations come from ``norm.rms_norm_fp8`` or ``norm.quantize_fp8``.  Block
products are summed on the tensor cores, scaled and added in fp32; the finished
sum is rounded once.  Asynchronous on the current stream.
"""
import torch

from .. import _native as N
from .norm import BLOCK, FP8, SCALE_FLOOR, E4M3_MAX

_pack = N.packer(N.SqMatmulArgs)


def quantize_weight_fp8(weight):
    """(w, scale) of weight [N, K]: float8_e4m3fn [N, K] and float32
    [ceil(N / 128), ceil(K / 128)], max(max |w|, 1e-30) / 448 of each block."""
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError("weight: expected [width, hidden]")
    rows, cols = weight.shape
    padded = torch.nn.functional.pad(weight.float(), (0, -cols % BLOCK, 0, -rows % BLOCK))
    blocks = padded.unflatten(1, (-1, BLOCK)).unflatten(0, (-1, BLOCK))  # [N / 128, 128, K / 128, 128]
    scale = blocks.abs().amax((1, 3)).clamp_min(SCALE_FLOOR) / E4M3_MAX
    values = (blocks / scale[:, None, :, None]).reshape(padded.shape)[:rows, :cols]
    return values.contiguous().to(FP8), scale


def _operand(x, name):
    """e4m3 rows as the copy engine takes them: 16-byte aligned base and row stride (copied otherwise)."""
    if x.dtype != FP8:
        raise ValueError(f"{name}: expected {FP8}, got {x.dtype}")
    if x.stride(1) != 1 or x.data_ptr() % 16 or (x.shape[0] > 1 and (x.stride(0) % 16 or x.stride(0) < x.shape[1])):
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
    return x


def _scales(scale, shape, name):
    if scale.dtype != torch.float32 or scale.shape != shape:
        raise ValueError(f"{name}: expected float32 {list(shape)}, got {scale.dtype} {list(scale.shape)}")
    return scale.contiguous()


def matmul_fp8(x, x_scale, weight, weight_scale, *, residual=None, out_dtype=torch.bfloat16, status=None):
    """out[m, n] = residual[m, n] + sum_k x[m, k] x_scale[m, k / 128] weight[n, k] weight_scale[n / 128, k / 128].

    x: [..., K] and weight: [N, K] float8_e4m3fn, K a multiple of 16; x_scale:
    [..., ceil(K / 128)], weight_scale: [ceil(N / 128), ceil(K / 128)] float32;
    residual: [..., N] in out_dtype (float32, bfloat16 or float16), or None.
    Should a bounded device wait give up, the outputs left undone are NaN and
    ``status`` (an int32 word, or None) has SQ_STATUS_TIMEOUT.
    """
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError("x and weight: expected [..., hidden] and [width, hidden]")
    lead, hidden, width = x.shape[:-1], x.shape[-1], weight.shape[0]
    if hidden < 1 or width < 1:
        raise ValueError("hidden and width must be positive")
    if hidden % 16:
        raise NotImplementedError("the product is built for a hidden size that is a multiple of 16")
    dtype = N.dtype_code(out_dtype)
    index = N.device_index(x, weight, x_scale, weight_scale, residual, N.status_word(status))
    blocks = (hidden + BLOCK - 1) // BLOCK
    rows = _operand(x if x.dim() == 2 else x.reshape(-1, hidden), "x")
    weight = _operand(weight, "weight")
    x_scale = _scales(x_scale, (*lead, blocks), "x_scale")
    weight_scale = _scales(weight_scale, ((width + BLOCK - 1) // BLOCK, blocks), "weight_scale")
    if residual is not None:
        if residual.shape != (*lead, width) or residual.dtype != out_dtype:
            raise ValueError(f"residual: expected {out_dtype} {[*lead, width]}")
        residual = N.rows_of(residual, "residual")
    out = x_scale.new_empty((*lead, width), dtype=out_dtype)
    count = rows.shape[0]
    N.launch(N.lib().sq_matmul_fp8,
             _pack(rows.data_ptr(), x_scale.data_ptr(), weight.data_ptr(), weight_scale.data_ptr(), N.address(residual),
                   out.data_ptr(), N.address(status), rows.stride(0) if count > 1 else hidden,
                   weight.stride(0) if width > 1 else hidden, 0 if residual is None else residual.stride(0), count, width,
                   hidden, dtype, 0), index)
    return out
