"""Rotary positions of attention layers (csrc/sq_rotary.cu).

``rotary``              heads rotated by their token's position.
``rotary_frequencies``  the angles a token, plain or scaled for long contexts.

Pairs of channels (x1, x2), the halves' i-th or (interleaved) channels 2i and
2i + 1, become magnitude (x1 cos a - x2 sin a, x1 sin a + x2 cos a) with
a = position frequencies[i].  ``kv_cache.kv_append`` rotates keys the same way.
Angles are exact to 10^-7 turns at any position below 2^31.  Asynchronous on the
current stream.
"""
import math

import torch

from .. import _native as N

MOST_DIM = 1024
MOST_FLOAT = torch.finfo(torch.float32).max

_pack = N.packer(N.SqRotaryArgs)


def rotary_frequencies(turned, base=10000.0, *, scaling=None, factor=1.0, original_length=None, slow=1.0, fast=32.0, device="cuda"):
    """float64 [turned / 2] radians a token: base^(-2 i / turned), scaled by

    None       not at all
    "linear"   all divided by ``factor``
    "base"     a base larger by factor^(turned / (turned - 2)): the fastest pair kept, the slowest divided by ``factor``
    "bands"    pairs that turn less than ``slow`` times in ``original_length`` tokens divided by ``factor``, those
               that turn more than ``fast`` times kept, linear in the turns between
    "ramp"     the same, linear in the pair's number between (which is linear in the turns' logarithm)
    """
    if turned < 2 or turned % 2 or not base > 0 or not math.isfinite(base) or not factor > 0 or not math.isfinite(factor):
        raise ValueError(f"expected an even number of channels, a base and a factor above zero, got {turned}, {base}, {factor}")
    if scaling not in (None, "linear", "base", "bands", "ramp"):
        raise ValueError(f"scaling: expected None, 'linear', 'base', 'bands' or 'ramp', got {scaling!r}")
    pair = torch.arange(turned // 2, dtype=torch.float64)
    if scaling == "base" and turned > 2:
        base = base * factor ** (turned / (turned - 2))
    f = base ** (-2 * pair / turned)
    if scaling == "linear":
        f = f / factor
    elif scaling in ("bands", "ramp"):
        if original_length is None or not original_length > 0 or not 0 < slow < fast:
            raise ValueError("bands and ramps need original_length > 0 and 0 < slow < fast")
        turns = original_length * f / (2 * math.pi)
        if scaling == "ramp":
            if base == 1:
                raise ValueError("a ramp needs a base other than 1")
            number = lambda t: turned * math.log(original_length / (2 * math.pi * t)) / (2 * math.log(base))  # noqa: E731
            low, high = max(math.floor(number(fast)), 0), min(math.ceil(number(slow)), turned - 1)
            kept = 1 - ((pair - low) / max(high - low, 1e-3)).clamp(0, 1)
        else:
            kept = ((turns - slow) / (fast - slow)).clamp(0, 1)
        f = f * kept + f / factor * (1 - kept)
    return f.to(device)


def checked_frequencies(frequencies, dim):
    """float64 contiguous frequencies (or None) of at most dim channels."""
    if frequencies is None:
        return None
    if frequencies.dim() != 1 or 2 * frequencies.numel() > dim:
        raise ValueError(f"frequencies: expected [turned / 2] for at most {dim} channels, got {list(frequencies.shape)}")
    return frequencies if frequencies.dtype is torch.float64 and frequencies.is_contiguous() else frequencies.double().contiguous()


def checked_positions(positions, tokens):
    """int32 or int64 contiguous positions of ``tokens`` tokens."""
    if positions.shape != (tokens,) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions: expected int32 or int64 [{tokens}], got {positions.dtype} {list(positions.shape)}")
    return positions if tokens < 2 or positions.stride(0) == 1 else positions.contiguous()


def check_magnitude(magnitude):
    if not abs(magnitude) <= MOST_FLOAT:
        raise ValueError("magnitude must be finite in float32")


def rotary(x, positions, frequencies, *, interleaved=False, magnitude=1.0, inverse=False, out=None):
    """x [T, H, D] with the first 2 len(frequencies) channels of each head rotated.

    x: float32, bfloat16 or float16, tokens and heads any stride apart; positions:
    [T] int32 or int64; frequencies: [R / 2] radians a token, float64 (others are
    converted on every call).  ``magnitude`` scales the rotated channels;
    ``inverse`` turns them back (the rotation's gradient).
    ``out``: x itself, a tensor like x whose memory is apart from it, or None (a new one).
    """
    if x.dim() != 3 or not 1 <= x.shape[2] <= MOST_DIM:
        raise ValueError(f"x: expected [tokens, heads, dim] with 1 <= dim <= {MOST_DIM}, got {list(x.shape)}")
    tokens, heads, dim = x.shape
    dtype = N.dtype_code(x.dtype)
    frequencies, positions = checked_frequencies(frequencies, dim), checked_positions(positions, tokens)
    if frequencies is None:
        raise ValueError("frequencies is required")
    check_magnitude(magnitude)
    source = x if dim == 1 or x.stride(2) == 1 else x.contiguous()
    if out is None:
        out = x.new_empty(x.shape)
    elif out.shape != x.shape or out.dtype != x.dtype or (dim > 1 and out.stride(2) != 1):
        raise ValueError(f"out: expected {x.dtype} {list(x.shape)} with a contiguous last axis")
    elif out.data_ptr() == x.data_ptr() and any(n > 1 and a != b for n, a, b in zip(x.shape, x.stride(), out.stride())):
        raise ValueError(f"out: x's memory in another order, strides {list(out.stride())} for {list(x.stride())}")
    index = N.device_index(source, positions, frequencies, out)
    p, (xs, xh, _), (os, oh, _) = N.address, source.stride(), out.stride()
    N.launch(N.lib().sq_rotary, _pack(p(source), p(out), p(positions), p(frequencies), xs, xh, os, oh, tokens, heads, dim,
                                      2 * frequencies.numel(), dtype, positions.dtype == torch.int64, bool(interleaved),
                                      bool(inverse), magnitude), index)
    return out
