"""Frequencies of half a turn a token and more, for which whole turns go before the fixed point
(csrc/sq_kv.cuh): the tolerances of test_gpu_rotary.py, bytes of the cache equal.

For the bytes the oracle takes angles modulo a turn in exact arithmetic: a frequency of
pi leaves keys within 10^-14 of bfloat16 values, where the side of a border depends on
less than position times frequency loses when it is rounded to 64 bits.  Even so a rotated
key is a sum of two products in 64 bits, on either side: sine and cosine within 2^-52,
products and sum within 2^-53 each, together below 2^-50 (|x1| + |x2|).  Where a group's
minimum is that close to a bfloat16 (for a frequency of pi the first few positions), the
minimum held may be the one below: codes then stand within half of a step that is larger by
no more than (2^-7 |m|) / 15 and a unit of the scale.
"""
import math
from fractions import Fraction

import pytest
import torch

from kv_reference import quantize
from test_gpu_rotary import _check, _data

pytestmark = pytest.mark.gpu


def _cases():
    from stepquant_b200.kernels.rotary import rotary_frequencies
    return [rotary_frequencies(64, scaling="linear", factor=0.25), rotary_frequencies(64, 0.01),
            torch.linspace(3.0, 13.0, 32, dtype=torch.float64, device="cuda"),
            torch.tensor([math.pi, -math.pi, 2 * math.pi, -4.0, 3.14159265, 1e4 + 0.1, 7.0, -100.0] * 4, dtype=torch.float64, device="cuda")]


@pytest.mark.parametrize("case", range(4))
@pytest.mark.parametrize("first", [0, 10 ** 6, -40])
def test_fast_pairs(case, first):
    from stepquant_b200.kernels.rotary import rotary
    f = _cases()[case]
    assert float(f.abs().max()) > 3.2
    x, positions = _data(40, 2, 128, torch.float32), torch.arange(first, first + 40, device="cuda")
    for interleaved in (False, True):
        _check(rotary(x, positions, f, interleaved=interleaved), x, positions, f, interleaved)


TURN = 2 * Fraction(314159265358979323846264338327950288419716939937510582097494459, 10 ** 62)


def _turn(x, frequencies):
    """x [T, H, D] of positions 0 .. T - 1 rotated, in 64 bits; the angles exact modulo a turn and then rounded."""
    n, y = frequencies.numel(), x.double().clone()
    exact = [Fraction(f) for f in frequencies.tolist()]
    angle = torch.tensor([[float(p * f - TURN * round(p * f / TURN)) for f in exact] for p in range(x.shape[0])],
                         dtype=torch.float64, device=x.device)[:, None]
    u, v = x[..., :n].double(), x[..., n:2 * n].double()
    y[..., :n], y[..., n:2 * n] = u * angle.cos() - v * angle.sin(), u * angle.sin() + v * angle.cos()
    return y


@pytest.mark.parametrize("case", range(4))
def test_fast_pairs_in_the_cache(case):
    from stepquant_b200.kernels.kv_cache import QuantizedKVPool
    f = _cases()[case]
    pool = QuantizedKVPool(4, 2, 128, page_size=64)
    k = _data(150, 2, 128, torch.bfloat16)
    table, lengths, cu = (torch.tensor(x, device="cuda", dtype=torch.int32) for x in ([[3, 1, 2]], [150], [0, 150]))
    pool.append(k, k, table, lengths, cu_seqlens=cu, frequencies=f)
    got, _ = pool.read(table, lengths, cu_seqlens=cu, tokens=150, dtype=torch.float32)
    y = _turn(k, f)
    c, step, low = quantize(y)
    y, got = y.unflatten(-1, (-1, 64)), got.unflatten(-1, (-1, 64))
    size = 2 * k.double().abs().amax(-1)[..., None, None]
    least = y.amin(-1, keepdim=True)
    either = (least - least.bfloat16().double()).abs() <= 2.0 ** -50 * size
    either[:, :, 1] = False  # not rotated
    assert torch.equal(torch.where(either, 0.0, got), torch.where(either, 0.0, (low + step * c).float()))
    assert bool(((got - y).abs() <= (step * (1 + 2.0 ** -7) + 2.0 ** -7 * low.abs() / 15) / 2 + 2.0 ** -24 * size).all())
    assert float(either.float().mean()) < 0.1
    pool.check_status()
