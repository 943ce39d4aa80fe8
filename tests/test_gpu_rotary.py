"""rotary (csrc/sq_rotary.cu) against 64-bit arithmetic.

Tolerances: the angle's fraction of a half turn is rounded to fp32 (pi 2^-25
radians), sine and cosine are within 2 units in the last place (2^-23), the
magnitude's product and the two products and the sum round three times (2^-24
each): ACC = 10 * 2^-24 of magnitude (|x1| + |x2|).  The 64-bit angle itself is
off by 2^-52 of its size, which counts at far positions.  Rounding is monotone,
so an output lies between the roundings of both ends of that interval.
"""
import pytest
import torch

from kv_reference import turn

pytestmark = pytest.mark.gpu

ACC = 10 * 2.0 ** -24


def _check(got, x, positions, frequencies, interleaved=False, magnitude=1.0, inverse=False):
    want = turn(x, positions, frequencies, interleaved, magnitude, inverse)
    n = frequencies.numel()
    size = torch.zeros_like(want)
    a = x.double().abs()
    one, two = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    angle = (positions.double()[:, None] * frequencies.double()).abs()[:, None]
    size[..., one] = size[..., two] = (a[..., one] + a[..., two]) * abs(magnitude) * (ACC + 2.0 ** -52 * angle)
    assert got.dtype == x.dtype and got.shape == x.shape
    inside = ((want - size).to(x.dtype) <= got) & (got <= (want + size).to(x.dtype))
    assert bool(inside.all()), (got[~inside], want[~inside])


def _data(tokens, heads, dim, dtype, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(tokens, heads, dim, generator=gen, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,turned", [(1, 1, 2, 2), (1, 32, 128, 128), (3, 5, 64, 32), (700, 1, 64, 64), (17, 3, 70, 34),
                                                     (40, 2, 6, 2), (33, 16, 256, 64), (2500, 4, 80, 80), (5, 300, 128, 64), (9, 2, 1024, 1024),
                                                     (6, 3, 77, 20)])
def test_shapes(tokens, heads, dim, turned, interleaved, dtype):
    from stepquant_b200.kernels.rotary import rotary, rotary_frequencies
    x = _data(tokens, heads, dim, dtype)
    positions = torch.randint(0, 4096, (tokens,), device="cuda", dtype=torch.int32 if heads % 2 else torch.int64)
    f = rotary_frequencies(turned)
    got = rotary(x, positions, f, interleaved=interleaved, magnitude=1.25)
    _check(got, x, positions, f, interleaved, 1.25)
    _check(rotary(x, positions, f, interleaved=interleaved, inverse=True), x, positions, f, interleaved, 1.0, True)
    same = x.clone()
    assert rotary(same, positions, f, interleaved=interleaved, magnitude=1.25, out=same) is same
    assert torch.equal(same, got)


@pytest.mark.parametrize("pad", [0, 8, 2, 1])
def test_strides_and_outputs(pad):
    """Heads inside a wider projection, tokens in another order of axes, an output that is a slice."""
    from stepquant_b200.kernels.rotary import rotary, rotary_frequencies
    f, positions = rotary_frequencies(64), torch.arange(50, device="cuda") * 37
    wide = _data(50, 1, 3 * 128 + pad, torch.bfloat16)[:, 0]
    x = wide[:, pad:pad + 256].unflatten(1, (2, 128))
    want = rotary(x.contiguous(), positions, f)
    assert torch.equal(rotary(x, positions, f), want)
    other = x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(rotary(other, positions, f), want)
    assert torch.equal(rotary(x.transpose(1, 2).contiguous().transpose(1, 2), positions, f), want)
    out = torch.full((50, 4, 128 + pad), 7.0, device="cuda", dtype=torch.bfloat16)
    part = out[:, 1:3, :128]
    assert rotary(x, positions, f, out=part) is part and torch.equal(part, want)
    assert bool((out[:, 0] == 7).all()) and bool((out[:, 3] == 7).all()) and bool((out[:, :, 128:] == 7).all())


@pytest.mark.parametrize("first", [2 ** 20 + 1, 2 ** 31 - 40, 10 ** 9 + 7, -5])
def test_far_positions(first):
    from stepquant_b200.kernels.rotary import rotary, rotary_frequencies
    x, f = _data(30, 2, 128, torch.float32), rotary_frequencies(128, 1e6)
    positions = torch.arange(first, first + 30, device="cuda")
    _check(rotary(x, positions, f), x, positions, f)


def test_relative_positions_and_nothing():
    """Products of rotated heads depend on the distance alone; empty calls; position zero copies."""
    from stepquant_b200.kernels.rotary import rotary, rotary_frequencies
    f = rotary_frequencies(64)
    q, k = _data(8, 2, 64, torch.float32, 1), _data(8, 2, 64, torch.float32, 2)
    at = torch.arange(8, device="cuda")
    near = (rotary(q, at + 7, f).double() * rotary(k, at, f).double()).sum(-1)
    far = (rotary(q, at + 10 ** 6 + 7, f).double() * rotary(k, at + 10 ** 6, f).double()).sum(-1)
    assert bool(((near - far).abs() <= 4 * ACC * (q.abs().sum(-1) * k.abs().amax(-1) * 2)).all())
    assert torch.equal(rotary(q, torch.zeros_like(at), f), q)
    assert rotary(q[:0], at[:0], f).shape == (0, 2, 64) and rotary(q[:, :0], at, f).shape == (8, 0, 64)
    assert torch.equal(rotary(q, at, f[:0]), q)
    assert torch.equal(rotary(q, at, f.float()), rotary(q, at, f.float().double()))
