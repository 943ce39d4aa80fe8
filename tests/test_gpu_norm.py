"""rms_norm, rms_norm_fp8 and quantize_fp8 (csrc/sq_norm.cu) against 64-bit arithmetic.

Tolerances: the mean of n squares is off by at most ~80 roundings (64 serial
terms of a thread, then a tree), half of that after the root, plus the
reciprocal root's two and the products': REL = 64 * 2^-24 of |y|.  Rounding is
monotone, so an output lies between the roundings of both ends of that
interval; e4m3 values are within half a step of theirs (2^-4 relative, 2^-10
below 2^-6) of y / scale.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

REL = 64 * 2.0 ** -24


def _reference(x, weight, residual, eps=1e-6):
    h = x.double() + (0 if residual is None else residual.double())
    return h, h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()


def _close(got, want, dtype, rel=REL):
    off = want.abs() * rel + 1e-40
    inside = ((want - off).to(dtype) <= got) & (got <= (want + off).to(dtype))
    assert bool(inside.all()), (got[~inside], want[~inside])


def _blocks(y):
    pad = torch.nn.functional.pad(y, (0, -y.shape[-1] % 128))
    return pad.unflatten(-1, (-1, 128))


def _close_fp8(q, scale, y):
    want = _blocks(y).abs().amax(-1).clamp_min(1e-30) / 448
    assert scale.shape == want.shape
    assert bool(((scale.double() - want).abs() <= want * (REL + 2.0 ** -22)).all())
    v = (_blocks(y) / want[..., None]).flatten(-2)[..., :y.shape[-1]]
    limit = torch.clamp_min(v.abs() * 2.0 ** -4, 2.0 ** -10) + v.abs() * (2 * REL + 2.0 ** -21)
    got = q.double()
    assert bool(((got - v).abs() <= limit).all()), float(((got - v).abs() / limit).max())


def _data(rows, hidden, dtype, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x = (rand(rows, hidden) * torch.where(rand(hidden).abs() > 2.5, 30.0, 1.0)).to(dtype)
    return x, (rand(rows, hidden) * 3).to(dtype), (1 + 0.2 * rand(hidden)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,hidden", [(1, 1), (3, 7), (2, 8), (5, 127), (9, 128), (17, 129), (8, 256), (33, 512), (4, 520),
                                         (1, 5120), (3, 4100), (700, 1000), (601, 2056), (2, 8200), (600, 9001), (2, 65536)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm(rows, hidden, dtype, with_residual):
    from stepquant_b200.kernels.norm import rms_norm, rms_norm_fp8
    x, residual, weight = _data(rows, hidden, dtype)
    residual = residual if with_residual else None
    h, y = _reference(x, weight, residual)
    got = rms_norm(x, weight, residual)
    got8 = rms_norm_fp8(x, weight, residual)
    if with_residual:
        assert torch.equal(got[1], h.to(dtype) if dtype != torch.float32 else x + residual)
        assert torch.equal(got8[2], got[1])
    _close(got[0] if with_residual else got, y, dtype)
    assert got8[0].dtype == torch.float8_e4m3fn and got8[0].shape == x.shape
    _close_fp8(got8[0], got8[1], y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,hidden", [(2047, 1024), (2048, 520), (2049, 1000), (3001, 5120), (2500, 8192), (2100, 8200),
                                         (2100, 16384), (2100, 2052)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_many_rows(rows, hidden, dtype, with_residual):
    """Batches that take the persistent kernel (16-byte aligned rows) and those beside it, rows of a wider tensor."""
    from stepquant_b200.kernels.norm import rms_norm, rms_norm_fp8
    x, residual, weight = _data(rows, hidden + 8, dtype, 5)
    x, weight = x[:, 8:], weight[8:].float()
    residual = residual[:, :hidden] if with_residual else None
    h, y = _reference(x, weight, residual)
    got, got8 = rms_norm(x, weight, residual), rms_norm_fp8(x, weight, residual)
    if with_residual:
        want = h.to(dtype) if dtype != torch.float32 else x + residual
        assert torch.equal(got[1], want) and torch.equal(got8[2], want)
    _close(got[0] if with_residual else got, y, dtype)
    _close_fp8(got8[0], got8[1], y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,hidden", [(40003, 128), (40003, 96), (40003, 100), (40003, 127), (20001, 256), (20001, 204),
                                         (20001, 255), (20001, 512), (20001, 300), (20001, 509), (20001, 1)])
def test_many_short_rows(rows, hidden, dtype):
    """Short rows, half a warp or a warp each, more than the grid takes at once, the last turn not full."""
    from stepquant_b200.kernels.norm import quantize_fp8, rms_norm, rms_norm_fp8
    x, residual, weight = _data(rows, hidden, dtype, 7)
    h, y = _reference(x, weight, residual)
    want = h.to(dtype) if dtype != torch.float32 else x + residual
    got, got8 = rms_norm(x, weight, residual), rms_norm_fp8(x, weight, residual)
    assert torch.equal(got[1], want) and torch.equal(got8[2], want)
    _close(got[0], y, dtype)
    _close_fp8(got8[0], got8[1], y)
    _close_fp8(*quantize_fp8(x), x.double())
    _close(rms_norm(x, weight), _reference(x, weight, None)[1], dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,hidden", [(1, 1), (7, 130), (3, 4096), (640, 5120)])
def test_quantize(rows, hidden, dtype):
    from stepquant_b200.kernels.norm import quantize_fp8
    x, _, _ = _data(rows, hidden, dtype, 1)
    q, scale = quantize_fp8(x)
    _close_fp8(q, scale, x.double())


def test_weight_types_strides_and_batches():
    """fp32 weights with bf16 rows; rows of a wider tensor, 16-byte aligned or
    not; columns of a transposed one; more than two axes; a repeated row."""
    from stepquant_b200.kernels.norm import rms_norm, rms_norm_fp8
    x, residual, weight = _data(24, 1032, torch.bfloat16, 2)
    wide = torch.randn(24, 2 * 1032 + 3, device="cuda").bfloat16()
    for view in (wide[:, :1032], wide[:, 1032:2064], wide[:, 3:1035], torch.randn(1032, 24, device="cuda").bfloat16().T,
                 x[:1].expand(24, -1)):
        h, y = _reference(view, weight, residual)
        out, total = rms_norm(view, weight.float(), residual)
        _close(out, y, torch.bfloat16)
        assert torch.equal(total, h.bfloat16())
        q, scale, _ = rms_norm_fp8(view, weight.half().float(), residual)
        _close_fp8(q, scale, _reference(view, weight.half(), residual)[1])
    out = rms_norm(x.view(2, 3, 4, 1032), weight)
    assert out.shape == (2, 3, 4, 1032)
    _close(out.view(24, 1032), _reference(x, weight, None)[1], torch.bfloat16)
    q, scale = rms_norm_fp8(x.view(2, 12, 1032), weight)
    assert q.shape == (2, 12, 1032) and scale.shape == (2, 12, 9)


def test_extremes():
    """Zero rows, rows of the type's largest and smallest values, NaN and
    infinity: each row by itself, no other row touched."""
    from stepquant_b200.kernels.norm import quantize_fp8, rms_norm, rms_norm_fp8
    x, _, weight = _data(8, 640, torch.bfloat16, 3)
    x[1] = 0
    x[2] = 1e-30
    x[3] = 1e15
    x[4, 100] = float("nan")
    x[5, 639] = float("inf")
    y = rms_norm(x, weight)
    q, scale = rms_norm_fp8(x, weight)
    assert bool((y[1] == 0).all()) and bool((q[1].float() == 0).all()) and bool((scale[1] == torch.tensor(1e-30) / 448).all())
    assert bool(y[4].isnan().all()) and bool(q[4].float().isnan().all()) and bool(scale[4].isnan().all())
    assert bool(y[5, 639].isnan()) and bool(q[5, 639].float().isnan())
    for row in (0, 2, 3, 6, 7):
        _close(y[row:row + 1], _reference(x[row:row + 1], weight, None)[1], torch.bfloat16)
        _close_fp8(q[row:row + 1], scale[row:row + 1], _reference(x[row:row + 1], weight, None)[1])
    q, scale = quantize_fp8(x)
    assert bool(scale[4, 0].isnan()) and bool(scale[4, 1:].isfinite().all())
    assert bool(scale[5, 4].isinf()) and bool((q[5, 512:639].float() == 0).all())


def test_empty_and_refusals():
    from stepquant_b200.kernels.norm import rms_norm, rms_norm_fp8
    w = torch.ones(64, device="cuda")
    assert rms_norm(torch.empty(0, 64, device="cuda"), w).shape == (0, 64)
    assert rms_norm_fp8(torch.empty(0, 64, device="cuda"), w)[1].shape == (0, 1)
    with pytest.raises(ValueError):
        rms_norm(torch.ones(2, 64, device="cuda"), w.cpu())
    with pytest.raises(NotImplementedError):
        rms_norm(torch.ones(1, 65537, device="cuda"), torch.ones(65537, device="cuda"))


def test_other_stream_and_graph():
    """On a stream of the caller's, and replayed from a graph on new inputs."""
    from stepquant_b200.kernels.norm import rms_norm_fp8
    x, residual, weight = _data(16, 512, torch.bfloat16, 4)
    want = [t.float() for t in rms_norm_fp8(x, weight, residual)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = rms_norm_fp8(x, weight, residual)
    side.synchronize()
    assert all(torch.equal(g.float(), w) for g, w in zip(got, want))
    still = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rms_norm_fp8(still, weight, residual)
    still.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(g.float(), w) for g, w in zip(out, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,hidden", [(4100, 2048), (4099, 2051), (30000, 300), (30000, 128)])
def test_codes_are_rounded_quotients(rows, hidden, dtype):
    """Every code is e4m3 of y over the stored scale, a quotient rounded to fp32
    once (a product with the rounded reciprocal differs at some ties), and the
    same on every run.  y: x itself, or what the norm of fp32 rows returns."""
    from stepquant_b200.kernels.norm import quantize_fp8, rms_norm, rms_norm_fp8
    x, _, weight = _data(rows, hidden, dtype, 9)
    most = torch.full((), 448.0, device="cuda")  # a quotient of tensors: by a number, torch multiplies with its reciprocal

    def same(q, scale, y):
        wide = scale.repeat_interleave(128, 1)[:, :hidden]
        assert torch.equal(scale, torch.clamp_min(_blocks(y).abs().amax(-1), 1e-30) / most)
        assert torch.equal(q.view(torch.uint8), (y / wide).to(torch.float8_e4m3fn).view(torch.uint8))

    first = quantize_fp8(x)
    same(*first, x.float())
    again = quantize_fp8(x)
    assert torch.equal(first[0].view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(first[1], again[1])
    if dtype == torch.float32:
        same(*rms_norm_fp8(x, weight), rms_norm(x, weight))


@pytest.mark.parametrize("rows,hidden", [(5, 96), (5, 256), (40001, 300), (5, 509), (3, 1003), (700, 5120), (2100, 5120), (2, 65536)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_whose_squares_overflow(rows, hidden, dtype):
    """Finite rows up to the type's largest values are normed as any other; a row with an
    infinity is NaN there (and in its block's codes and scale) and 0 elsewhere; a NaN is all of its row."""
    from stepquant_b200.kernels.norm import rms_norm, rms_norm_fp8
    x, residual, weight = _data(rows, hidden, torch.float32, 21)
    x[0], x[1] = x[0].clamp(-40, 40) * 1e25, x[1].clamp(-40, 40) / 50 * 3e38
    x[-1], x[-1, -1] = x[-1].clamp(-40, 40), 2e38  # one large value
    x = x.to(dtype)
    weight = weight.clamp(0.5, 1.0).to(dtype)
    _, y = _reference(x, weight, None)
    y = torch.where(y.abs() < 2.0 ** -120, 0.0, y)  # below: no longer normal
    got, (q, scale) = rms_norm(x, weight), rms_norm_fp8(x, weight)
    off = y.abs() * REL + 2.0 ** -119
    inside = ((y - off).to(dtype) <= got) & (got <= (y + off).to(dtype))
    assert bool(inside.all()), (got[~inside], y[~inside])
    _close_fp8(q, scale, y)
    if rows == 2:
        return
    x[0, hidden // 2], x[2, hidden - 1] = float("inf"), float("nan")
    before = got
    got, (q, scale) = rms_norm(x, weight), rms_norm_fp8(x, weight)
    at = torch.arange(hidden, device="cuda")
    block = torch.arange(scale.shape[1], device="cuda") == hidden // 2 // 128
    assert bool(got[0, hidden // 2].isnan()) and not bool(got[0, at != hidden // 2].any())
    assert bool(q[0].float().isnan()[hidden // 2]) and not bool(q[0].float()[at // 128 != hidden // 2 // 128].any())
    assert bool(scale[0][block].isnan().all()) and bool((scale[0][~block] == torch.tensor(1e-30) / 448).all())
    assert bool(got[2].isnan().all()) and bool(q[2].float().isnan().all()) and bool(scale[2].isnan().all())
    assert torch.equal(got[1], before[1]) and torch.equal(got[3:], before[3:])


@pytest.mark.parametrize("rows", [3, 2100])
def test_residual_updated_in_place(rows):
    """The C entry with residual_out in residual's own buffer, ordinary and overflowing rows."""
    import ctypes
    from stepquant_b200 import _native as N
    from stepquant_b200.kernels.norm import rms_norm
    hidden = 1024
    x, residual, weight = _data(rows, hidden, torch.float32, 23)
    x[1] *= 1e22
    h, (y, _) = x + residual, rms_norm(x, weight, residual)
    assert bool(y[1].abs().amax() > 0.5)
    out = torch.empty_like(x)
    args = N.SqNormArgs(x.data_ptr(), residual.data_ptr(), weight.data_ptr(), residual.data_ptr(), out.data_ptr(), None, hidden,
                        hidden, rows, hidden, N.SQ_F32, N.SQ_F32, 1, 1e-6)
    N.check(N.lib().sq_rms_norm(ctypes.byref(args), N.stream_handle()))
    assert torch.equal(residual, h)
    assert torch.equal(out, y)

