"""matmul_fp8 (csrc/sq_matmul.cu) against 64-bit arithmetic.

Tolerances: products of e4m3 values are exact in fp32.  A block's 128 are summed
by the tensor cores with at most 2^-13 of the sum of their magnitudes lost
(alignment to the largest term, at least 14 bits kept per step of 32); scaling,
the sum over the blocks and the residual add at most (blocks + 4) roundings of
2^-24 of the sum of magnitudes.  Rounding is monotone, so an output lies between
the roundings of both ends of that interval.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _expand(scale, rows, shape):
    return scale.double().repeat_interleave(rows, 0)[:shape[0]].repeat_interleave(128, 1)[:, :shape[1]]


def _reference(x, sx, w, sw, residual):
    a, b = x.double() * _expand(sx, 1, x.shape), w.double() * _expand(sw, 128, w.shape)
    y, size = a @ b.T, a.abs() @ b.abs().T
    if residual is not None:
        y, size = y + residual.double(), size + residual.double().abs()
    return y, size


def _close(got, x, sx, w, sw, residual=None, core=2.0 ** -13):
    want, size = _reference(x, sx, w, sw, residual)
    off = size * (core + (sx.shape[1] + 4) * 2.0 ** -24) + 1e-30
    inside = ((want - off).to(got.dtype) <= got) & (got <= (want + off).to(got.dtype))
    assert bool(inside.all()), (int((~inside).sum()), got[~inside][:8], want[~inside][:8])


def _data(rows, width, hidden, seed=0):
    from stepquant_b200.kernels.matmul import quantize_weight_fp8
    from stepquant_b200.kernels.norm import quantize_fp8
    gen = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(rows, hidden, generator=gen, device="cuda")
    x *= torch.where(torch.rand(hidden, generator=gen, device="cuda") < 0.02, 20.0, 1.0)
    w = torch.randn(width, hidden, generator=gen, device="cuda") * hidden ** -0.5
    w *= torch.rand(width, 1, generator=gen, device="cuda") + 0.1
    return (*quantize_fp8(x), *quantize_weight_fp8(w))


# Rows on both sides of every switch of kernel and tile; widths and depths that no tile divides.
SHAPES = [(1, 1, 16), (1, 128, 128), (3, 130, 144), (16, 300, 256), (17, 100, 2048), (33, 1000, 400), (64, 256, 1024),
          (65, 8, 1040), (128, 640, 128), (129, 136, 272), (200, 1, 128), (300, 777, 1008), (513, 2050, 384),
          (1000, 1500, 640), (140, 20000, 96), (2500, 260, 128), (4, 9000, 640), (1, 5120, 4096)]


@pytest.mark.parametrize("rows,width,hidden", [(8, 16384, 8192), (16, 9000, 8192), (32, 16384, 4096), (64, 5000, 8192),
                                               (128, 5120, 8192), (512, 5120, 8192), (512, 6500, 8192), (700, 8200, 8192)])
def test_deep_products(rows, width, hidden):
    """Many blocks a CTA, weights that do not stay in L2: the copies of different blocks land in any order."""
    from stepquant_b200.kernels.matmul import matmul_fp8
    x, sx, w, sw = _data(rows, width, hidden, 7)
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    flush = torch.empty(1 << 26, device="cuda")
    want = None
    for _ in range(6):
        flush.zero_()
        got = matmul_fp8(x, sx, w, sw, status=status)
        want = got if want is None else want
        assert torch.equal(got, want)
    _close(want, x, sx, w, sw)
    assert int(status) == 0


@pytest.mark.parametrize("rows,width,hidden", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_product(rows, width, hidden, dtype):
    from stepquant_b200.kernels.matmul import matmul_fp8
    x, sx, w, sw = _data(rows, width, hidden)
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    got = matmul_fp8(x, sx, w, sw, out_dtype=dtype, status=status)
    assert got.shape == (rows, width) and got.dtype == dtype
    _close(got, x, sx, w, sw)
    residual = torch.randn(rows, width + 3, device="cuda").to(dtype)[:, :width]
    _close(matmul_fp8(x, sx, w, sw, residual=residual, out_dtype=dtype), x, sx, w, sw, residual)
    residual = residual.contiguous()
    _close(matmul_fp8(x, sx, w, sw, residual=residual, out_dtype=dtype), x, sx, w, sw, residual)
    assert int(status) == 0


@pytest.mark.parametrize("rows,width,hidden", [(8, 384, 640), (300, 384, 640)])
def test_whole_numbers_are_exact(rows, width, hidden):
    """Small whole values, scales that are powers of two of the block's index:
    every partial sum fits 14 bits, so the result is exact and shows any block
    or row that met another's scale."""
    from stepquant_b200.kernels.matmul import matmul_fp8
    gen = torch.Generator("cuda").manual_seed(1)
    x = torch.randint(-4, 5, (rows, hidden), generator=gen, device="cuda").float()
    w = torch.randint(-4, 5, (width, hidden), generator=gen, device="cuda").float()
    sx = 2.0 ** torch.randint(-3, 4, (rows, hidden // 128), generator=gen, device="cuda").float()
    sw = 2.0 ** torch.randint(-3, 4, (width // 128, hidden // 128), generator=gen, device="cuda").float()
    x, w = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
    got = matmul_fp8(x, sx, w, sw, out_dtype=torch.float32)
    assert torch.equal(got.double(), _reference(x, sx, w, sw, None)[0])


def test_all_e4m3_values():
    """Every finite e4m3 value against one-hot rows comes back as itself."""
    from stepquant_b200.kernels.matmul import matmul_fp8
    codes = torch.arange(256, device="cuda", dtype=torch.uint8)
    codes = codes[(codes & 0x7f) != 0x7f].view(torch.float8_e4m3fn)  # 254 values
    x = torch.zeros(254, 256, device="cuda")
    x[:, :254] = torch.eye(254, device="cuda")
    w = torch.zeros(3, 256, device="cuda")
    w[:, :254] = codes.float()
    one = torch.ones
    for rows in (254, 7):
        got = matmul_fp8(x[:rows].to(torch.float8_e4m3fn), one(rows, 2, device="cuda"), w.to(torch.float8_e4m3fn),
                         one(1, 2, device="cuda"), out_dtype=torch.float32)
        assert torch.equal(got, w[:, :rows].T)


def test_nan_scale_extremes():
    """A NaN code reaches its row or column only; huge and zero scales."""
    from stepquant_b200.kernels.matmul import matmul_fp8
    for rows in (9, 200):
        x, sx, w, sw = _data(rows, 260, 256, 2)
        xf = x.float()
        xf[3, 200] = float("nan")
        x = xf.to(torch.float8_e4m3fn)
        sx[5, 0], sx[6] = 1e30, 0
        got = matmul_fp8(x, sx, w, sw, out_dtype=torch.float32)
        assert bool(got[3].isnan().all()) and bool((got[6] == 0).all())
        keep = [i for i in range(rows) if i != 3]
        _close(got[keep], x[keep], sx[keep], w, sw)


def test_strided_operands_and_batches():
    from stepquant_b200.kernels.matmul import matmul_fp8
    for rows in (24, 150):
        x, sx, w, sw = _data(rows, 256, 384, 3)
        want = matmul_fp8(x, sx, w, sw)
        for pad in (16, 7):
            wide = torch.zeros(rows, 384 + 2 * pad, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
            wide[:, pad:pad + 384] = x
            assert torch.equal(matmul_fp8(wide[:, pad:pad + 384], sx, w, sw), want)
        wt = w.view(torch.uint8).T.contiguous().T.view(torch.float8_e4m3fn)  # columns contiguous: copied
        assert torch.equal(matmul_fp8(x, sx.T.contiguous().T, wt, sw), want)
        assert torch.equal(matmul_fp8(x.view(2, -1, 384), sx.view(2, -1, 3), w, sw).view(rows, 256), want)
    assert matmul_fp8(x[:0], sx[:0], w, sw).shape == (0, 256)


def test_repeatability_stream_and_graph():
    """Split sums join in a fixed order: the same bits again, on another stream and from a graph."""
    from stepquant_b200.kernels.matmul import matmul_fp8
    for rows in (5, 100, 700):
        x, sx, w, sw = _data(rows, 1000, 2048, 4)
        want = matmul_fp8(x, sx, w, sw)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = matmul_fp8(x, sx, w, sw)
        side.synchronize()
        assert torch.equal(got, want)
        still = torch.zeros(rows, 2048, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = matmul_fp8(still, sx, w, sw)
        still.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_weight_quantization():
    from stepquant_b200.kernels.matmul import quantize_weight_fp8
    w = torch.randn(200, 300, device="cuda")
    w[128:, 256:] = 0
    q, scale = quantize_weight_fp8(w)
    assert q.shape == w.shape and scale.shape == (2, 3) and bool(scale[1, 2] > 0)
    back = q.double() * _expand(scale, 128, w.shape)
    assert bool(((back - w.double()).abs() <= torch.clamp_min(w.double().abs() * 2.0 ** -4, 1e-4)).all())


@pytest.mark.parametrize("rows,width,hidden", [(8, 16384, 8192), (30, 5000, 4096), (60, 2000, 8192), (128, 9001, 4096), (129, 700, 8192),
                                               (300, 2050, 8192), (512, 6500, 8192), (700, 8200, 4096), (4096, 5120, 1024)])
def test_waits_that_run_out(rows, width, hidden):
    """Device waits limited to one try or a few clocks give up in the middle of copies and products: every
    output is what it should be or NaN, NaN only where the status is flagged (and, up to 128 rows,
    then; a tile's warp without rows of its own may give up alone), and the calls after are whole."""
    import ctypes
    from stepquant_b200 import _native as N
    from stepquant_b200.kernels.matmul import matmul_fp8
    x, sx, w, sw = _data(rows, width, hidden, 31)
    want = matmul_fp8(x, sx, w, sw)
    flush = torch.empty(1 << 26, device="cuda")
    seen = 0
    for limit in (-1, -1, 1, 300, 1000, 3000, 10000, 100000):
        out, status = torch.zeros_like(want), torch.zeros(1, device="cuda", dtype=torch.int32)
        flush.zero_()  # the operands leave L2: the first copies take longer than a try
        args = N.SqMatmulArgs(x.data_ptr(), sx.data_ptr(), w.data_ptr(), sw.data_ptr(), None, out.data_ptr(), status.data_ptr(),
                              hidden, hidden, 0, rows, width, hidden, N.SQ_BF16, limit)
        N.check(N.lib().sq_matmul_fp8(ctypes.byref(args), N.stream_handle()))
        gone = out.isnan()
        assert torch.equal(out[~gone], want[~gone])
        flagged = int(status) == N.SQ_STATUS_TIMEOUT
        assert flagged or (not bool(gone.any()) and int(status) == 0)
        assert bool(gone.any()) or not flagged or rows > 128
        seen += bool(gone.any())
        assert torch.equal(matmul_fp8(x, sx, w, sw, status=status.zero_()), want) and int(status) == 0
    assert seen or width * hidden < 1 << 25  # thousands of waits with one try each


@pytest.mark.parametrize("rows,width,hidden", [(5, 1000, 4096), (16, 128, 8192), (30, 5120, 2048), (60, 300, 4096), (100, 9000, 1024)])
def test_few_rows_on_few_sms(rows, width, hidden):
    """Clusters on a stream of 16 SMs, K split over fewer CTAs than on the whole GPU: the same bounds."""
    from stepquant_b200.kernels.matmul import matmul_fp8
    from stepquant_b200.kernels.resources import writeback_resources
    x, sx, w, sw = _data(rows, width, hidden, 6)
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    stream = writeback_resources("cuda", 16).stream
    with torch.cuda.stream(stream):
        got = matmul_fp8(x, sx, w, sw, out_dtype=torch.float32, status=status)
    stream.synchronize()
    _close(got, x, sx, w, sw)
    assert int(status) == 0
