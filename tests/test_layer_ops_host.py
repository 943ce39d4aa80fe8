"""Refusals of the layer operators that need no GPU: shapes, types and arguments are
checked before any launch, and tensors off the GPU are refused."""
import ctypes

import pytest
import torch

from stepquant_b200 import _native as N
from stepquant_b200.kernels.conv import causal_conv1d, causal_conv1d_extend, causal_conv1d_step
from stepquant_b200.kernels.matmul import matmul_fp8, quantize_weight_fp8
from stepquant_b200.kernels.norm import quantize_fp8, rms_norm, rms_norm_fp8
from stepquant_b200.kernels.scan import SelectiveStatePool, selective_scan, selective_scan_extend, selective_scan_step

ones = torch.ones
FP8 = torch.float8_e4m3fn


def test_packed_arguments_are_the_structures():
    """packer() lays the fields out as the ctypes Structure (and the C header) does."""
    for kind in (N.SqNormArgs, N.SqMatmulArgs, N.SqConvArgs, N.SqScanArgs):
        values = [i + 1 for i in range(len(kind._fields_))]
        assert N.packer(kind)(*values) == bytes(kind(*values))


def test_norm_refusals():
    x, w = ones(3, 8), ones(8)
    for bad in (lambda: rms_norm(x, ones(7)), lambda: rms_norm(x, None), lambda: rms_norm(x, w, ones(3, 7)),
                lambda: rms_norm(x, w, ones(3, 8).half()), lambda: rms_norm(x.double(), w), lambda: rms_norm(x, w.double()),
                lambda: rms_norm(x, w, eps=-1.0), lambda: rms_norm(x, w, eps=float("nan")), lambda: rms_norm_fp8(x, None),
                lambda: quantize_fp8(x.long()), lambda: rms_norm(ones(3, 0), ones(0)), lambda: rms_norm(torch.tensor(1.0), w),
                lambda: rms_norm(x, w), lambda: quantize_fp8(x)):  # the last two: not on a GPU
        with pytest.raises(ValueError):
            bad()


def test_matmul_refusals():
    x, w = ones(3, 32).to(FP8), ones(5, 32).to(FP8)
    sx, sw = ones(3, 1), ones(1, 1)
    with pytest.raises(NotImplementedError):
        matmul_fp8(ones(3, 24).to(FP8), sx, ones(5, 24).to(FP8), sw)
    for bad in (lambda: matmul_fp8(x, sx, ones(5, 16).to(FP8), sw), lambda: matmul_fp8(x, sx, w[0], sw),
                lambda: matmul_fp8(x, sx, w, sw, out_dtype=torch.float64), lambda: matmul_fp8(x, sx, w, sw),
                lambda: quantize_weight_fp8(ones(4))):
        with pytest.raises(ValueError):
            bad()


def test_conv_refusals():
    x, w = ones(5, 6), ones(6, 4)
    state = torch.zeros(2, 6, 3)
    with pytest.raises(NotImplementedError):
        causal_conv1d(x, ones(6, 5))
    for bad in (lambda: causal_conv1d(x, ones(7, 4)), lambda: causal_conv1d(x, w, ones(5)),
                lambda: causal_conv1d(x, w, activation="relu"), lambda: causal_conv1d(ones(2, 5, 6), w),
                lambda: causal_conv1d(x.long(), w), lambda: causal_conv1d(x, w), lambda: causal_conv1d(ones(6), w),
                lambda: causal_conv1d_step(x[None], state, w), lambda: causal_conv1d_step(x, state, w),
                lambda: causal_conv1d_extend(x, state, w, slots=torch.tensor([1]))):
        with pytest.raises(ValueError):
            bad()


def test_scan_refusals():
    u, a, b = ones(5, 6), -ones(6, 8), ones(5, 1, 8)
    with pytest.raises(NotImplementedError):
        selective_scan(u, u, -ones(6, 12), ones(5, 1, 12), ones(5, 1, 12))
    state = torch.zeros(5, 6, 8)
    for bad in (lambda: selective_scan(u, ones(4, 6), a, b, b), lambda: selective_scan(u, u.half(), a, b, b),
                lambda: selective_scan(u, u, a.half(), b, b), lambda: selective_scan(u, u, -ones(5, 8), b, b),
                lambda: selective_scan(u, u, a, ones(4, 1, 8), b), lambda: selective_scan(u, u, a, ones(5, 4, 8), ones(5, 4, 8)),
                lambda: selective_scan(u, u, a, b, ones(5, 2, 8)), lambda: selective_scan(u, u, a, b, b, d=ones(5)),
                lambda: selective_scan(u, u, a, b, b, z=ones(5, 5)), lambda: selective_scan(ones(2, 5, 6), u, a, b, b),
                lambda: selective_scan(u, u, a, b, b), lambda: selective_scan_step(state, u, u, a, b, b),
                lambda: selective_scan_step(state, u[None], u, a, b, b),
                lambda: selective_scan_extend(state, u, u, a, b, b, slots=torch.tensor([1])),
                lambda: SelectiveStatePool(0, 6, 8, device="cpu"), lambda: SelectiveStatePool(2, 6, 9, device="cpu"),
                lambda: SelectiveStatePool(2, 6, 8, taps=5, device="cpu"),
                lambda: SelectiveStatePool(2, 6, 8, dtype=torch.float64, device="cpu")):
        with pytest.raises(ValueError):
            bad()


def test_c_entries_refuse_before_launch():
    """Error codes of the C entries for arguments no launch should see; empty batches are no error."""
    lib, fake = N.lib(), 4096

    def code(entry, kind, **fields):
        return entry(ctypes.byref(kind(**fields)), None)

    norm = dict(x=fake, weight=fake, out=fake, rows=2, hidden=8, normalize=1, eps=1e-6, x_stride=8)
    assert lib.sq_rms_norm(None, None) == N.SQ_ERR_ARGUMENT
    for change, want in ((dict(x=None), 1), (dict(hidden=0), 1), (dict(rows=-1), 1), (dict(eps=-1.0), 1), (dict(dtype=3), 1),
                         (dict(residual=fake), 1), (dict(normalize=0), 1), (dict(x_stride=-8), 2), (dict(hidden=65537), 3),
                         (dict(rows=0, x=None), 0)):
        assert code(lib.sq_rms_norm, N.SqNormArgs, **{**norm, **change}) == want, change
    matmul = dict(x=fake, x_scale=fake, w=fake, w_scale=fake, out=fake, x_stride=32, w_stride=32, rows=2, width=3, hidden=32)
    for change, want in ((dict(w=None), 1), (dict(width=0), 1), (dict(dtype=-1), 1), (dict(hidden=40, x_stride=48), 3),
                         (dict(x=fake + 8), 2), (dict(x_stride=40), 2), (dict(w_stride=16), 2), (dict(rows=0), 0)):
        assert code(lib.sq_matmul_fp8, N.SqMatmulArgs, **{**matmul, **change}) == want, change
    conv = dict(x=fake, weight=fake, y=fake, cu_seqlens=fake, final_state=fake, x_stride=8, tokens=2, num_seqs=1, channels=8, taps=4)
    for change, want in ((dict(weight=None), 1), (dict(taps=5), 3), (dict(taps=1), 3), (dict(channels=0), 1), (dict(tokens=-1), 1),
                         (dict(slots=fake), 1), (dict(x_stride=-1), 2), (dict(cu_seqlens=None), 1), (dict(num_seqs=0), 0)):
        assert code(lib.sq_causal_conv, N.SqConvArgs, **{**conv, **change}) == want, change
    assert code(lib.sq_causal_conv_step, N.SqConvArgs, **{**conv, "final_state": None}) == N.SQ_ERR_ARGUMENT
    scan = dict(u=fake, dt=fake, b=fake, c=fake, a=fake, y=fake, cu_seqlens=fake, tokens=2, num_seqs=1, channels=8, states=16, groups=1)
    for change, want in ((dict(a=None), 1), (dict(states=12), 3), (dict(groups=3), 2), (dict(groups=0), 1), (dict(a=fake + 4), 2),
                         (dict(cu_seqlens=None), 1), (dict(u_stride=-1), 2), (dict(num_seqs=0), 0), (dict(initial_state=fake + 8), 2),
                         (dict(tokens=8192, workspace=fake, workspace_bytes=16), 5)):
        assert code(lib.sq_selective_scan, N.SqScanArgs, **{**scan, **change}) == want, change
    assert code(lib.sq_selective_scan_step, N.SqScanArgs, **scan) == N.SQ_ERR_ARGUMENT
    assert lib.sq_selective_scan_workspace_bytes(-1, 1, 8, 16, 1) == -1
    assert lib.sq_selective_scan_workspace_bytes(8192, 1, 2048, 16, 1) > 0
    assert lib.sq_selective_scan_workspace_bytes(16, 1, 2048, 16, 1) == 0


def test_pool_forms_need_slots():
    """Without slots a sequence's row would be its number, which may lie past the pool."""
    x, state, ends = ones(5, 6), torch.zeros(2, 6, 3), torch.tensor([0, 1, 3, 5])
    with pytest.raises(ValueError, match="slots"):
        causal_conv1d_extend(x, state, ones(6, 4), slots=None, cu_seqlens=ends)
    a, b = -ones(6, 8), ones(5, 1, 8)
    with pytest.raises(ValueError, match="slots"):
        selective_scan_extend(torch.zeros(2, 6, 8), x, x, a, b, b, slots=None, cu_seqlens=ends)
    pool = SelectiveStatePool(2, 6, 8, dtype=torch.float32, device="cpu")
    with pytest.raises(ValueError, match="slots"):
        pool.convolve(x, ones(6, 4), slots=None, cu_seqlens=ends)
    with pytest.raises(ValueError, match="slots"):
        pool.extend(x, x, a, b, b, None, ends)
    lib, fake = N.lib(), 4096
    conv = dict(x=fake, weight=fake, y=fake, cu_seqlens=fake, initial_state=fake, final_state=fake, x_stride=6, tokens=5,
                num_seqs=3, channels=6, taps=4, num_slots=2)
    scan = dict(u=fake, dt=fake, b=fake, c=fake, a=fake, y=fake, cu_seqlens=fake, initial_state=fake, final_state=fake, tokens=5,
                num_seqs=3, channels=6, states=8, groups=1, num_slots=2)
    for entry, kind, fields in ((lib.sq_causal_conv, N.SqConvArgs, conv), (lib.sq_causal_conv_step, N.SqConvArgs, conv),
                                (lib.sq_selective_scan, N.SqScanArgs, scan), (lib.sq_selective_scan_step, N.SqScanArgs, scan)):
        assert entry(ctypes.byref(kind(**fields)), None) == N.SQ_ERR_CAPACITY


def test_batches_are_not_one_stream():
    """Prompts are concatenated: a batch of several would run on from one into the next."""
    state, slots, ends = torch.zeros(3, 6, 3), torch.tensor([1, 2]), torch.tensor([0, 5, 10])
    for x in (ones(2, 5, 6), ones(2, 1, 5, 6), ones(6)):
        for call in (lambda: causal_conv1d(x, ones(6, 4), cu_seqlens=ends),
                     lambda: causal_conv1d_extend(x, state, ones(6, 4), slots=slots, cu_seqlens=ends)):
            with pytest.raises(ValueError, match="x: expected"):
                call()


def test_sizes_near_2_31():
    """Counts whose last tile would end past an int are refused, and those an int cannot hold are a ValueError."""
    lib, fake, near = N.lib(), 4096, 2 ** 31 - 64

    def code(entry, kind, **fields):
        return entry(ctypes.byref(kind(**fields)), None)

    matmul = dict(x=fake, x_scale=fake, w=fake, w_scale=fake, out=fake, x_stride=32, w_stride=32, rows=2, width=3, hidden=32)
    for change in (dict(rows=near), dict(width=near), dict(hidden=near, x_stride=near, w_stride=near)):
        assert code(lib.sq_matmul_fp8, N.SqMatmulArgs, **{**matmul, **change}) == N.SQ_ERR_UNSUPPORTED, change
    conv = dict(x=fake, weight=fake, y=fake, cu_seqlens=fake, final_state=fake, x_stride=8, tokens=near, num_seqs=1, channels=8, taps=4)
    assert code(lib.sq_causal_conv, N.SqConvArgs, **conv) == N.SQ_ERR_UNSUPPORTED
    scan = dict(u=fake, dt=fake, b=fake, c=fake, a=fake, y=fake, cu_seqlens=fake, tokens=near, num_seqs=1, channels=8, states=16, groups=1)
    assert code(lib.sq_selective_scan, N.SqScanArgs, **scan) == N.SQ_ERR_UNSUPPORTED
    for kind in (N.SqNormArgs, N.SqMatmulArgs, N.SqConvArgs, N.SqScanArgs):
        names = [name for name, _ in kind._fields_]
        with pytest.raises(ValueError, match="range"):
            N.packer(kind)(*[2 ** 31 if n in ("rows", "tokens") else 1 for n in names])
