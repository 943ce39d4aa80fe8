"""Refusals of the rotary and cache operators that need no GPU, and the frequencies."""
import ctypes
import math

import pytest
import torch

from stepquant_b200 import _native as N
from stepquant_b200.kernels.kv_cache import QuantizedKVPool, kv_append, kv_attention, kv_read
from stepquant_b200.kernels.rotary import rotary, rotary_frequencies

ones, zeros = torch.ones, torch.zeros


def test_packed_arguments_are_the_structures():
    for kind in (N.SqRotaryArgs, N.SqKvArgs, N.SqKvAttentionArgs):
        values = [i + 1 for i in range(len(kind._fields_))]
        assert N.packer(kind)(*values) == bytes(kind(*values))


def test_frequencies():
    f = lambda n, *a, **o: rotary_frequencies(n, *a, device="cpu", **o)  # noqa: E731
    plain = torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64)
    assert torch.allclose(f(64), plain, rtol=1e-15) and f(64).dtype == torch.float64
    assert torch.allclose(f(64, scaling="linear", factor=4), plain / 4, rtol=1e-15)
    longer = f(64, scaling="base", factor=8)
    assert longer[0] == 1 and math.isclose(longer[-1], plain[-1] / 8, rel_tol=1e-12)
    for kind in ("bands", "ramp"):
        g = f(64, scaling=kind, factor=8, original_length=4096, slow=1, fast=32)
        turns = 4096 * plain / (2 * math.pi)
        ratio = plain / g
        assert bool((ratio >= 1 - 1e-12).all()) and bool((ratio <= 8 + 1e-12).all()) and bool((ratio.diff() >= -1e-9).all())
        assert torch.allclose(ratio[turns > 40], ones(1).double()) and torch.allclose(ratio[turns < 0.6], 8 * ones(1).double())
    middle = f(64, scaling="bands", factor=8, original_length=4096, slow=1, fast=32)
    for i in range(32):
        t = 4096 * float(plain[i]) / (2 * math.pi)
        kept = min(max((t - 1) / 31, 0), 1)
        assert math.isclose(float(middle[i]), float(plain[i]) * (kept + (1 - kept) / 8), rel_tol=1e-12)
    for bad in (lambda: f(7), lambda: f(0), lambda: f(8, -1.0), lambda: f(8, factor=0), lambda: f(8, scaling="other"),
                lambda: f(8, scaling="bands"), lambda: f(8, scaling="ramp", original_length=100, slow=4, fast=2),
                lambda: f(8, float("nan")), lambda: f(8, scaling="ramp", base=1, original_length=100)):
        with pytest.raises(ValueError):
            bad()


def test_rotary_refusals():
    x, at, f = ones(3, 2, 8), torch.arange(3), ones(4).double()
    for bad in (lambda: rotary(x[0], at, f), lambda: rotary(x, at[:2], f), lambda: rotary(x, at.float(), f), lambda: rotary(x, at, ones(5)),
                lambda: rotary(x.long(), at, f), lambda: rotary(x.double(), at, f), lambda: rotary(x, at, None),
                lambda: rotary(x, at, f[None]), lambda: rotary(x, at, f, magnitude=math.inf), lambda: rotary(x, at, f, out=ones(3, 2, 6)),
                lambda: rotary(x, at, f, out=x.half()), lambda: rotary(x, at, f, out=ones(3, 8, 2).transpose(1, 2)),
                lambda: rotary(ones(3, 2, 1026), at, f), lambda: rotary(x, at, f)):  # the last: not on a GPU
        with pytest.raises(ValueError):
            bad()


def test_cache_refusals():
    data = zeros(4, 2, 1, 18 * 64, dtype=torch.uint8)
    k, q = ones(3, 2, 64), ones(3, 4, 64).half()
    table, lengths, cu = zeros(3, 1, dtype=torch.int32), ones(3, dtype=torch.int32), torch.tensor([0, 1, 2, 3])
    ok = (data, k, k, table, lengths)
    for bad in (lambda: kv_append(data[:, :, 0], *ok[1:]), lambda: kv_append(data.int(), *ok[1:]), lambda: kv_append(data[..., :1000], *ok[1:]),
                lambda: kv_append(data[:, :1], *ok[1:]), lambda: kv_append(data, k[:2], *ok[2:]), lambda: kv_append(data, k[0], *ok[2:]),
                lambda: kv_append(data, k, k.half(), table, lengths), lambda: kv_append(data, k.double(), k.double(), table, lengths),
                lambda: kv_append(data, k, k, table[:2], lengths), lambda: kv_append(data, k, k, table[0], lengths),
                lambda: kv_append(*ok, cu_seqlens=cu[:3]), lambda: kv_append(*ok, frequencies=ones(33)),
                lambda: kv_append(*ok, positions=ones(3)), lambda: kv_append(*ok, positions=torch.arange(2)),
                lambda: kv_append(*ok, magnitude=math.nan), lambda: kv_append(*ok, status=ones(1)), lambda: kv_append(*ok),
                lambda: kv_read(data, table, lengths, cu_seqlens=cu), lambda: kv_read(data, table, lengths, tokens=2),
                lambda: kv_read(data, table, lengths, tokens=-1, cu_seqlens=cu), lambda: kv_read(data, table, lengths, dtype=torch.int8),
                lambda: kv_read(data, table, lengths),
                lambda: kv_attention(q[0], data, table, lengths), lambda: kv_attention(q[:, :3], data, table, lengths),
                lambda: kv_attention(q[:, :0], data, table, lengths), lambda: kv_attention(ones(3, 4, 128).half(), data, table, lengths),
                lambda: kv_attention(q, data, table, lengths, scale=0.0), lambda: kv_attention(q, data, table, lengths, scale=-1.0),
                lambda: kv_attention(q, data, table, lengths, scale=math.inf), lambda: kv_attention(q, data, table, lengths, window=0),
                lambda: kv_attention(q[:2], data, table, lengths), lambda: kv_attention(q, data, table, lengths),
                lambda: QuantizedKVPool(0, 1, 64, device="cpu"), lambda: QuantizedKVPool(2, 0, 64, device="cpu"),
                lambda: QuantizedKVPool(2, 1, 64, page_size=24, device="cpu"), lambda: QuantizedKVPool(2, 1, 64, page_size=0, device="cpu")):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: kv_attention(q.float(), data, table, lengths), lambda: QuantizedKVPool(2, 1, 96, device="cpu")):
        with pytest.raises(NotImplementedError):
            bad()
    assert QuantizedKVPool(3, 2, 128, page_size=32, device="cpu").data.shape == (3, 2, 2, 18 * 128)


def test_c_entries_refuse_before_launch():
    lib, fake = N.lib(), 4096

    def code(entry, kind, **fields):
        return entry(ctypes.byref(kind(**fields)), None)

    rope = dict(x=fake, out=fake, positions=fake, frequencies=fake, tokens=2, heads=1, dim=8, turned=8, x_stride=8, x_head_stride=8,
                out_stride=8, out_head_stride=8, magnitude=1.0)
    assert lib.sq_rotary(None, None) == N.SQ_ERR_ARGUMENT
    for change, want in ((dict(x=None), 1), (dict(out=None), 1), (dict(positions=None), 1), (dict(turned=7), 2), (dict(turned=10), 2),
                         (dict(turned=-2), 1), (dict(dim=0), 1), (dict(dim=2000), 3), (dict(dtype=3), 1), (dict(x_stride=-8), 2),
                         (dict(tokens=2 ** 31 - 1), 3), (dict(tokens=-1), 1), (dict(tokens=0, x=None), 0), (dict(heads=0), 0)):
        assert code(lib.sq_rotary, N.SqRotaryArgs, **{**rope, **change}) == want, change
    kv = dict(k=fake, v=fake, data=fake, page_table=fake, lengths=fake, k_stride=64, k_head_stride=64, v_stride=64, v_head_stride=64,
              table_stride=1, num_pages=2, tokens=2, num_seqs=2, table_width=1, heads=1, dim=64, page_size=16)
    for entry in (lib.sq_kv_append, lib.sq_kv_read):
        assert entry(None, None) == N.SQ_ERR_ARGUMENT
        for change, want in ((dict(k=None), 1), (dict(v=None), 1), (dict(data=None), 1), (dict(page_table=None), 1), (dict(lengths=None), 1),
                             (dict(dim=96), 3), (dict(page_size=24), 2), (dict(page_size=0), 2), (dict(heads=0), 1), (dict(num_seqs=3), 1),
                             (dict(data=fake + 8), 2), (dict(table_stride=-1), 2), (dict(k_stride=-1), 2), (dict(dtype=5), 1),
                             (dict(num_pages=-1), 1), (dict(table_width=1 << 27), 3), (dict(tokens=0, num_seqs=0), 0)):
            assert code(entry, N.SqKvArgs, **{**kv, **change}) == want, change
    assert code(lib.sq_kv_append, N.SqKvArgs, **{**kv, "turned": 64}) == 1  # without frequencies
    assert code(lib.sq_kv_append, N.SqKvArgs, **{**kv, "turned": 66, "frequencies": fake}) == 2
    assert code(lib.sq_kv_read, N.SqKvArgs, **{**kv, "k": fake + 2}) == 2
    size = lib.sq_kv_attention_workspace_bytes(2, 2, 4, 1, 64)
    assert size > 0 and lib.sq_kv_attention_workspace_bytes(2, 2, 4, 1, 80) == -1 and lib.sq_kv_attention_workspace_bytes(0, 0, 4, 1, 64) == 0
    attend = dict(q=fake, data=fake, out=fake, page_table=fake, lengths=fake, workspace=fake, workspace_bytes=size, q_stride=256,
                  q_head_stride=64, table_stride=1, num_pages=2, tokens=2, num_seqs=2, table_width=1, q_heads=4, heads=1, dim=64,
                  page_size=16, dtype=1, scale=0.125)
    assert lib.sq_kv_attention(None, None) == N.SQ_ERR_ARGUMENT
    for change, want in ((dict(q=None), 1), (dict(out=None), 1), (dict(lengths=None), 1), (dict(dtype=0), 3), (dict(dtype=4), 1), (dict(dim=72), 3),
                         (dict(scale=0.0), 1), (dict(scale=math.nan), 1), (dict(scale=math.inf), 1), (dict(window=-1), 1), (dict(q_heads=0), 1),
                         (dict(heads=3), 2), (dict(q_stride=4), 2), (dict(q=fake + 2), 2), (dict(out=fake + 8), 2), (dict(workspace=None), 5),
                         (dict(workspace_bytes=size - 1), 5), (dict(num_seqs=1), 1), (dict(table_width=1 << 27), 3), (dict(page_size=8), 2), (dict(tokens=0, num_seqs=0), 0)):
        assert code(lib.sq_kv_attention, N.SqKvAttentionArgs, **{**attend, **change}) == want, change
