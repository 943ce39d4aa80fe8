"""kv_attention where values, weights, keys or lengths leave the ordinary range.

Tolerances are those of test_gpu_kv_attention.py.  f16 outputs are 2^-14 and more in
size but for single channels, whose rounding by 2^-25 is 2^-11 of 2^-14, a small part of
4 u W, so no absolute term is needed.  The scores' share of the bound grows with the
sharpest key, the bound in norm does not.
"""
import math

import pytest
import torch

from kv_reference import attend, cached
from test_gpu_kv_attention import _check, _pool, _scaled
from test_gpu_kv_cache import _rand, _sequences

pytestmark = pytest.mark.gpu

BOTH = [torch.bfloat16, torch.float16]


def _fill(pool, k, v, table, lengths):
    ends = torch.tensor([0, k.shape[0]], device="cuda", dtype=torch.int32)
    pool.append(k, v, table, lengths, cu_seqlens=ends)


def _sharp(length, count, dim, values, boost, sink, dtype, q_heads=4, page=64, cache=None):
    """(pool, q, table, lengths, cu): one key in each of the first eight units of 32 lies `boost` above the others, whose
    scores have a deviation of one.  Each channel's values have a mean of their own, of size values[0], and the deviation
    values[1]; those of the sharp keys are 0 with `sink`."""
    table, lengths, cu, pages = _sequences([length], page, None if count is None else [count])
    pool = _pool(pages, 1, page, dim)
    tokens = count or 1
    k, v = _rand(length, 1, dim, seed=3), values[0] * _rand(1, 1, dim, seed=6) + values[1] * _rand(length, 1, dim, seed=4)
    q = _rand(tokens, q_heads, dim, seed=5)
    k[:, :, 0], q[:, :, 0] = 0, 8
    k[5:256:32, :, 0] = boost / (8 * dim ** -0.5)
    if sink:
        v[5:256:32] = 0
    cache = cache or dtype
    _fill(pool, k.to(cache), v.to(cache), table, lengths)
    return pool, q.to(dtype), table, lengths, cu


@pytest.mark.parametrize("count", [None, 3])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("values,boost,sink", [
    ((0.01, 0.003), 10, False), ((5e-4, 1e-4), 0, False), ((5e-4, 1e-4), 10, False), ((5e-4, 1e-4), 12, False),
    ((0.03, 0.01), 12, True), ((0.1, 0.03), 14, True), ((2.0, 0.6), 18, True)])
def test_small_weights_of_few_rows(values, boost, sink, dim, count):
    """Weights times values' scales far below 2^-14, in f16."""
    pool, q, table, lengths, cu = _sharp(16384, count, dim, values, boost, sink, torch.float16)
    got = pool.attend(q, table, lengths, cu_seqlens=cu)
    _check(got, q, pool.data, table, [16384], [count or 1], 64)


@pytest.mark.parametrize("count", [None, 3])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_large_scales_of_few_rows(dim, count):
    """f16 queries over a cache of bf16 values that f16 does not reach, whose average it does."""
    pool, q, table, lengths, cu = _sharp(16384, count, dim, (1e4, 2e5), 0, False, torch.float16, cache=torch.bfloat16)
    got = pool.attend(q, table, lengths, cu_seqlens=cu)
    _check(got, q, pool.data, table, [16384], [count or 1], 64)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("boost", [12, 14, 18])
def test_small_weights_of_prompts(boost, dim, dtype):
    """A few keys without values take nearly all the weight: the output is what the others give."""
    pool, q, table, lengths, cu = _sharp(16384, 200, dim, (64.0, 20.0), boost, True, dtype)
    got = pool.attend(q, table, lengths, cu_seqlens=cu)
    _check(got, q, pool.data, table, [16384], [200], 64)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("count", [None, 130])
@pytest.mark.parametrize("power", [-60, -30, -17, 17, 60, 100])
def test_keys_of_any_size(power, count, dim, dtype):
    """Keys from tiny to huge, of both signs, against a scale that brings the scores back."""
    page = 32
    table, lengths, cu, pages = _sequences([400], page, None if count is None else [count])
    pool = _pool(pages, 2, page, dim)
    k, v = _rand(400, 2, dim, seed=3) * 2.0 ** power, _rand(400, 2, dim, seed=4)
    _fill(pool, k.bfloat16(), v.bfloat16(), table, lengths)
    q, scale = (2 * _rand(count or 1, 8, dim, seed=5)).to(dtype), dim ** -0.5 * 2.0 ** -power
    got = pool.attend(q, table, lengths, cu_seqlens=cu, scale=scale)
    _check(got, q, pool.data, table, [400], [count or 1], page, scale=scale)


@pytest.mark.parametrize("count", [None, 130])
def test_scores_that_vanish(count):
    """Queries, keys and a scale whose product is nothing in fp32: every key has the same weight."""
    page, dim = 16, 128
    table, lengths, cu, pages = _sequences([400], page, None if count is None else [count])
    pool = _pool(pages, 1, page, dim)
    k, v = _rand(400, 1, dim, seed=3) * 1e-30, _rand(400, 1, dim, seed=4)
    _fill(pool, k.bfloat16(), v.bfloat16(), table, lengths)
    q = (_rand(count or 1, 4, dim, seed=5) * 1e-37).bfloat16()
    got = pool.attend(q, table, lengths, cu_seqlens=cu, scale=1e-20)
    _check(got, q, pool.data, table, [400], [count or 1], page, scale=1e-20)


@pytest.mark.parametrize("power", [-118, 104, 116, 120])
def test_values_of_prompts_of_any_size(power):
    page, dim, count = 16, 128, 130
    table, lengths, cu, pages = _sequences([400], page, [count])
    pool = _pool(pages, 1, page, dim)
    k, v = _rand(400, 1, dim, seed=3), _rand(400, 1, dim, seed=4) * 2.0 ** power
    _fill(pool, k.bfloat16(), v.bfloat16(), table, lengths)
    q = _rand(count, 4, dim, seed=6).bfloat16()
    got = pool.attend(q, table, lengths, cu_seqlens=cu)
    _check(got / 2.0 ** power, q, _scaled(pool.data, 2.0 ** power), table, [400], [count], page)


@pytest.mark.parametrize("q_heads,heads", [(8, 2), (1, 1)])
@pytest.mark.parametrize("pad,stride", [(0, 4), (8, 3), (3, 8), (1, 0)])
@pytest.mark.parametrize("cu", [False, True])
def test_one_token_of_any_stride(cu, pad, stride, q_heads, heads):
    """The strides of an axis of one are nobody's; a base off 16 bytes is copied."""
    page, dim = 32, 128
    table, lengths, ends, pages = _sequences([77], page, [1] if cu else None)
    pool = _pool(pages, heads, page, dim)
    q = _rand(1, q_heads, dim).bfloat16()
    want = pool.attend(q, table, lengths, cu_seqlens=ends)
    flat = torch.zeros(pad + q_heads * dim + stride, device="cuda", dtype=torch.bfloat16)
    flat[pad:pad + q_heads * dim] = q.flatten()
    wide = flat[None, pad:pad + q_heads * dim].as_strided((1, q_heads, dim), (q_heads * dim + stride, dim, 1))
    assert torch.equal(pool.attend(wide, table, lengths, cu_seqlens=ends), want)
    if q_heads == 1:
        wide = flat.as_strided((1, 1, dim), (dim, dim + stride, 1), pad)
        assert torch.equal(pool.attend(wide, table, lengths, cu_seqlens=ends), want)


@pytest.mark.parametrize("dim,q_heads,heads", [(64, 4, 2), (128, 8, 1), (256, 4, 2)])
@pytest.mark.parametrize("window", [30, 100, 1000])
@pytest.mark.parametrize("count", [None, 5, 60])
def test_windows_past_the_table(count, window, dim, q_heads, heads):
    """Tokens past the page table see what their own window reaches of it."""
    page, held, length = 16, 400, 421
    table, _, _, pages = _sequences([held], page)
    table = table[:, :held // page].contiguous()
    pool = _pool(pages, heads, page, dim)
    tokens = count or 1
    q = (2 * _rand(tokens, q_heads, dim, seed=5)).bfloat16()
    cu = None if count is None else torch.tensor([0, count], device="cuda", dtype=torch.int32)
    got = pool.attend(q, table, torch.tensor([length], device="cuda", dtype=torch.int32), cu_seqlens=cu, window=window).double()
    with pytest.raises(IndexError):
        pool.check_status()
    k, v, sizes = cached(pool.data, table[0].tolist(), page, held)
    want, size = attend(q, k, v, sizes, length - tokens, dim ** -0.5, window)
    u = torch.finfo(q.dtype).eps / 2
    error = dim ** -0.5 * (q.double().abs() * k.abs().amax((0, 1))).sum(-1, keepdim=True) * 2.0 ** -11
    assert bool(((got - want).abs() <= u * want.abs() + (4 * u + 2 * error) * size).all())
    assert float((got - want).norm()) <= 2 * u * float(want.norm())


@pytest.mark.parametrize("page,lengths,window", [(16, [16, 33, 1, 80], None), (48, [48, 40, 144, 100], None), (16, [100, 65, 16, 500], 20)])
@pytest.mark.parametrize("count", [None, 2])
def test_entries_that_hold_no_token_of_the_sequence(page, lengths, window, count):
    """What a table holds past a sequence's last page, or in front of its window, may be anything."""
    counts = None if count is None else [min(count, n) for n in lengths]
    table, device_lengths, cu, pages = _sequences(lengths, page, counts)
    pool = _pool(pages, 2, page, 128)
    q = _rand(sum(counts or [1] * len(lengths)), 8, 128, seed=5).bfloat16()
    want = pool.attend(q, table, device_lengths, cu_seqlens=cu, window=window)
    for n, length in enumerate(lengths):
        table[n, -(-length // page):] = 2 ** 31 - 1
        if window is not None:
            table[n, :max(0, length - (1 if counts is None else counts[n]) - window + 1) // page] = pages + 5
    assert torch.equal(pool.attend(q, table, device_lengths, cu_seqlens=cu, window=window), want)
    pool.check_status()


@pytest.mark.parametrize("dim,q_heads,heads", [(64, 8, 2), (128, 16, 4), (256, 8, 2)])
@pytest.mark.parametrize("lengths,counts", [([4000] * 40 + [17, 0, 300], None), ([3000, 900, 40], [700, 1, 33]), ([6000], [300])],
                         ids=["tokens", "both", "prompt"])
def test_waits_that_run_out(lengths, counts, dim, q_heads, heads):
    """Device waits limited to one look or a few clocks give up in the middle of copies and products: every output
    is what it should be or NaN, NaN only where the status is flagged, and the calls after are whole."""
    import ctypes
    from stepquant_b200 import _native as N
    page = 64
    table, device_lengths, cu, pages = _sequences(lengths, page, counts)
    pool = _pool(pages, heads, page, dim)
    tokens = sum(counts or [1] * len(lengths))
    q = _rand(tokens, q_heads, dim, seed=5).bfloat16()
    want = pool.attend(q, table, device_lengths, cu_seqlens=cu)
    flush = torch.empty(1 << 26, device="cuda")
    size = N.lib().sq_kv_attention_workspace_bytes(tokens, len(lengths), q_heads, heads, dim)
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    seen = 0
    for limit in (-1, -1, -1, -1, 1, 1000, 100000):
        out, status = torch.full_like(want, 7.0), torch.zeros(1, device="cuda", dtype=torch.int32)
        flush.zero_()  # the pages leave L2: copies take longer
        args = N.SqKvAttentionArgs(q.data_ptr(), pool.data.data_ptr(), out.data_ptr(), table.data_ptr(), device_lengths.data_ptr(),
                                   N.address(cu), status.data_ptr(), workspace.data_ptr(), size, q.stride(0), q.stride(1),
                                   table.stride(0), pages, tokens, len(lengths), table.shape[1], q_heads, heads, dim, page, N.SQ_BF16,
                                   0, dim ** -0.5, limit)
        N.check(N.lib().sq_kv_attention(ctypes.byref(args), N.stream_handle()))
        gone = out.isnan()
        assert torch.equal(out[~gone], want[~gone])
        flagged = int(status) == N.SQ_STATUS_TIMEOUT
        assert flagged or (not bool(gone.any()) and int(status) == 0)
        seen += bool(gone.any())
        assert torch.equal(pool.attend(q, table, device_lengths, cu_seqlens=cu), want)
        pool.check_status()
    assert seen  # a copy or a product that was just begun is not there at one look


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim,q_heads", [(64, 2), (128, 4), (256, 7)])
@pytest.mark.parametrize("lengths,counts", [([31, 40, 230], [9, 12, 8]), ([1, 36], [1, 4]), ([70, 33], [3, 2]), ([300], [130])])
@pytest.mark.parametrize("scale", [0.5, 1.0, 30.0, 1e6, 1e20])
def test_large_scales_of_scores(scale, lengths, counts, dim, q_heads, dtype):
    """A scale above one over small keys, where some tokens see nothing of what others in their block see."""
    page = 32
    table, device_lengths, cu, pages = _sequences(lengths, page, counts)
    pool = _pool(pages, 1, page, dim)
    k, v = (_rand((pages - 1) * page, 1, dim, seed=s) for s in (3, 4))
    ends = torch.tensor([0, k.shape[0]], device="cuda", dtype=torch.int32)
    pool.append((k * dim ** -0.5 / scale).bfloat16(), v.bfloat16(), torch.arange(1, pages, device="cuda")[None], ends[1:], cu_seqlens=ends)
    q = _rand(sum(counts), q_heads, dim, seed=5).to(dtype)
    got = pool.attend(q, table, device_lengths, cu_seqlens=cu, scale=scale)
    _check(got, q, pool.data, table, lengths, counts, page, scale=scale)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim,q_heads", [(64, 16), (128, 16), (128, 256), (256, 16)])
@pytest.mark.parametrize("scale", [0.05, 1.0])
def test_long_sums(scale, dim, q_heads, dtype):
    """Thousands of tokens a warp: more requests and heads than CTAs, each of one long document that all share."""
    length, page, seqs, heads = 32768, 64, 20, 16
    table, lengths, _, pages = _sequences([length], page)
    pool = _pool(pages, heads, page, dim)
    k, v = _rand(length, heads, dim, seed=3), _rand(length, heads, dim, seed=4)
    _fill(pool, k.to(dtype), v.to(dtype), table, lengths)
    q = _rand(seqs, q_heads, dim, seed=5).to(dtype)
    got = pool.attend(q, table.expand(seqs, -1), lengths.expand(seqs), scale=scale * dim ** -0.5)
    pool.check_status()
    for n in (0, 7):
        _check(got[n:n + 1], q[n:n + 1], pool.data, table, [length], [1], page, scale=scale * dim ** -0.5)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim,count", [(64, None), (128, None), (128, 7), (256, None), (128, 40)])
@pytest.mark.parametrize("skewed", [False, True])
@pytest.mark.parametrize("spread", [0.0, 1e-4, 3e-4, 1e-3, 3e-3, 0.03])
def test_nearly_flat_scores(spread, skewed, dim, count, dtype):
    """Weights alike, whose roundings are then alike too, over values that all but cancel (in one channel of skewed
    groups they do not: the extremes are far from symmetric).  What is rounded has to be what cancels."""
    length, page = 20000, 64
    table, lengths, cu, pages = _sequences([length], page, None if count is None else [count])
    pool = _pool(pages, 1, page, dim)
    k, v = _rand(length, 1, dim, seed=3), _rand(length, 1, dim, seed=4)
    if skewed:
        v = v.exp() - math.exp(0.5)
    _fill(pool, k.bfloat16(), v.bfloat16(), table, lengths)
    q = _rand(count or 1, 4, dim, seed=5).to(dtype)
    scale = max(spread, 1e-9) * dim ** -0.5
    got = pool.attend(q, table, lengths, cu_seqlens=cu, scale=scale)
    _check(got, q, pool.data, table, [length], [count or 1], page, scale=scale)


@pytest.mark.parametrize("scale", [0.05, 1.0])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_sums_of_skewed_values(dim, scale):
    """Sums of codes about the middle that cancel against the middle's, over 16000 tokens a warp, in f16."""
    length, page, seqs, heads = 131072, 64, 20, 16
    table, lengths, _, pages = _sequences([length], page)
    pool = _pool(pages, heads, page, dim)
    k, v = _rand(length, heads, dim, seed=3), _rand(length, heads, dim, seed=4).exp() - math.exp(0.5)
    _fill(pool, k.half(), v.half(), table, lengths)
    q = _rand(seqs, heads, dim, seed=5).half()
    got = pool.attend(q, table.expand(seqs, -1), lengths.expand(seqs), scale=scale * dim ** -0.5)
    del k, v
    _check(got[3:4], q[3:4], pool.data, table, [length], [1], page, scale=scale * dim ** -0.5)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("counts", [None, [1, 1, 7], [40, 3, 170]])
@pytest.mark.parametrize("window", [None, 50])
def test_hidden_bytes_in_f16(window, counts, dim):
    """Bytes past the lengths, in front of the window, of other pages and of pages <= 0 change no bit of what is seen,
    whatever they hold."""
    lengths, page = [61, 3, 200], 16
    table, device_lengths, cu, pages = _sequences(lengths, page, counts)
    pool = _pool(pages, 2, page, dim, dtype=torch.float16)
    q = (2 * _rand(sum(counts or [1] * 3), 8, dim, seed=5)).half()
    table[2, 10], table[2, 11] = 0, -3
    want = pool.attend(q, table, device_lengths, cu_seqlens=cu, window=window)
    assert bool(want.isfinite().all())
    for fill in (255, 0x7F, 0xBF, 0x3C):
        new = torch.full_like(pool.data, fill)
        for n, length in enumerate(lengths):
            first = 0 if window is None else max(0, length - (1 if counts is None else counts[n]) - window + 1)
            for p in range(first // page, -(-length // page)):
                held = int(table[n, p])
                if held > 0:
                    new[held] = pool.data[held]
                    rest = length - p * page
                    if rest < page:  # the pairs of the tokens past the end (their codes share no word with others)
                        for u in range(rest, page):
                            row = 2 * (u % 4) + u // 4 % 2 + u // 8 * 8
                            for at in (8 * dim, 17 * dim):
                                new[held, :, :, at + row * dim // 16:at + (row + 1) * dim // 16] = fill
        old, pool.data = pool.data, new
        got = pool.attend(q, table, device_lengths, cu_seqlens=cu, window=window)
        pool.data = old
        assert torch.equal(got, want), fill
