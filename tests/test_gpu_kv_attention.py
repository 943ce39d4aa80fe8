"""kv_attention (csrc/sq_attention.cu) against 64-bit arithmetic over the cache's own values.

Tolerances, u = eps / 2 of the type: an output is rounded once (u of itself).  A
value is v = (m + 8 s) + s (c - 8), and its weight p s is rounded before it meets
c - 8 (u of p s |c - 8|, which can be far above p |v| where the two parts cancel);
prompts round p and v (2 u of p |v|).  Either is below 2 u W with W = sum p
(|m + 8 s| + s |c - 8|), taken as 4 u W for the sums in fp32.  (bf16 codes are
summed as 128 + c and 136 times the weights' sum is taken off: terms of up to 143
p s, whose roundings to fp32 stay where a value's two parts happen to vanish, m =
-8 s and c = 8.  At most 4 roundings of 2^-24 count there, as every further tile
of tokens brings other codes: 143 * 4 * 2^-24 < 2^-14 of p s, and that is 4 u
times 2^-8 s, so W takes 2^-8 s more.)  A score is off by
no more than 2^-12 of scale sum |q| |k| (queries and codes are exact in 16 bits;
the fp32 sums of their products, 128 times a code's step beside it, lose 2^-17),
which moves weights by E = 2^-11 of that at most.  In norm roundings
add up as independent ones do: three of u / sqrt(3) each, u together, taken as 2 u.
"""
import math

import pytest
import torch

from kv_reference import attend, cached
from test_gpu_kv_cache import _rand, _sequences

pytestmark = pytest.mark.gpu


def _check(got, q, data, table, lengths, counts, page, scale=None, window=None, holes=()):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    begin, off, norm = 0, 0.0, 0.0
    assert got.dtype == q.dtype and got.shape == q.shape
    for n, (length, count) in enumerate(zip(lengths, counts)):
        if count and (n < 20 or n % 16 == 0):
            part, out = q[begin:begin + count], got[begin:begin + count].double()
            if length <= 0:
                assert not bool(out.any())
            else:
                k, v, sizes = cached(data, table[n].tolist(), page, length)
                hidden = torch.zeros(length, dtype=torch.bool, device="cuda")
                for m, p in holes:
                    if m == n:
                        hidden[p * page:(p + 1) * page] = True
                want, size = attend(part, k, v, sizes, length - count, scale, window, hidden)
                heads = k.shape[0]
                most = torch.where(hidden[:, None], 0.0, k.abs()).nan_to_num().amax((0, 1))  # [D]
                error = scale * (part.double().abs() * most).sum(-1, keepdim=True) * 2.0 ** -11
                assert heads and bool(((out - want).abs() <= u * want.abs() + (4 * u + 2 * error) * size + 1e-30).all()), (
                    n, float(((out - want).abs() / (size + 1e-30)).max()))
                off, norm = off + float((out - want).square().sum()), norm + float(want.square().sum())
        begin += count
    assert math.sqrt(off) <= 2 * u * math.sqrt(norm) + 1e-30, math.sqrt(off / norm)


def _pool(pages, heads, page, dim, seed=0, dtype=torch.bfloat16):
    """A pool of quantized random keys and values, every page filled."""
    from stepquant_b200.kernels.kv_cache import QuantizedKVPool
    pool = QuantizedKVPool(pages, heads, dim, page_size=page)
    n = (pages - 1) * page
    k, v = (_rand(n, heads, dim, seed=seed + s).to(dtype) for s in (1, 2))
    pool.append(k, v, torch.arange(1, pages, device="cuda", dtype=torch.int32)[None], torch.tensor([n], device="cuda", dtype=torch.int32),
                cu_seqlens=torch.tensor([0, n], device="cuda", dtype=torch.int32))
    return pool


TOKENS = [  # lengths of single-token requests
    [1], [0], [16, 17, 15, 0, 1, 33], [1000], [700, 3, 129, 64, 2048, 31, 500, 1, 1, 90], [40] * 20, [20000, 5], [16] * 300,
]
HEADS = [(64, 2, 2), (64, 16, 1), (128, 8, 2), (128, 20, 2), (128, 3, 3), (256, 8, 1), (256, 32, 2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,q_heads,heads", HEADS)
@pytest.mark.parametrize("lengths", TOKENS, ids=lambda x: f"{len(x)}x{max(x)}")
def test_single_tokens(lengths, dim, q_heads, heads, dtype):
    page = 16 if dim == 64 else 64
    table, device_lengths, _, pages = _sequences(lengths, page)
    pool = _pool(pages, heads, page, dim, dtype=dtype)
    q = (2 * _rand(len(lengths), q_heads, dim, seed=5)).to(dtype)
    got = pool.attend(q, table, device_lengths)
    pool.check_status()
    _check(got, q, pool.data, table, lengths, [1] * len(lengths), page)


PROMPTS = [  # (lengths, new tokens)
    ([1], [1]), ([2, 5], [2, 3]), ([20, 0, 40, 7], [3, 0, 4, 7]), ([64], [64]), ([300, 17, 500], [300, 1, 129]), ([700], [5]),
    ([1000, 100], [513, 100]), ([3000], [20]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,q_heads,heads", HEADS)
@pytest.mark.parametrize("lengths,counts", PROMPTS, ids=lambda x: "-".join(map(str, x)))
def test_prompts(lengths, counts, dim, q_heads, heads, dtype):
    page = 48 if dim == 64 else 32
    table, device_lengths, cu, pages = _sequences(lengths, page, counts)
    pool = _pool(pages, heads, page, dim, dtype=dtype)
    q = (2 * _rand(sum(counts), q_heads, dim, seed=5)).to(dtype)
    got = pool.attend(q, table, device_lengths, cu_seqlens=cu)
    pool.check_status()
    _check(got, q, pool.data, table, lengths, counts, page)


@pytest.mark.parametrize("window", [1, 15, 16, 17, 100, 4096])
@pytest.mark.parametrize("lengths,counts", [([1, 16, 17, 500, 0, 4200], None), ([300, 40], [200, 40]), ([900, 20, 33], [30, 4, 1])])
@pytest.mark.parametrize("dim,q_heads,heads", [(64, 4, 2), (128, 8, 1), (256, 4, 2)])
def test_windows(window, lengths, counts, dim, q_heads, heads):
    page = 16
    table, device_lengths, cu, pages = _sequences(lengths, page, counts)
    pool = _pool(pages, heads, page, dim)
    counts = counts or [1] * len(lengths)
    q = (2 * _rand(sum(counts), q_heads, dim, seed=5)).bfloat16()
    got = pool.attend(q, table, device_lengths, cu_seqlens=cu, window=window)
    _check(got, q, pool.data, table, lengths, counts, page, window=window)
    # Pages that the window has left behind may be given back.
    freed = table.clone()
    for n, (length, count) in enumerate(zip(lengths, counts)):
        freed[n, :max(0, length - count - window + 1) // page] = 0
    assert torch.equal(pool.attend(q, freed, device_lengths, cu_seqlens=cu, window=window), got)
    pool.check_status()


@pytest.mark.parametrize("counts", [None, [1, 1, 90], [40, 3, 170]])
def test_what_is_hidden_may_be_anything(counts):
    """Bytes past the lengths, pages of others and pages <= 0 in the middle change nothing, whatever they hold."""
    lengths, page, dim = [61, 3, 200], 16, 128
    table, device_lengths, cu, pages = _sequences(lengths, page, counts)
    pool = _pool(pages, 2, page, dim)
    q = (2 * _rand(sum(counts or [1] * 3), 8, dim, seed=5)).bfloat16()
    table[2, 4], table[2, 6], table[0, 0] = 0, -3, 0
    want = pool.attend(q, table, device_lengths, cu_seqlens=cu)
    _check(want, q, pool.data, table.clamp_min(0), lengths, counts or [1] * 3, page, holes=[(2, 4), (2, 6), (0, 0)])
    k, v = (torch.full((page, 2, dim), x, device="cuda").bfloat16() for x in (math.nan, math.inf))
    ends = lambda n: torch.tensor([0, n], device="cuda", dtype=torch.int32)  # noqa: E731
    for n, length in enumerate(lengths):  # the rest of the last page
        last, rest = table[n:n + 1, (length - 1) // page:(length - 1) // page + 1], -length % page
        if rest:
            pool.append(k[:rest], v[:rest], last, torch.tensor([page], device="cuda"), cu_seqlens=ends(rest))
    used = set(table.flatten().tolist())
    for p in range(pages):
        if p not in used:
            pool.data[p] = 255
    pool.data[0] = 255
    assert torch.equal(pool.attend(q, table, device_lengths, cu_seqlens=cu), want)
    pool.check_status()


def test_values_that_are_not_finite_reach_those_who_see_them():
    lengths, page = [40, 40], 16
    table, device_lengths, _, pages = _sequences(lengths, page)
    pool = _pool(pages, 1, page, 64)
    q = _rand(2, 2, 64).bfloat16()
    before = pool.attend(q, table, device_lengths)
    bad = torch.full((1, 1, 64), math.nan, device="cuda").bfloat16()
    pool.append(bad, bad, table[1:], torch.tensor([7], device="cuda"))
    after = pool.attend(q, table, device_lengths)
    assert torch.equal(after[0], before[0]) and bool(after[1].isnan().all())


def test_padded_batches_and_flags():
    """Tokens of no sequence get zeros; lengths past the table and pages past the pool are left out and flagged."""
    lengths, page, dim = [50, 20], 16, 128
    table, device_lengths, _, pages = _sequences(lengths, page)
    pool = _pool(pages, 2, page, dim)
    for cu in ([3, 5, 9], [3, 33, 50]):
        tokens = cu[-1] + 7
        q = _rand(tokens, 4, dim).bfloat16()
        got = pool.attend(q, table, device_lengths, cu_seqlens=torch.tensor(cu, device="cuda"))
        assert not bool(got[:3].any()) and not bool(got[cu[-1]:].any())
        _check(got[3:cu[-1]], q[3:cu[-1]], pool.data, table, lengths, [cu[1] - cu[0], cu[2] - cu[1]], page)
    pool.check_status()
    q = _rand(2, 4, dim).bfloat16()
    pool.attend(q, table[:, :2], device_lengths)
    with pytest.raises(IndexError):
        pool.check_status()
    wrong = table.clone()
    wrong[0, 1] = pages
    got = pool.attend(q, wrong, device_lengths)
    with pytest.raises(IndexError):
        pool.check_status()
    _check(got, q, pool.data, table, lengths, [1, 1], page, holes=[(0, 1)])
    more = pool.attend(_rand(5, 4, dim).bfloat16(), table[:1], device_lengths[1:] - 17, cu_seqlens=torch.tensor([0, 5], device="cuda"))
    assert not bool(more[:2].any()) and bool(more[2:].any(-1).all())  # positions below zero see nothing
    assert pool.attend(q[:0], table[:0], device_lengths[:0]).shape == (0, 4, dim)
    empty = pool.attend(q, table[:0], device_lengths[:0], cu_seqlens=torch.tensor([0], device="cuda"))
    assert not bool(empty.any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts", [None, [300]])
def test_sharp_and_flat_scores(dtype, counts):
    """Scores in the hundreds, growing along the sequence (each maximum moves), and all alike."""
    lengths, page, dim = [900], 64, 128
    table, device_lengths, cu, pages = _sequences(lengths, page, counts)
    pool = _pool(pages, 1, page, dim)
    k, v = _rand(900, 1, dim, seed=3), _rand(900, 1, dim, seed=4)
    k = (0.1 * k + torch.linspace(-3, 3, 900, device="cuda")[:, None, None]).to(dtype)
    pool.append(k, v.to(dtype), table, device_lengths, cu_seqlens=torch.tensor([0, 900], device="cuda"))
    tokens = 1 if counts is None else 300
    q = (_rand(tokens, 4, dim, seed=6) + torch.tensor([3.0, -3.0, 0.0, 8.0], device="cuda")[:, None]).to(dtype)
    _check(pool.attend(q, table, device_lengths, cu_seqlens=cu), q, pool.data, table, lengths, counts or [1], page)
    _check(pool.attend(0 * q, table, device_lengths, cu_seqlens=cu), 0 * q, pool.data, table, lengths, counts or [1], page)
    _check(pool.attend(q, table, device_lengths, cu_seqlens=cu, scale=1e-3), q, pool.data, table, lengths, counts or [1], page, scale=1e-3)


def test_strided_queries():
    lengths, page, dim = [77, 200], 32, 128
    table, device_lengths, _, pages = _sequences(lengths, page)
    pool = _pool(pages, 2, page, dim)
    q = _rand(2, 8, dim).bfloat16()
    want = pool.attend(q, table, device_lengths)
    for pad in (8, 3):
        wide = torch.zeros(2, 8 * dim + 2 * pad, device="cuda", dtype=torch.bfloat16)
        wide[:, pad:pad + 8 * dim] = q.flatten(1)
        assert torch.equal(pool.attend(wide[:, pad:pad + 8 * dim].unflatten(1, (8, dim)), table, device_lengths), want)
    assert torch.equal(pool.attend(q.transpose(0, 1).contiguous().transpose(0, 1), table.long(), device_lengths.long()), want)


@pytest.mark.parametrize("dim,q_heads,heads", [(64, 128, 1), (128, 8, 2), (256, 128, 1), (128, 66, 1)])
def test_prompts_longer_than_what_is_held(dim, q_heads, heads):
    """More new tokens than a sequence holds: those at positions below zero see nothing; many heads a kv head."""
    page, length, count = 32, 150, 200
    table, device_lengths, _, pages = _sequences([length], page)
    pool = _pool(pages, heads, page, dim)
    q = _rand(count, q_heads, dim, seed=5).bfloat16()
    for window in (None, 40):
        got = pool.attend(q, table, device_lengths, cu_seqlens=torch.tensor([0, count], device="cuda"), window=window)
        assert not bool(got[:count - length].any())
        _check(got[count - length:], q[count - length:], pool.data, table, [length], [length], page, window=window)
    pool.check_status()


@pytest.mark.parametrize("factor", [2.0 ** -100, 2.0 ** -20, 2.0 ** 13])
@pytest.mark.parametrize("counts", [None, [130]])
def test_values_of_any_size(factor, counts):
    """Values far from one, some of them much larger than the others; tiny and large queries."""
    lengths, page, dim = [400], 16, 128
    table, device_lengths, cu, pages = _sequences(lengths, page, counts)
    pool = _pool(pages, 1, page, dim)
    k, v = _rand(400, 1, dim, seed=3).bfloat16(), _rand(400, 1, dim, seed=4) * factor
    v[::50] *= 100
    pool.append(k, v.bfloat16(), table, device_lengths, cu_seqlens=torch.tensor([0, 400], device="cuda"))
    tokens = 1 if counts is None else 130
    q = (_rand(tokens, 4, dim, seed=6) * torch.tensor([1.0, 1e-20, 20.0, 3.0], device="cuda")[:, None]).bfloat16()
    got = pool.attend(q, table, device_lengths, cu_seqlens=cu)
    _check(got / factor, q, _scaled(pool.data, factor), table, lengths, counts or [1], page)


def _scaled(data, factor):
    """The pool's bytes with values' scales and minima over `factor`, a power of two: values are near one again."""
    dim = data.shape[3] // 18
    out = data.clone()
    pairs = out[..., 17 * dim:].contiguous().view(torch.bfloat16)
    out[..., 17 * dim:] = (pairs.double() / factor).bfloat16().view(torch.uint8)
    return out
