"""kv_append and kv_read (csrc/sq_kv.cu) against the definition in 64 bits.

Codes, scales and minima are those of exact arithmetic, so bytes and values are
equal: a value read in fp32 is m + s c rounded once.
"""
import math

import pytest
import torch

from kv_reference import quantize, tile_places, turn, unpack, value

pytestmark = pytest.mark.gpu


def _rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")


def _sequences(lengths, page, counts=None, spare=2, seed=0):
    """(table, lengths, cu, pages): pages in no order, the table two columns wider than it need be."""
    need = [-(-max(n, 0) // page) for n in lengths]
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)) + 1
    table = torch.zeros(len(lengths), max(need) + 2, dtype=torch.int32)
    at = 0
    for n, c in enumerate(need):
        table[n, :c] = order[at:at + c]
        at += c
    cu = None
    if counts is not None:
        cu = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    return table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), cu, sum(need) + spare + 1


def _positions(lengths, counts):
    counts = [1] * len(lengths) if counts is None else counts
    return torch.tensor([n - c + i for n, c in zip(lengths, counts) for i in range(c)], device="cuda", dtype=torch.long)


CASES = [([1], None), ([16, 17, 0, 33, 1], None), ([5], [5]), ([40, 3, 100, 7, 0], [13, 3, 0, 1, 0]), ([130, 300], [129, 77]), ([3, 8], [5, 2])]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lengths,counts", CASES)
def test_append_and_read(lengths, counts, dim, dtype):
    """Every byte: the new tokens' by the definition, all others as they were."""
    from stepquant_b200.kernels.kv_cache import kv_append, kv_read
    from stepquant_b200.kernels.rotary import rotary_frequencies
    heads, page, interleaved = (3, 16, True) if dim == 64 else (2, 48, False) if dim == 128 else (1, 32, True)
    table, device_lengths, cu, pages = _sequences(lengths, page, counts)
    positions = _positions(lengths, counts)
    tokens = len(positions)
    k, v = (_rand(tokens, heads, dim, seed=s) * torch.where(_rand(dim) > 1.5, 20.0, 1.0) for s in (1, 2))
    k, v = k.to(dtype), v.to(dtype)
    data = torch.randint(0, 256, (pages, heads, page // 16, 18 * dim), device="cuda").to(torch.uint8)
    want = data.clone()
    f = None if dtype == torch.float16 else rotary_frequencies(dim if dim == 64 else dim // 2, 1e4)
    turned = k.double() if f is None else turn(k, positions, f, interleaved, 1.5)
    shown = []
    for at, x in enumerate((turned, v.double())):
        c, s, m = quantize(x)
        shown.append((m + s * c).flatten(-2))
        byte, shift, pair = (p.cuda() for p in tile_places(dim)[at])
        c = c.flatten(-2).to(torch.uint8)
        seq = torch.tensor([n for n, count in enumerate(counts or [1] * len(lengths)) for _ in range(count)], device="cuda")
        for i in range(tokens):
            p = int(positions[i])
            if p < 0:
                continue
            tile = want[int(table[seq[i], p // page]), :, p % page // 16]
            u = p % 16
            for half in (0, 4):
                put = shift[u] == half
                old = tile[:, byte[u][put]]
                tile[:, byte[u][put]] = (old & (0xF0 if half == 0 else 0x0F)) | (c[i][:, put] << half)
            both = torch.stack([s[i, :, :, 0], m[i, :, :, 0]], -1).bfloat16().view(torch.uint8).flatten(1)  # [H, 4 G]
            first = int(pair[u, 0])
            tile[:, first:first + both.shape[1]] = both
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv_append(data, k, v, table, device_lengths, cu_seqlens=cu, frequencies=f, interleaved=interleaved,
              magnitude=1.0 if f is None else 1.5, status=status)
    assert torch.equal(data, want)
    got = kv_read(data, table, device_lengths, cu_seqlens=cu, tokens=tokens, dtype=torch.float32, status=status)
    for x, y in zip(got, shown):
        assert torch.equal(x, torch.where((positions >= 0)[:, None, None], y, 0.0).float())
    low = kv_read(data, table, device_lengths, cu_seqlens=cu, tokens=tokens, dtype=torch.float16)
    assert all(torch.equal(a, b.half()) for a, b in zip(low, got))
    assert int(status) == 0


def test_layout_is_the_headers():
    from stepquant_b200.kernels.kv_cache import QuantizedKVPool
    pool = QuantizedKVPool(3, 2, 128, page_size=32)
    k, v = _rand(29, 2, 128, seed=3).bfloat16(), _rand(29, 2, 128, seed=4).bfloat16()
    table, lengths = torch.tensor([[2]], device="cuda"), torch.tensor([29], device="cuda")
    pool.append(k, v, table, lengths, cu_seqlens=torch.tensor([0, 29], device="cuda"))
    got = unpack(pool.data[2], 128)
    for x, y in zip(got, (k, v)):
        assert torch.equal(x.flatten(1, 2)[:, :29].transpose(0, 1), value(y))
    pool.check_status()


def test_within_half_a_step():
    """The bound that the form promises, and groups of one value or of tiny ones."""
    from stepquant_b200.kernels.kv_cache import kv_append, kv_read
    tokens, dim = 400, 128
    data = torch.zeros(30, 1, 1, 18 * dim, dtype=torch.uint8, device="cuda")
    k = _rand(tokens, 1, dim) * 10.0 ** torch.randint(-6, 6, (tokens, 1, 1), device="cuda") + 100 * _rand(tokens, 1, 1, seed=5)
    v = torch.cat([torch.full((50, 1, dim), x, device="cuda") for x in (0.0, 1.0, -3.0, 1e-40, -1e-40, 65504.0, 1e-30, 0.1)])
    table = torch.arange(1, 26, device="cuda", dtype=torch.int32)[None]
    lengths, cu = torch.tensor([tokens], device="cuda", dtype=torch.int32), torch.tensor([0, tokens], device="cuda", dtype=torch.int32)
    kv_append(data, k, v, table, lengths, cu_seqlens=cu)
    got = kv_read(data, table, lengths, cu_seqlens=cu, tokens=tokens, dtype=torch.float32)
    for x, y in zip(got, (k, v)):
        assert torch.equal(x, value(y).float())
        _, s, _ = quantize(y)
        assert bool(((x - y).double().unflatten(-1, (-1, 64)).abs() <= s / 2 + 2.0 ** -24 * y.double().abs().unflatten(-1, (-1, 64))).all())


def test_what_is_not_finite():
    from stepquant_b200.kernels.kv_cache import kv_append, kv_read
    data = torch.zeros(3, 1, 1, 18 * 128, dtype=torch.uint8, device="cuda")
    k, v = _rand(16, 1, 128, seed=6), _rand(16, 1, 128, seed=7)
    k[3, 0, 5], k[4, 0, 70], v[5, 0, 127], v[6, 0, 0], v[7, 0, 64] = math.nan, math.inf, -math.inf, 3.4e38, -3.38e38
    table, lengths, cu = (torch.tensor(x, device="cuda", dtype=torch.int32) for x in ([[2]], [16], [0, 16]))
    kv_append(data, k, v, table, lengths, cu_seqlens=cu)
    for x, y in zip(kv_read(data, table, lengths, cu_seqlens=cu, tokens=16, dtype=torch.float32), (k, v)):
        want = value(y).float()
        assert torch.equal(x.isnan(), want.isnan()) and torch.equal(x.nan_to_num(), want.nan_to_num())
    assert int(want.isnan().sum()) == 64 * 2


def test_pages_that_hold_nothing():
    """Pages <= 0 are skipped; pages past the pool and positions past the table are, and are flagged; so is nothing else."""
    from stepquant_b200.kernels.kv_cache import QuantizedKVPool
    k, v = _rand(40, 1, 64, seed=8).half(), _rand(40, 1, 64, seed=9).half()
    cu = torch.tensor([0, 40], device="cuda", dtype=torch.int32)
    lengths = torch.tensor([40], device="cuda", dtype=torch.int32)
    for table, held, bad in (([1, 0, 2], [0, 2], False), ([1, -7, 2], [0, 2], False), ([4, 2, 3], [1, 2], True), ([3, 1], [0, 1], True),
                             ([3, 1, 2], [0, 1, 2], False), ([2 ** 31 - 1, 1, 3], [1, 2], True)):
        pool = QuantizedKVPool(4, 1, 64, page_size=16)
        rows = torch.tensor([table], device="cuda", dtype=torch.int32)
        pool.append(k, v, rows, lengths, cu_seqlens=cu)
        got = pool.read(rows, lengths, cu_seqlens=cu, tokens=40, dtype=torch.float16)
        kept = torch.tensor([p // 16 in held for p in range(40)], device="cuda")[:, None, None]
        for x, y in zip(got, (k, v)):
            assert torch.equal(x, torch.where(kept, value(y), 0.0).half())
        assert not bool(pool.data[0].any())
        if bad:
            with pytest.raises(IndexError):
                pool.check_status()
        pool.check_status()


def test_tokens_of_no_sequence_and_given_positions():
    """Tokens before the first boundary and past the last are not written and read as zeros; rotation by other positions."""
    from stepquant_b200.kernels.kv_cache import kv_append, kv_read
    from stepquant_b200.kernels.rotary import rotary_frequencies
    wide = _rand(12, 2, 2, 128, seed=10).bfloat16()
    k, v = wide[:, 0], wide[:, 1]  # strided, as slices of a projection
    data = torch.zeros(4, 2, 1, 18 * 128, dtype=torch.uint8, device="cuda")
    table, lengths, cu = (torch.tensor(x, device="cuda", dtype=torch.int32) for x in ([[1], [3]], [4, 9], [2, 5, 10]))
    at = torch.arange(100, 112, device="cuda", dtype=torch.int32)
    f = rotary_frequencies(128)
    kv_append(data, k, v, table, lengths, cu_seqlens=cu, frequencies=f, positions=at)
    got = kv_read(data, table, lengths, cu_seqlens=cu, tokens=12, dtype=torch.float32)
    inside = torch.tensor([2 <= i < 10 for i in range(12)], device="cuda")[:, None, None]
    assert torch.equal(got[0], torch.where(inside, value(turn(k, at, f)), 0.0).float())
    assert torch.equal(got[1], torch.where(inside, value(v), 0.0).float())
    assert not bool(data[2].any())
    odd = torch.zeros(12, 2, 2, 129, device="cuda", dtype=torch.bfloat16)
    odd[..., 1:] = wide
    again = torch.zeros_like(data)
    kv_append(again, odd[:, 0, :, 1:], odd[:, 1, :, 1:], table.long(), lengths.long(), cu_seqlens=cu.long(), frequencies=f, positions=at)
    assert torch.equal(again, data)


def test_pool_methods():
    from stepquant_b200.kernels.kv_cache import QuantizedKVPool
    pool = QuantizedKVPool(6, 2, 64, page_size=16)
    k, v = _rand(3, 2, 64).bfloat16(), _rand(3, 2, 64, seed=1).bfloat16()
    table = torch.tensor([[1], [2], [3]], device="cuda", dtype=torch.int32)
    lengths = torch.tensor([1, 5, 16], device="cuda", dtype=torch.int32)
    pool.append(k, v, table, lengths)
    pool.copy(torch.tensor([2], device="cuda"), torch.tensor([5], device="cuda"))
    moved = table.clone()
    moved[1] = 5
    for a, b in zip(pool.read(table, lengths), pool.read(moved, lengths)):
        assert torch.equal(a, b)
    pool.clear(torch.tensor([2], device="cuda"))
    assert not bool(pool.data[2].any()) and not bool(pool.read(table, lengths)[0][1].any())
