"""Pages, lengths and boundaries of 64 bits that 32 do not hold stay outside the pool, the table and the tokens."""
import pytest
import torch

from stepquant_b200.kernels.kv_cache import QuantizedKVPool, _int32


def test_conversion():
    x = torch.tensor([0, 5, -1, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, -2 ** 32 + 1, 2 ** 62])
    want = [0, 5, -1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1]
    got = _int32(x, -1, x.device)
    assert got.dtype == torch.int32 and got.tolist() == want
    assert _int32(x[:3].int(), -1, x.device).tolist() == want[:3] and _int32(x[:3].to(torch.int16), -1, x.device).tolist() == want[:3]
    assert _int32(torch.stack([x, x], 1)[:, :1], -1, x.device).flatten().tolist() == want


@pytest.mark.gpu
def test_wide_pages_and_lengths():
    pool = QuantizedKVPool(4, 1, 64, page_size=16)
    k = torch.randn(16, 1, 64, device="cuda").bfloat16()
    cu = torch.tensor([0, 16], device="cuda")
    for table, length in (([[2 ** 32 + 1]], 16), ([[1]], 2 ** 32 + 16), ([[2 ** 33]], 16)):
        table, lengths = torch.tensor(table, device="cuda"), torch.tensor([length], device="cuda")
        pool.append(k, k, table, lengths, cu_seqlens=cu)
        with pytest.raises(IndexError):
            pool.check_status()
        assert not bool(pool.data.any())
        got, _ = pool.read(table, lengths, cu_seqlens=cu, tokens=16)
        assert not bool(got.any())
        pool.attend(k, table, lengths, cu_seqlens=cu)
        with pytest.raises(IndexError):
            pool.check_status()
    pool.append(k, k, torch.tensor([[-2 ** 32 + 1]], device="cuda"), torch.tensor([16], device="cuda"), cu_seqlens=cu)
    pool.check_status()
    assert not bool(pool.data.any())
