"""Further refusals of the rotary and cache operators that need no GPU."""
import ctypes
import math

import pytest
import torch

from stepquant_b200 import _native as N
from stepquant_b200.kernels.kv_cache import kv_append
from stepquant_b200.kernels.rotary import rotary, rotary_frequencies


def test_outputs_in_another_order():
    """Heads and tokens of x's own memory exchanged: what one pair writes another has yet to read."""
    x = torch.randn(4, 4, 8)
    f, positions = rotary_frequencies(8, device="cpu"), torch.arange(4)
    with pytest.raises(ValueError, match="another order"):
        rotary(x, positions, f, out=x.transpose(0, 1))
    with pytest.raises(ValueError, match="CUDA"):  # in place is no such case, nor is the stride of an axis of one
        rotary(x, positions, f, out=x)
    one = x[:1]
    with pytest.raises(ValueError, match="CUDA"):
        rotary(one, positions[:1], f, out=one.as_strided((1, 4, 8), (7, 8, 1)))


@pytest.mark.parametrize("magnitude", [1e39, -1e39, math.inf, math.nan])
def test_magnitudes_beyond_fp32(magnitude):
    """A number that the C structure would hold as infinity."""
    x, data, table = torch.randn(1, 1, 64), torch.zeros(2, 1, 1, 18 * 64, dtype=torch.uint8), torch.ones(1, 1, dtype=torch.int32)
    f, positions = rotary_frequencies(64, device="cpu"), torch.zeros(1, dtype=torch.long)
    with pytest.raises(ValueError, match="magnitude"):
        rotary(x, positions, f, magnitude=magnitude)
    with pytest.raises(ValueError, match="magnitude"):
        kv_append(data, x, x, table, table[0], frequencies=f, magnitude=magnitude)
    for entry, kind in ((N.lib().sq_rotary, N.SqRotaryArgs), (N.lib().sq_kv_append, N.SqKvArgs), (N.lib().sq_kv_read, N.SqKvArgs)):
        args = kind(dim=64, heads=1, page_size=16, magnitude=magnitude) if kind is N.SqKvArgs else kind(dim=64, heads=1, magnitude=magnitude)
        assert entry(ctypes.byref(args), None) == N.SQ_ERR_ARGUMENT
