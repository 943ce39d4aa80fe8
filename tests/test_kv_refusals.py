"""Further refusals of the rotary and cache operators that need no GPU."""
import pytest
import torch

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
