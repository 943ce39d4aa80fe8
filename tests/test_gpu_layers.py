"""The layer operators together (examples/recurrent_layers.py), and offsets past 32 bits."""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("recurrent_layers", os.path.join(ROOT, "examples", "recurrent_layers.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_example_decodes_what_whole_passes_give():
    """Decoded tokens against whole-sequence passes.  The two differ by the 8-bit
    states (a step of 1 / 127 of a row's range), bf16 activations (2^-8) and e4m3
    ones (2^-4 of single values, averaged over 512 to 1536 terms of a product), on
    top of a residual stream that is equal: 5 % of the norm bounds them, and a
    wrong state, slot or shift is of the size of the stream's change itself."""
    same, off = _example().run()
    assert same < 0.25 and off < 0.05


def test_places_past_32_bits():
    """Pool rows, rows of x and outputs that lie more than 2^32 bytes and 2^31 values in."""
    from stepquant_b200.kernels.conv import causal_conv1d_step
    from stepquant_b200.kernels.norm import rms_norm
    from stepquant_b200.kernels.scan import selective_scan_step
    slots, channels = 34000, 4096
    pool = torch.empty(slots, channels, 16, device="cuda")  # 2.2e9 values
    at = torch.tensor([1, slots - 1], device="cuda")
    pool[at] = 1.0
    u = torch.randn(2, channels, device="cuda")
    dt, a = torch.full_like(u, 0.5), -torch.rand(channels, 16, device="cuda")
    b = torch.randn(2, 1, 16, device="cuda")
    y = selective_scan_step(pool, u, dt, a, b, b, dt_softplus=False, slots=at)
    want = torch.exp(0.5 * a) + 0.5 * u[:, :, None] * b
    torch.testing.assert_close(pool[at], want, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(y, (want * b).sum(2), rtol=1e-4, atol=1e-4)
    del pool
    conv = torch.empty(180000, channels, 3, device="cuda", dtype=torch.bfloat16)  # 2.2e9 values
    conv[179999] = 2.0
    x = u[:1].bfloat16()
    y = causal_conv1d_step(x, conv, torch.ones(channels, 4, device="cuda"), slots=torch.tensor([179999], device="cuda"),
                           activation=None)
    torch.testing.assert_close(y, (x.float() + 6).bfloat16())
    assert torch.equal(conv[179999, :, 2], x[0]) and bool((conv[179999, :, :2] == 2).all())
    del conv
    rows = 530000
    x = torch.empty(rows, channels, device="cuda", dtype=torch.bfloat16)  # 2.2e9 values
    x[-3:] = u[:1].bfloat16()
    y = rms_norm(x, torch.ones(channels, device="cuda"))
    last = x[-1].double()
    torch.testing.assert_close(y[-1].double(), last / (last.square().mean() + 1e-6).sqrt(), rtol=2 ** -7, atol=1e-6)
    assert torch.equal(y[-1], y[-2])


def test_product_with_rows_past_32_bits():
    from stepquant_b200.kernels.matmul import matmul_fp8, quantize_weight_fp8
    from stepquant_b200.kernels.norm import quantize_fp8
    rows, width = 280000, 8192  # 2.3e9 outputs
    x = torch.zeros(rows, 128, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    scale = torch.ones(rows, 1, device="cuda")
    x[-2:], scale[-2:] = quantize_fp8(torch.randn(2, 128, device="cuda"))
    w, sw = quantize_weight_fp8(torch.randn(width, 128, device="cuda"))
    got = matmul_fp8(x, scale, w, sw)
    want = matmul_fp8(x[-2:], scale[-2:], w, sw)
    torch.testing.assert_close(got[-2:], want, rtol=2 ** -7, atol=1e-3)
    assert not bool(got[-300:-2].any())


def test_status_is_an_int32_word():
    """A word of another size would be written past its end."""
    from stepquant_b200.kernels.conv import causal_conv1d_extend, causal_conv1d_step
    from stepquant_b200.kernels.matmul import matmul_fp8, quantize_weight_fp8
    from stepquant_b200.kernels.norm import quantize_fp8
    from stepquant_b200.kernels.scan import selective_scan_extend, selective_scan_step
    x, slots = torch.randn(2, 32, device="cuda"), torch.tensor([1, 2], device="cuda")
    ends, filters = torch.tensor([0, 1, 2], device="cuda"), torch.ones(32, 4, device="cuda")
    conv, state = torch.zeros(3, 32, 3, device="cuda"), torch.zeros(3, 32, 16, device="cuda")
    a, b = -torch.ones(32, 16, device="cuda"), torch.ones(2, 1, 16, device="cuda")
    operands = (*quantize_fp8(x), *quantize_weight_fp8(torch.ones(8, 32, device="cuda")))
    for status in (torch.zeros(1, device="cuda", dtype=torch.int8), torch.zeros(0, device="cuda", dtype=torch.int32),
                   torch.zeros(1, device="cuda", dtype=torch.int64)):
        for call in (lambda: causal_conv1d_step(x, conv, filters, slots=slots, status=status),
                     lambda: causal_conv1d_extend(x, conv, filters, slots=slots, cu_seqlens=ends, status=status),
                     lambda: selective_scan_step(state, x, x, a, b, b, slots=slots, status=status),
                     lambda: selective_scan_extend(state, x, x, a, b, b, slots=slots, cu_seqlens=ends, status=status),
                     lambda: matmul_fp8(*operands, status=status)):
            with pytest.raises(ValueError, match="status"):
                call()
