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


class _Log(list):
    """Results of the example's calls, in their order, on the CPU in 64 bits."""

    def tap(self, function):
        def tapped(*args, **kwargs):
            result = function(*args, **kwargs)
            self.append(result.detach().cpu().double())
            return result
        return tapped

    def take(self):
        taken = list(self)
        self.clear()
        return taken


def _convolved(x, lead, weight, bias):
    """SiLU of the convolution of x [T, D] after the inputs `lead` [W - 1, D]."""
    window = torch.cat([lead, x])
    y = sum(weight[:, j] * window[j:j + len(x)] for j in range(weight.shape[1])) + bias
    return y * torch.sigmoid(y)


def _selective(u, dt, z, b, c, h, a, d, dt_bias):
    """(y, state) of the selective scan of one request's tokens from state h [D, N]."""
    dt = torch.nn.functional.softplus(dt + dt_bias, threshold=50.0)
    ys = []
    for t in range(len(u)):
        h = torch.exp(dt[t][:, None] * a) * h + (dt[t] * u[t])[:, None] * b[t]
        ys.append((h @ c[t] + d * u[t]) * z[t] * torch.sigmoid(z[t]))
    return torch.stack(ys), h


def _delta(qkv, gates, s, a_log, dt_bias):
    """(out, state) of the gated delta rule of one request's tokens from state s [H, K, V]."""
    heads = len(a_log)
    outs = []
    for t in range(len(qkv)):
        q, k, v = qkv[t].view(3, heads, 128)
        q, k = (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt() for x in (q, k))
        a, beta = gates[t].view(2, heads)
        s = s * torch.exp(-a_log.exp() * torch.nn.functional.softplus(a + dt_bias, threshold=50.0))[:, None, None]
        s = s + k[:, :, None] * (beta.sigmoid()[:, None] * (v - torch.einsum("hk,hkv->hv", k, s)))[:, None]
        outs.append(torch.einsum("hk,hkv->hv", q, s).flatten() * 128 ** -0.5)
    return torch.stack(outs), s


def test_every_kept_state_of_the_layers(monkeypatch):
    """What each state of the example's two layers gives the decoded tokens, against the
    recurrences in 64 bits on the CPU, from the same projections.

    Bounds on the norm of the difference over the norm: bf16 outputs of fp32 sums 2^-8; the
    delta rule's states have steps of 1 / 127 of a row's largest value, 0.6 % of its root mean
    square, taken up to seven times (1.6 %), its prompt pass bf16 operands (0.4 %): 5 %.  With a
    state dropped, or taken from another request, in the oracle, the difference has to be three
    times that at least: the bounds tell a wrong state from a right one.
    """
    example, log = _example(), _Log()
    monkeypatch.setattr(example, "causal_conv1d_step", log.tap(example.causal_conv1d_step))
    monkeypatch.setattr(example, "causal_conv1d_extend", log.tap(example.causal_conv1d_extend))
    monkeypatch.setattr(example.Projection, "__call__", log.tap(example.Projection.__call__))

    def quantize(x, wrapped=example.quantize_fp8):
        log.append(x.detach().cpu().double())
        return wrapped(x)

    monkeypatch.setattr(example, "quantize_fp8", quantize)
    lengths, decode, hidden, heads, channels = (37, 5, 64, 18), 6, 512, 4, 768
    batch, total = len(lengths), sum(lengths)
    gen = torch.Generator("cuda").manual_seed(5)
    delta = example.DeltaLayer(gen, batch + 1, hidden, heads)
    selective = example.SelectiveLayer(gen, batch + 1, hidden, channels)
    slots = torch.tensor([3, 1, 4, 2], device="cuda")
    ends = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], device="cuda", dtype=torch.int32)
    x = torch.randn(total + decode * batch, hidden, generator=gen, device="cuda").bfloat16()
    prompt, tokens = {}, {}
    for name, layer in (("delta", delta), ("selective", selective)):
        log.clear()
        layer(x[:total], slots, ends)
        prompt[name] = [list(part.split(list(lengths))) for part in log.take()]
        steps = []
        for i in range(decode):
            layer(x[total + i * batch:total + (i + 1) * batch], slots)
            steps.append(log.take())
        tokens[name] = [list(torch.stack(parts, 1)) for parts in zip(*steps)]  # each [request][token]

    def off(got, want):
        got, want = torch.stack(got), torch.stack(want)
        return float((got - want).norm() / want.norm())

    def tell(got, want, states, bound):
        """want(state of each request): near got with the right states, and with no wrong ones."""
        assert off(got, [want(n, s) for n, s in enumerate(states)]) < bound
        assert off(got, [want(n, torch.zeros_like(s)) for n, s in enumerate(states)]) > 3 * bound
        assert off(got, [want(n, states[n - 1]) for n in range(batch)]) > 3 * bound

    cpu = lambda t: t.detach().cpu().double()  # noqa: E731
    wide = 3 * heads * 128
    projected, qkv, _, _ = prompt["delta"]
    step_projected, step_qkv, step_out, _ = tokens["delta"]
    filters, none = cpu(delta.filter), torch.zeros(wide, dtype=torch.float64)
    leads = [torch.cat([torch.zeros(3, wide, dtype=torch.float64), p[:, :wide]])[-3:] for p in projected]
    tell(step_qkv, lambda n, lead: _convolved(step_projected[n][:, :wide], lead, filters, none), leads, 2.0 ** -8)
    gates = (cpu(delta.a_log), cpu(delta.dt_bias))
    empty = torch.zeros(heads, 128, 128, dtype=torch.float64)
    states = [_delta(q, p[:, wide:], empty, *gates)[1] for q, p in zip(qkv, projected)]
    tell(step_out, lambda n, s: _delta(step_qkv[n], step_projected[n][:, wide:], s, *gates)[0], states, 0.05)

    def scanned(parts, n, h):
        projected, u, low, _, dt, _, _ = (p[n] for p in parts)
        b, c = low[:, selective.rank:].split(selective.states, 1)
        return _selective(u, dt, projected[:, channels:], b, c, h, *(cpu(t) for t in (selective.a, selective.d, selective.dt_bias)))

    projected, step_projected = prompt["selective"][0], tokens["selective"][0]
    leads = [torch.cat([torch.zeros(3, channels, dtype=torch.float64), p[:, :channels]])[-3:] for p in projected]
    tell(tokens["selective"][1], lambda n, lead: _convolved(step_projected[n][:, :channels], lead, cpu(selective.filter),
                                                            cpu(selective.bias)), leads, 2.0 ** -8)
    states = [scanned(prompt["selective"], n, torch.zeros(channels, selective.states, dtype=torch.float64))[1] for n in range(batch)]
    tell(tokens["selective"][5], lambda n, h: scanned(tokens["selective"], n, h)[0], states, 2.0 ** -8)
