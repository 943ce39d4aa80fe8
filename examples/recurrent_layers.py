"""A stack of recurrent layers on the package's operators: prompts, then tokens.

    residual norm -> e4m3 activations -> e4m3 projection -> short convolution
                  -> state pass -> e4m3 projection added to the residual

once with a gated delta rule layer, whose states live packed in a
``PackedStatePool``, and once with a selective layer (``SelectiveStatePool``);
with ``attention`` a softmax attention layer stands between them, its keys and
values in 4 bits (``QuantizedKVPool``), queries and keys rotated.
Random weights; ``python examples/recurrent_layers.py`` runs a batch of ragged
prompts, decodes from the kept states and compares the decoded tokens' outputs
with one pass over the whole sequences.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from stepquant_b200 import QuantizationPlan  # noqa: E402
from stepquant_b200.kernels.conv import causal_conv1d_extend, causal_conv1d_step  # noqa: E402
from stepquant_b200.kernels.kv_cache import QuantizedKVPool  # noqa: E402
from stepquant_b200.kernels.matmul import matmul_fp8, quantize_weight_fp8  # noqa: E402
from stepquant_b200.kernels.norm import quantize_fp8, rms_norm_fp8  # noqa: E402
from stepquant_b200.kernels.pool import PackedStatePool  # noqa: E402
from stepquant_b200.kernels.rotary import rotary, rotary_frequencies  # noqa: E402
from stepquant_b200.kernels.scan import SelectiveStatePool  # noqa: E402


class Projection:
    """y = x w^T (+ residual) with e4m3 weights, from the (values, scales) of e4m3 activations."""

    def __init__(self, gen, width, hidden):
        w = torch.randn(width, hidden, generator=gen, device="cuda") * hidden ** -0.5
        self.weight, self.scale = quantize_weight_fp8(w)
        self.status = torch.zeros(1, device="cuda", dtype=torch.int32)

    def __call__(self, activations, residual=None):
        return matmul_fp8(*activations, self.weight, self.scale, residual=residual, status=self.status)


class SelectiveLayer:
    def __init__(self, gen, slots, hidden, channels, states=16, rank=32, taps=4):
        self.channels, self.states, self.rank = channels, states, rank
        self.norm = torch.ones(hidden, device="cuda", dtype=torch.bfloat16)
        self.w_in = Projection(gen, 2 * channels, hidden)
        self.w_x = Projection(gen, rank + 2 * states, channels)
        self.w_dt = Projection(gen, channels, rank)
        self.w_out = Projection(gen, hidden, channels)
        self.filter = torch.randn(channels, taps, generator=gen, device="cuda") * taps ** -0.5
        self.bias = torch.zeros(channels, device="cuda")
        self.a = -torch.arange(1, states + 1, device="cuda", dtype=torch.float32).repeat(channels, 1)
        self.d = torch.ones(channels, device="cuda")
        self.dt_bias = torch.full((channels,), -4.0, device="cuda")  # steps around softplus(-4)
        self.pool = SelectiveStatePool(slots, channels, states, taps)

    def __call__(self, x, slots, cu_seqlens=None):
        """x: [tokens, hidden], prompts with cu_seqlens, else one token of each slot."""
        xz = self.w_in(rms_norm_fp8(x, self.norm))
        u = self.pool.convolve(xz[:, :self.channels], self.filter, self.bias, slots=slots, cu_seqlens=cu_seqlens)
        low = self.w_x(quantize_fp8(u))
        dt = self.w_dt(quantize_fp8(low[:, :self.rank]))
        b, c = low[:, self.rank:].unflatten(1, (2, 1, self.states)).unbind(1)
        args = (u, dt, self.a, b, c, slots)
        options = dict(d=self.d, z=xz[:, self.channels:], dt_bias=self.dt_bias)
        y = self.pool.step(*args, **options) if cu_seqlens is None else self.pool.extend(*args, cu_seqlens, **options)
        return self.w_out(quantize_fp8(y), residual=x)


class DeltaLayer:
    """Gated delta rule with 8-bit packed states; q, k, v pass through the short convolution."""

    def __init__(self, gen, slots, hidden, heads, taps=4):
        self.heads = heads
        self.norm = torch.ones(hidden, device="cuda", dtype=torch.bfloat16)
        self.w_in = Projection(gen, 3 * heads * 128 + 2 * heads, hidden)
        self.w_out = Projection(gen, hidden, heads * 128)
        self.filter = torch.randn(3 * heads * 128, taps, generator=gen, device="cuda") * taps ** -0.5
        self.conv = torch.zeros(slots, 3 * heads * 128, taps - 1, device="cuda", dtype=torch.bfloat16)
        self.a_log = torch.zeros(heads, device="cuda")
        self.dt_bias = torch.full((heads,), -4.0, device="cuda")
        plan = QuantizationPlan("gdn", torch.full((heads, 128), 8, device="cuda"), torch.ones(heads, 128, device="cuda"))
        self.pool = PackedStatePool(plan, slots, 128)
        self.pool.clear(slice(None))

    def __call__(self, x, slots, cu_seqlens=None):
        proj = self.w_in(rms_norm_fp8(x, self.norm))
        wide = 3 * self.heads * 128
        if cu_seqlens is None:
            qkv = causal_conv1d_step(proj[:, :wide], self.conv, self.filter, slots=slots)
        else:
            qkv = causal_conv1d_extend(proj[:, :wide], self.conv, self.filter, slots=slots, cu_seqlens=cu_seqlens)
        q, k, v = qkv.unflatten(1, (3, self.heads, 128)).unbind(1)
        a, beta = proj[:, wide:].float().unflatten(1, (2, self.heads)).unbind(1)
        if cu_seqlens is None:
            out = self.pool.step(q, k, v.flatten(1), a.contiguous(), beta.contiguous(), slots, normalize=True,
                                 scale=128 ** -0.5, a_log=self.a_log, dt_bias=self.dt_bias)
        else:
            g = -self.a_log.exp() * torch.nn.functional.softplus(a + self.dt_bias)
            out = self.pool.extend(q, k, v, g, beta.sigmoid(), slots, cu_seqlens, scale=128 ** -0.5)
        return self.w_out(quantize_fp8(out.reshape(x.shape[0], -1)), residual=x)


class AttentionLayer:
    """Softmax attention over a 4-bit cache; slot n owns `pages` pages of it."""

    def __init__(self, gen, slots, hidden, heads, kv_heads, dim=128, pages=2, page_size=64):
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.norm = torch.ones(hidden, device="cuda", dtype=torch.bfloat16)
        self.w_in = Projection(gen, (heads + 2 * kv_heads) * dim, hidden)
        self.w_out = Projection(gen, hidden, heads * dim)
        self.frequencies = rotary_frequencies(dim)
        self.pool = QuantizedKVPool(1 + (slots - 1) * pages, kv_heads, dim, page_size)
        self.table = torch.arange(1 - pages, 1 + (slots - 1) * pages, device="cuda", dtype=torch.int32).view(slots, pages)
        self.lengths = torch.zeros(slots, device="cuda", dtype=torch.int32)

    def __call__(self, x, slots, cu_seqlens=None):
        heads = self.w_in(rms_norm_fp8(x, self.norm)).unflatten(1, (-1, self.dim))
        q, k, v = heads.split([self.heads, self.kv_heads, self.kv_heads], 1)
        if cu_seqlens is None:
            self.lengths[slots] += 1
            positions = self.lengths[slots] - 1
        else:
            self.lengths[slots] += cu_seqlens.diff()
            token = torch.arange(x.shape[0], device="cuda")
            seq = torch.searchsorted(cu_seqlens[1:].contiguous(), token, right=True)
            positions = (self.lengths[slots] - cu_seqlens[1:])[seq] + token
        table, lengths = self.table[slots], self.lengths[slots]
        q = rotary(q, positions, self.frequencies)
        self.pool.append(k, v, table, lengths, cu_seqlens=cu_seqlens, frequencies=self.frequencies)
        out = self.pool.attend(q, table, lengths, cu_seqlens=cu_seqlens)
        return self.w_out(quantize_fp8(out.flatten(1)), residual=x)


def run(lengths=(37, 5, 64, 18), decode=6, hidden=512, seed=0, attention=False):
    """Largest relative difference, per layer stack output, between tokens decoded
    from the prompts' states and the same tokens inside whole-sequence passes."""
    batch = len(lengths)
    slots = torch.arange(1, batch + 1, device="cuda")

    def stack():
        gen = torch.Generator("cuda").manual_seed(seed)
        middle = [AttentionLayer(gen, batch + 1, hidden, heads=4, kv_heads=2)] if attention else []
        return [DeltaLayer(gen, batch + 1, hidden, heads=4), *middle, SelectiveLayer(gen, batch + 1, hidden, channels=768)]

    gen = torch.Generator("cuda").manual_seed(seed + 1)
    rows = [torch.randn(n + decode, hidden, generator=gen, device="cuda").bfloat16() for n in lengths]
    ends = lambda sizes: torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], device="cuda", dtype=torch.int32)  # noqa: E731

    def forward(layers, x, cu=None):
        for layer in layers:
            x = layer(x, slots, cu)
        return x

    whole = forward(stack(), torch.cat(rows), ends([len(r) for r in rows])).split([len(r) for r in rows])
    layers = stack()
    prompt = forward(layers, torch.cat([r[:n] for r, n in zip(rows, lengths)]), ends(lengths)).split(list(lengths))
    same = max(float((p - w[:len(p)]).abs().max()) for p, w in zip(prompt, whole))
    steps = [forward(layers, torch.stack([r[n + i] for r, n in zip(rows, lengths)])) for i in range(decode)]
    for layer in layers:
        layer.pool.check_status()
        for part in vars(layer).values():
            if isinstance(part, Projection) and int(part.status):
                raise RuntimeError("a bounded device wait of a projection gave up; its outputs are NaN")
    got = torch.stack(steps, 1).float()
    want = torch.stack([w[n:] for w, n in zip(whole, lengths)]).float()
    return same, float((got - want).norm() / want.norm())


if __name__ == "__main__":
    for attention in (False, True):
        same, off = run(attention=attention)
        print(f"{'with' if attention else 'without'} attention: prompt outputs in two batchings differ by at most {same:.3g}; "
              f"decoded tokens by {off:.3g} of their norm")
