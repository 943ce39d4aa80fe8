"""The attention layer's operators as they are used together: queries rotated, keys
and values appended, attention over the cache; prompts in pieces, then single
tokens, on other streams, in captured graphs, two calls at once, and with places
past 32 bits.

What the cache holds is exact (kv_reference.value of the rotated keys), so outputs
are compared with 64-bit attention over those values by the tolerances of
test_gpu_kv_attention.py, the queries' own rounding after their rotation being part
of the computation on both sides.
"""
import pytest
import torch

from kv_reference import attend, cached, turn, value
from test_gpu_kv_attention import _check
from test_gpu_kv_cache import _rand, _sequences

pytestmark = pytest.mark.gpu


def _ends(counts):
    return torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], device="cuda", dtype=torch.int32)


class _Layer:
    """A pool with its frequencies; tokens of all sequences are drawn ahead, by position."""

    def __init__(self, longest, seqs, q_heads=8, heads=2, dim=128, page=32, dtype=torch.bfloat16, window=None):
        from stepquant_b200.kernels.kv_cache import QuantizedKVPool
        from stepquant_b200.kernels.rotary import rotary_frequencies
        self.table, _, _, pages = _sequences([longest] * seqs, page)
        self.pool = QuantizedKVPool(pages, heads, dim, page_size=page)
        self.frequencies = rotary_frequencies(dim // 2, 1e4)
        self.page, self.window = page, window
        self.q, self.k, self.v = (_rand(seqs, longest, h, dim, seed=i).to(dtype) for i, h in enumerate((q_heads, heads, heads)))
        self.seen = [0] * seqs

    def tokens(self, counts):
        """(q, k, v, positions) of the next `counts` tokens of each sequence; the sequences go on."""
        spans = [(n, s, s + c) for n, (s, c) in enumerate(zip(self.seen, counts))]
        parts = [torch.cat([x[n, a:b] for n, a, b in spans]) for x in (self.q, self.k, self.v)]
        self.seen = [b for _, _, b in spans]
        return *parts, torch.cat([torch.arange(a, b, device="cuda") for _, a, b in spans])

    def step(self, q, k, v, positions, lengths, cu):
        from stepquant_b200.kernels.rotary import rotary
        q = rotary(q, positions, self.frequencies)
        self.pool.append(k, v, self.table, lengths, cu_seqlens=cu, frequencies=self.frequencies)
        return q, self.pool.attend(q, self.table, lengths, cu_seqlens=cu, window=self.window)

    def run(self, counts):
        lengths = torch.tensor([s + c for s, c in zip(self.seen, counts)], device="cuda", dtype=torch.int32)
        data = self.tokens(counts)
        q, out = self.step(*data, lengths, None if set(counts) == {1} else _ends(counts))
        _check(out, q, self.pool.data, self.table, self.seen, counts, self.page, window=self.window)
        return out


@pytest.mark.parametrize("dtype,dim,q_heads,heads,page,window", [
    (torch.bfloat16, 128, 8, 2, 32, None), (torch.float16, 64, 6, 3, 16, 20), (torch.bfloat16, 256, 16, 2, 64, 100),
    (torch.bfloat16, 64, 160, 1, 16, None)])
def test_prompts_in_pieces_then_tokens(dtype, dim, q_heads, heads, page, window):
    layer = _Layer(260, 3, q_heads, heads, dim, page, dtype, window)
    for counts in ([100, 1, 40], [3, 0, 129], [1, 70, 2], *[[1, 1, 1]] * 3, [2, 3, 4], [60, 1, 1]):
        layer.run(counts)
    layer.pool.check_status()
    for n, length in enumerate(layer.seen):
        k, v, _ = cached(layer.pool.data, layer.table[n].tolist(), page, length)
        at = torch.arange(length, device="cuda")
        assert torch.equal(k.transpose(0, 1), value(turn(layer.k[n, :length], at, layer.frequencies)))
        assert torch.equal(v.transpose(0, 1), value(layer.v[n, :length]))


def test_how_a_prompt_is_cut_does_not_matter_to_the_cache():
    """The same tokens in one piece, in several and one by one leave the same bytes."""
    data = []
    for cuts in ([[150, 90]], [[64, 1], [86, 89]], [[30, 80], *[[1, 1]] * 10, [110, 0]]):
        layer = _Layer(240, 2)
        for counts in cuts:
            layer.run(counts)
        assert layer.seen == [150, 90]
        data.append(layer.pool.data)
    assert torch.equal(data[0], data[1]) and torch.equal(data[0], data[2])


@pytest.mark.parametrize("how", ["side", "budget", "graph"])
@pytest.mark.parametrize("counts", [[1] * 5, [200, 1, 0, 37, 64], [4000, 900, 1, 1, 1]])
def test_other_streams(counts, how):
    """Bytes equal; outputs within rounding (a stream of fewer SMs cuts long sequences at other places)."""
    from stepquant_b200.kernels.resources import writeback_resources
    cu = None if set(counts) == {1} else _ends(counts)
    layer, other = (_Layer(4096, 5) for _ in range(2))
    lengths = torch.tensor([c + 50 for c in counts], device="cuda", dtype=torch.int32)
    before = [50] * 5
    for one in (layer, other):
        data = one.tokens(before)
        one.step(*data, torch.tensor(before, device="cuda", dtype=torch.int32), _ends(before))
    data = layer.tokens(counts)
    q, want = layer.step(*data, lengths, cu)
    torch.cuda.synchronize()
    if how == "graph":
        still = [torch.zeros_like(x) for x in data]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _, got = other.step(*still, lengths, cu)
        for x, y in zip(still, data):
            x.copy_(y)
        graph.replay()
        first = got.clone()
        graph.replay()
        assert torch.equal(got, first)
    else:
        stream = torch.cuda.Stream() if how == "side" else writeback_resources("cuda", 16).stream
        with torch.cuda.stream(stream):
            _, got = other.step(*data, lengths, cu)
        stream.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(other.pool.data, layer.pool.data)
    if how != "budget":
        assert torch.equal(got, want)
    _check(got, q, layer.pool.data, layer.table, lengths.tolist(), counts, layer.page)
    layer.pool.check_status()


def test_two_calls_and_two_graphs_at_once():
    """Calls on two streams, eager and as graphs captured one after the other, do not meet in a workspace."""
    layers = [_Layer(3000, 2), _Layer(3000, 2, q_heads=4)]
    want, inputs = [], []
    for layer in layers:
        layer.run([2500, 700])
        lengths = torch.tensor(layer.seen, device="cuda", dtype=torch.int32)
        q = layer.q[:, 5].contiguous()
        inputs.append((q, layer.table, lengths))
        want.append(layer.pool.attend(*inputs[-1]))
    streams = [torch.cuda.Stream() for _ in layers]
    graphs, outs = [], []
    for layer, args in zip(layers, inputs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(layer.pool.attend(*args))
        graphs.append(graph)
    torch.cuda.synchronize()
    eager = []
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                graphs[i].replay()
                eager.append((i, layers[i].pool.attend(*inputs[i])))
    torch.cuda.synchronize()
    assert all(torch.equal(out, w) for out, w in zip(outs, want)) and all(torch.equal(out, want[i]) for i, out in eager)


@pytest.mark.parametrize("counts", [[1], [300]])
def test_places_past_32_bits(counts):
    """Pages whose bytes begin past 2^32, with a table that has them first, last and between."""
    from stepquant_b200.kernels.kv_cache import QuantizedKVPool
    page, heads, dim = 256, 16, 256
    pages = 2 ** 32 // (heads * page // 16 * 18 * dim) + 40
    pool = QuantizedKVPool(pages, heads, dim, page_size=page)
    assert pool.data.numel() > 2 ** 32
    table = torch.tensor([[pages - 1, 3, pages - 2, 7]], device="cuda", dtype=torch.int32)
    k, v = _rand(900, heads, dim, seed=1).bfloat16(), _rand(900, heads, dim, seed=2).bfloat16()
    lengths, cu = torch.tensor([900], device="cuda", dtype=torch.int32), _ends([900])
    pool.append(k, v, table, lengths, cu_seqlens=cu)
    got = pool.read(table, lengths, cu_seqlens=cu, tokens=900, dtype=torch.float32)
    assert all(torch.equal(x, value(y).float()) for x, y in zip(got, (k, v)))
    q = _rand(counts[0], heads, dim, seed=3).bfloat16()
    out = pool.attend(q, table, lengths, cu_seqlens=None if counts == [1] else _ends(counts))
    pool.check_status()
    _check(out, q, pool.data, table, [900], counts, page)


def test_nothing_at_all():
    """No sequences: zeros, and nothing is written."""
    from stepquant_b200.kernels.kv_cache import QuantizedKVPool
    pool = QuantizedKVPool(2, 1, 64, page_size=16)
    table, lengths, cu = (torch.zeros(s, device="cuda", dtype=torch.int32) for s in ((0, 3), (0,), (1,)))
    x = _rand(5, 1, 64).bfloat16()
    pool.append(x, x, table, lengths, cu_seqlens=cu)
    assert not bool(pool.data.any())
    assert not any(bool(y.any()) for y in pool.read(table, lengths, cu_seqlens=cu, tokens=5))
    assert not bool(pool.attend(x, table, lengths, cu_seqlens=cu).any())
    assert pool.attend(x[:0], table, lengths).shape == (0, 1, 64) and pool.read(table, lengths)[0].shape == (0, 1, 64)
    pool.check_status()


def test_rows_that_see_only_what_is_not_finite():
    """A whole unit of tokens whose keys are NaN, beside finite ones on other warps: NaN for who sees them, at
    any place in the sequence, as one token and in prompts, and groups of values on their own."""
    from stepquant_b200.kernels.kv_cache import QuantizedKVPool
    pool = QuantizedKVPool(40, 1, 128, page_size=16)
    n = 600
    k, v = _rand(n, 1, 128, seed=1).bfloat16(), _rand(n, 1, 128, seed=2).bfloat16()
    table, lengths = torch.arange(1, 39, device="cuda", dtype=torch.int32)[None], torch.tensor([n], device="cuda", dtype=torch.int32)
    q = _rand(n, 4, 128, seed=3).bfloat16()
    for spoil, first, groups in (("k", 64, 2), ("k", 320, 2), ("v", 300, 1)):
        a, b = k.clone(), v.clone()
        (a if spoil == "k" else b)[first:first + 32, :, 70:71 if spoil == "v" else 128] = float("nan")
        pool.append(a, b, table, lengths, cu_seqlens=_ends([n]))
        one = pool.attend(q[-1:], table, lengths)
        many = pool.attend(q, table, lengths, cu_seqlens=_ends([n]))
        bad = torch.zeros(n, 4, 128, dtype=torch.bool, device="cuda")
        bad[first:, :, 64 * (2 - groups):] = True
        assert torch.equal(many.isnan(), bad) and torch.equal(one.isnan(), bad[-1:])
        near = pool.attend(q, table, lengths, cu_seqlens=_ends([n]), window=50)
        bad[first + 32 + 49:] = False
        assert torch.equal(near.isnan(), bad)
    pool.check_status()


def test_attention_is_what_the_reference_computes_without_a_cache():
    """Against attention on the unquantized keys and values: off by what 4 bits cost, a few percent, and no more."""
    layer = _Layer(500, 1, 8, 8)
    q, k, v, at = layer.tokens([500])
    q, out = layer.step(q, k, v, at, torch.tensor([500], device="cuda", dtype=torch.int32), _ends([500]))
    sizes = v.double().abs().transpose(0, 1)
    want, _ = attend(q, turn(k, at, layer.frequencies).transpose(0, 1), v.double().transpose(0, 1), sizes, 0, 128 ** -0.5)
    # A value is within s / 2 of what is held, uniformly: s / sqrt(12) in the mean, s below 6 / 15 of a deviation, so
    # 0.12 of v; keys move a score by 0.12 of a deviation, which moves weights by as much. Twice their sum bounds it.
    assert float((out.double() - want).norm() / want.norm()) < 2 * 0.24


def test_the_example_runs_with_an_attention_layer():
    import importlib.util
    import os

    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("recurrent_layers", os.path.join(ROOT, "examples", "recurrent_layers.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    same, off = module.run(attention=True)
    assert same == same and off == off
