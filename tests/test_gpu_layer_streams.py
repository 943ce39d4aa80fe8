"""The layer operators on other streams than the default one: a side stream, a
stream of 16 SMs (persistent grids and clusters on fewer SMs) and a captured
graph replayed on new inputs.  Results are equal, states among them: sums have
a fixed order, which only the product of up to 128 rows chooses by the SMs (it
splits K over them; test_gpu_matmul.py has it on 16)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _norm(rows, hidden):
    from stepquant_b200.kernels.norm import rms_norm_fp8
    weight = torch.rand(hidden, device="cuda").bfloat16() + 0.5
    residual = torch.randn(rows, hidden, device="cuda").bfloat16()
    return torch.randn(rows, hidden, device="cuda").bfloat16(), [], lambda x: rms_norm_fp8(x, weight, residual)


def _matmul(rows, width, hidden):
    from stepquant_b200.kernels.matmul import matmul_fp8, quantize_weight_fp8
    from stepquant_b200.kernels.norm import quantize_fp8
    w, sw = quantize_weight_fp8(torch.randn(width, hidden, device="cuda"))
    return torch.randn(rows, hidden, device="cuda"), [], lambda x: [matmul_fp8(*quantize_fp8(x), w, sw)]


def _conv(tokens, channels, seqs):
    from stepquant_b200.kernels.conv import causal_conv1d, causal_conv1d_extend, causal_conv1d_step
    weight, pool = torch.randn(channels, 4, device="cuda"), torch.randn(seqs + 1, channels, 3, device="cuda").bfloat16()
    slots = torch.randperm(seqs, device="cuda") + 1
    ends = torch.tensor([tokens * i // seqs for i in range(seqs + 1)], device="cuda", dtype=torch.int32)

    def run(x):
        y, kept = causal_conv1d(x, weight, cu_seqlens=ends)
        return [y, kept, causal_conv1d_extend(x, pool, weight, slots=slots, cu_seqlens=ends),
                causal_conv1d_step(x[:seqs], pool, weight, slots=slots)]

    return torch.randn(tokens, channels, device="cuda").bfloat16(), [pool], run


def _scan(tokens, channels, seqs):
    from stepquant_b200.kernels.scan import selective_scan, selective_scan_extend, selective_scan_step
    a, b, c = -torch.rand(channels, 16, device="cuda"), *torch.randn(2, tokens, 1, 16, device="cuda").bfloat16()
    dt, z = torch.randn(2, tokens, channels, device="cuda").bfloat16()
    pool, slots = torch.randn(seqs + 1, channels, 16, device="cuda"), torch.randperm(seqs, device="cuda") + 1
    ends = torch.tensor([tokens * i // seqs for i in range(seqs + 1)], device="cuda", dtype=torch.int32)

    def run(u):
        y, kept = selective_scan(u, dt, a, b, c, z=z, cu_seqlens=ends)
        first = (t[:seqs] for t in (u, dt, b, c, z))
        u1, dt1, b1, c1, z1 = first
        return [y, kept, selective_scan_extend(pool, u, dt, a, b, c, z=z, slots=slots, cu_seqlens=ends),
                selective_scan_step(pool, u1, dt1, a, b1, c1, z=z1, slots=slots)]

    return torch.randn(tokens, channels, device="cuda").bfloat16(), [pool], run


CASES = [(_norm, 16, 512), (_norm, 4000, 1024), (_norm, 3000, 300), (_norm, 700, 5120), (_matmul, 5, 1000, 4096),
         (_matmul, 60, 5120, 2048), (_matmul, 100, 9000, 1024), (_matmul, 700, 1000, 2048), (_matmul, 2000, 5120, 512),
         (_conv, 70, 264, 3), (_conv, 5000, 1024, 7), (_scan, 40, 96, 2), (_scan, 3000, 256, 3), (_scan, 900, 1024, 60)]


WAYS = [(case, how) for case in CASES for how in ("side", "budget", "graph")
        if not (how == "budget" and case[0] is _matmul and case[1] <= 128)]


@pytest.mark.parametrize("case,how", WAYS, ids=lambda v: v if isinstance(v, str) else v[0].__name__[1:] + "-" + "x".join(map(str, v[1:])))
def test_other_streams(case, how):
    from stepquant_b200.kernels.resources import writeback_resources
    torch.manual_seed(3)
    x, states, run = case[0](*case[1:])
    kept = [s.clone() for s in states]

    def restore():
        for s, k in zip(states, kept):
            s.copy_(k)

    want = [t.clone() for t in run(x)] + [s.clone() for s in states]
    restore()
    torch.cuda.synchronize()
    if how == "graph":
        still = torch.zeros_like(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run(still)
        still.copy_(x)
        restore()
        graph.replay()
    else:
        stream = torch.cuda.Stream() if how == "side" else writeback_resources("cuda", 16).stream
        with torch.cuda.stream(stream):
            got = run(x)
        stream.synchronize()
    torch.cuda.synchronize()
    got = list(got) + states
    assert len(got) == len(want)
    for g, w in zip(got, want):
        bits = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
        assert torch.equal(bits(g), bits(w))
