"""causal_conv1d and its single-token form (csrc/sq_conv.cu) against 64-bit arithmetic.

Tolerances: five products and sums, each rounded to 2^-24 of the sum of
magnitudes M = |bias| + sum |w x|; SiLU passes that on with a slope of at most
1.1 and adds its exponential (arguments up to ~20: 24 roundings) and quotient:
ACC = 8 * 2^-24 of M and SILU = 32 * 2^-24 of |y|.  Rounding is monotone, so an
output lies between the roundings of both ends of that interval.  States are
copies and equal.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

ACC, SILU = 8 * 2.0 ** -24, 32 * 2.0 ** -24


def _reference(x, weight, bias, cu, initial, activation="silu"):
    """(y, sum of magnitudes, final state), one sequence after the other."""
    taps, w = weight.shape[1], weight.double()
    y, size, kept = torch.zeros_like(x, dtype=torch.float64), torch.zeros_like(x, dtype=torch.float64), []
    for n in range(len(cu) - 1):
        lead = torch.zeros(x.shape[1], taps - 1, device=x.device, dtype=x.dtype) if initial is None else initial[n]
        window = torch.cat([lead, x[cu[n]:cu[n + 1]].T], 1)
        kept.append(window[:, window.shape[1] - (taps - 1):])
        for j in range(taps):
            part = w[:, j:j + 1] * window[:, j:j + cu[n + 1] - cu[n]].double()
            y[cu[n]:cu[n + 1]] += part.T
            size[cu[n]:cu[n + 1]] += part.abs().T
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return (y * torch.sigmoid(y) if activation else y), size, torch.stack(kept)


def _close(got, want, size):
    off = 1.1 * ACC * size + want.abs() * SILU + 1e-40
    inside = ((want - off).to(got.dtype) <= got) & (got <= (want + off).to(got.dtype))
    assert bool(inside.all()), (got[~inside], want[~inside])


def _data(tokens, channels, taps, dtype, seqs, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    return rand(tokens, channels).to(dtype), rand(channels, taps), rand(channels), rand(seqs, channels, taps - 1).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("taps", [2, 3, 4])
@pytest.mark.parametrize("channels,cu", [(1, [0, 1]), (64, [0, 2]), (8, [0, 0, 1, 3, 3, 6, 70, 70]), (100, [0, 63, 64, 65, 193]),
                                         (1032, [0, 200]), (2000, [0, 8, 16, 24, 25, 153])])
@pytest.mark.parametrize("with_state", [False, True])
def test_prompts(channels, cu, taps, dtype, with_state):
    from stepquant_b200.kernels.conv import causal_conv1d
    x, weight, bias, initial = _data(cu[-1], channels, taps, dtype, len(cu) - 1)
    initial = initial if with_state else None
    bias = bias if with_state else None
    activation = "silu" if taps != 3 else None
    y, final = causal_conv1d(x, weight, bias, initial_state=initial, activation=activation,
                             cu_seqlens=torch.tensor(cu, device="cuda", dtype=torch.int32))
    want, size, kept = _reference(x, weight, bias, cu, initial, activation)
    assert y.dtype == dtype
    _close(y, want, size)
    assert torch.equal(final, kept)


def test_many_strips_and_strided_rows():
    """Enough tokens for the longest strips; rows that are slices of a wider
    projection, aligned for wide loads or not; a leading batch of 1."""
    from stepquant_b200.kernels.conv import causal_conv1d
    cu = [0, 5000, 5001, 30000]
    x, weight, bias, initial = _data(cu[-1], 1024, 4, torch.bfloat16, 3, 1)
    ends = torch.tensor(cu, device="cuda")
    want, size, kept = _reference(x, weight, bias, cu, initial)
    for pad in (0, 8, 3):
        wide = torch.zeros(cu[-1], 1024 + 2 * pad, device="cuda", dtype=torch.bfloat16)
        wide[:, pad:pad + 1024] = x
        y, final = causal_conv1d(wide[:, pad:pad + 1024], weight, bias, initial_state=initial, cu_seqlens=ends)
        _close(y, want, size)
        assert torch.equal(final, kept)
    y1, none = causal_conv1d(x[None, :5000], weight[:, None], bias, initial_state=initial[:1], output_final_state=False)
    assert none is None and y1.shape == (1, 5000, 1024) and torch.equal(y1[0], y[:5000])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("taps,channels,batch", [(2, 8, 1), (3, 33, 5), (4, 1, 2), (4, 1024, 7), (4, 2052, 3), (3, 1032, 300)])
def test_step(taps, channels, batch, dtype):
    from stepquant_b200.kernels.conv import causal_conv1d_step
    x, weight, bias, _ = _data(batch, channels, taps, dtype, batch, 2)
    pool = torch.randn(batch + 2, channels, taps - 1, device="cuda").to(dtype)
    before = pool.clone()
    slots = (torch.randperm(batch, device="cuda") + 1)
    y = causal_conv1d_step(x, pool, weight, bias, slots=slots)
    want, size, kept = _reference(x, weight, bias, list(range(batch + 1)), before[slots])
    _close(y, want, size)
    assert torch.equal(pool[slots], kept)
    assert torch.equal(pool[0], before[0]) and torch.equal(pool[-1], before[-1])
    again = before[1:batch + 1].clone()  # no slots: row i for request i
    y2 = causal_conv1d_step(x, again, weight, bias)
    want, size, kept = _reference(x, weight, bias, list(range(batch + 1)), before[1:batch + 1])
    _close(y2, want, size)
    assert torch.equal(again, kept)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("taps", [2, 3, 4])
@pytest.mark.parametrize("channels", [2, 258, 770, 771])
def test_rows_aligned_for_pairs(channels, taps, dtype):
    """Channels that four do not divide, by pairs or singly; prompts, then a token of each."""
    from stepquant_b200.kernels.conv import causal_conv1d, causal_conv1d_step
    cu = [0, 1, 1, 71, 72, 300]
    x, weight, bias, initial = _data(cu[-1], channels, taps, dtype, len(cu) - 1, 9)
    y, final = causal_conv1d(x, weight, bias, initial_state=initial, cu_seqlens=torch.tensor(cu, device="cuda"))
    want, size, kept = _reference(x, weight, bias, cu, initial)
    _close(y, want, size)
    assert torch.equal(final, kept)
    x, pool = x[:5], kept.clone()
    y = causal_conv1d_step(x, pool, weight, bias)
    want, size, kept = _reference(x, weight, bias, list(range(6)), kept)
    _close(y, want, size)
    assert torch.equal(pool, kept)


def test_prompt_in_parts_and_tokens():
    """A prompt in one pass = in two passes = a pass and single tokens, bit for bit."""
    from stepquant_b200.kernels.conv import causal_conv1d, causal_conv1d_extend, causal_conv1d_step
    x, weight, bias, _ = _data(90, 264, 4, torch.bfloat16, 1, 3)
    whole, final = causal_conv1d(x, weight, bias)
    first, state = causal_conv1d(x[:47], weight, bias)
    second, state2 = causal_conv1d(x[47:], weight, bias, initial_state=state)
    assert torch.equal(torch.cat([first, second]), whole) and torch.equal(state2, final)
    pool = torch.zeros(4, 264, 3, device="cuda", dtype=torch.bfloat16)
    slot = torch.tensor([2], device="cuda")
    part = causal_conv1d_extend(x[:80], pool, weight, bias, slots=slot)
    tokens = [causal_conv1d_step(x[t:t + 1], pool, weight, bias, slots=slot) for t in range(80, 90)]
    assert torch.equal(torch.cat([part] + tokens), whole) and torch.equal(pool[2:3], final)


def test_padding_and_slots_outside():
    """Slots 0, -1 and past the pool: zero outputs, no state touched, the last one flagged."""
    from stepquant_b200.kernels.conv import causal_conv1d_extend, causal_conv1d_step
    x, weight, bias, _ = _data(6, 72, 4, torch.bfloat16, 1, 4)
    pool = torch.randn(3, 72, 3, device="cuda").bfloat16()
    before = pool.clone()
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    y = causal_conv1d_step(x[:3], pool, weight, bias, slots=torch.tensor([0, -1, 1], device="cuda"), status=status)
    assert bool((y[:2] == 0).all()) and bool((y[2] != 0).any()) and int(status) == 0
    assert torch.equal(pool[0], before[0]) and torch.equal(pool[2], before[2])
    y = causal_conv1d_extend(x, pool, weight, bias, slots=torch.tensor([3, 2], device="cuda"), status=status,
                             cu_seqlens=torch.tensor([0, 4, 6], device="cuda"))
    assert bool((y[:4] == 0).all()) and int(status) == 1
    want, size, kept = _reference(x[4:], weight, bias, [0, 2], before[2:3])
    _close(y[4:], want, size)
    assert torch.equal(pool[2:3], kept)


def test_no_tokens_and_extremes():
    from stepquant_b200.kernels.conv import causal_conv1d, causal_conv1d_step
    x, weight, bias, initial = _data(5, 24, 4, torch.float32, 2, 5)
    y, final = causal_conv1d(x[:0], weight, bias, initial_state=initial, cu_seqlens=torch.tensor([0, 0, 0], device="cuda"))
    assert y.shape == (0, 24) and torch.equal(final, initial)
    assert causal_conv1d_step(x[:0], initial[:0], weight, bias).shape == (0, 24)
    x[2, 3], x[3, 5], x[4, 7] = float("nan"), 1e30, -1e30
    weight[:] = 1
    y, _ = causal_conv1d(x, weight)
    assert bool(y[2:, 3].isnan().all()) and bool(y[:2].isfinite().all())
    assert float(y[3, 5]) == 1e30 or abs(float(y[3, 5]) / 1e30 - 1) < 1e-6
    assert float(y[4, 7].abs()) == 0.0
    assert bool(y[:, :3].isfinite().all())


def test_default_boundaries_under_capture():
    """One sequence without cu_seqlens, captured and replayed on new inputs: no copy from the host."""
    from stepquant_b200.kernels.conv import causal_conv1d, sequence_ends
    for tokens in (0, 1, 77, 2 ** 31 - 1):
        ends = sequence_ends(None, tokens, torch.device("cuda", 0))
        assert ends.tolist() == [0, tokens] and ends.dtype == torch.int32
    x, weight, bias, _ = _data(77, 264, 4, torch.bfloat16, 1, 11)
    want = causal_conv1d(x, weight, bias)
    still = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = causal_conv1d(still, weight, bias)
    still.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("channels", [264, 131])
@pytest.mark.parametrize("cu,tokens", [([0, 30, 41], 41), ([0, 30, 41], 300), ([5, 30, 30, 99], 99), ([131, 131, 402], 5000),
                                       ([0], 50), ([7], 7), ([0, 0], 333), ([300, 300, 300], 300), ([77, 78], 79)])
def test_tokens_of_no_sequence_are_zero(cu, tokens, channels, dtype):
    """Tokens before the first boundary and past the last, as a padded batch has them, in memory that held NaN."""
    from stepquant_b200.kernels.conv import causal_conv1d
    x, weight, bias, _ = _data(tokens, channels, 4, dtype, 1, 12)
    x[:cu[0]] = x[cu[-1]:] = float("nan")
    want = torch.zeros(tokens, channels, device="cuda", dtype=dtype)
    if len(cu) > 1:
        inner = torch.tensor(cu, device="cuda") - cu[0]
        want[cu[0]:cu[-1]], kept = causal_conv1d(x[cu[0]:cu[-1]], weight, bias, cu_seqlens=inner)
    for _ in range(3):
        torch.full((tokens, channels), float("nan"), device="cuda", dtype=dtype)  # freed at once: the next output's memory
        y, final = causal_conv1d(x, weight, bias, cu_seqlens=torch.tensor(cu, device="cuda"))
        assert torch.equal(y, want)
        assert len(cu) == 1 or torch.equal(final, kept)
