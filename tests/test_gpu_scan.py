"""selective_scan and its single-token form (csrc/sq_scan.cu) against the recurrence in 64 bits.

Tolerances follow the recurrence.  With e = 2^-24 and M_t = sum of the
magnitudes that h_t is made of (M_t = decay M_{t-1} + |dt' u B|), a step adds to
h an error of at most

    decay M_{t-1} (8 + 16 |dt' A|) e + 12 |dt' u B| e

(softplus and the argument of the exponential off by a few roundings, the
exponential by four, the product and the sum by one each), and passes on decay
times the error so far; E_t is that sum.  y adds N + 4 roundings of sum |C| M +
|D u| and 32 for SiLU.  Rounding is monotone, so an output lies between the
roundings of both ends of that interval.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

E24 = 2.0 ** -24


def _reference(t, cu, initial, softplus=True):
    """(y, its limit before rounding, final state, its limit), token by token."""
    u, dt, z, b, c = (None if t[k] is None else t[k].double() for k in ("u", "dt", "z", "b", "c"))
    channels, groups = u.shape[1], b.shape[1]
    of = torch.arange(channels, device=u.device) // (channels // groups)
    a = t["a"].double()
    step = dt + (0 if t["dt_bias"] is None else t["dt_bias"].double())
    step = torch.nn.functional.softplus(step, threshold=40.0) if softplus else step
    skip = torch.zeros(channels, device=u.device) if t["d"] is None else t["d"]
    y, limit, finals, final_limits = torch.zeros_like(u), torch.zeros_like(u), [], []
    for n in range(len(cu) - 1):
        h = torch.zeros_like(a) if initial is None else initial[n].double()
        size, error = h.abs(), torch.zeros_like(h)
        for i in range(cu[n], cu[n + 1]):
            x = step[i][:, None] * a
            decay, put = torch.exp(x), (step[i] * u[i])[:, None] * b[i][of]
            error = decay * error + decay * size * (8 + 16 * x.abs()) * E24 + 12 * put.abs() * E24
            h, size = decay * h + put, decay * size + put.abs()
            y[i] = (h * c[i][of]).sum(1) + skip.double() * u[i]
            limit[i] = (c[i][of].abs() * (error + (a.shape[1] + 4) * E24 * size)).sum(1) + 4 * E24 * (skip.double() * u[i]).abs()
        finals.append(h)
        final_limits.append(error + E24 * size)
    if z is not None:
        gate = z * torch.sigmoid(z)
        y, limit = y * gate, limit * gate.abs() * 1.01 + 32 * E24 * (y * gate).abs()
    return y, limit, torch.stack(finals), torch.stack(final_limits)


def _close(y, final, reference):
    want, limit, state, state_limit = reference
    limit = limit + 1e-38
    inside = ((want - limit).to(y.dtype) <= y) & (y <= (want + limit).to(y.dtype))
    assert bool(inside.all()), (y[~inside], want[~inside])
    if final is not None:
        error = (final.double() - state).abs()
        assert bool((error <= state_limit + 1e-38).all()), float((error / (state_limit + 1e-38)).max())


def _data(tokens, channels, states, groups, dtype, seed=0, plain=False):
    gen = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    t = {"u": rand(tokens, channels).to(dtype), "dt": rand(tokens, channels).to(dtype),
         "z": None if plain else rand(tokens, channels).to(dtype),
         "b": rand(tokens, groups, states).to(dtype), "c": rand(tokens, groups, states).to(dtype),
         "a": -torch.rand(channels, states, generator=gen, device="cuda") * states,
         "d": None if plain else rand(channels), "dt_bias": None if plain else rand(channels) * 2 - 4}
    return t


def _options(t):
    return {k: t[k] for k in ("d", "z", "dt_bias")}


def _core(t):
    return [t[k] for k in ("u", "dt", "a", "b", "c")]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("channels,states,groups,cu", [
    (1, 4, 1, [0, 1]), (40, 8, 1, [0, 0, 3, 3, 35, 36]), (64, 16, 1, [0, 33, 64, 128]), (66, 16, 2, [0, 31, 95, 95]),
    (60, 32, 4, [0, 70]), (21, 64, 3, [0, 5, 38]), (300, 16, 1, [0, 2, 40])])
def test_prompts(channels, states, groups, cu, dtype):
    from stepquant_b200.kernels.scan import selective_scan
    t = _data(cu[-1], channels, states, groups, dtype)
    initial = torch.randn(len(cu) - 1, channels, states, device="cuda")
    for start, ends in ((initial, cu), (None, cu)):
        y, final = selective_scan(*_core(t), **_options(t), initial_state=start,
                                  cu_seqlens=torch.tensor(ends, device="cuda", dtype=torch.int32))
        assert y.dtype == dtype and final.dtype == torch.float32
        _close(y, final, _reference(t, ends, start))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("channels,groups,batch", [(40, 1, 1), (70, 2, 5), (300, 3, 40), (2048, 1, 9)])
def test_four_states(channels, groups, batch, dtype):
    """Rows of B and C of half a 16-byte piece, many tokens; a token of many requests."""
    from stepquant_b200.kernels.scan import selective_scan, selective_scan_step
    t = _data(90, channels, 4, groups, dtype, 12)
    cu = [0, 33, 34, 90]
    initial = torch.randn(3, channels, 4, device="cuda")
    y, final = selective_scan(*_core(t), **_options(t), initial_state=initial, cu_seqlens=torch.tensor(cu, device="cuda"))
    _close(y, final, _reference(t, cu, initial))
    t = _data(batch, channels, 4, groups, dtype, 13)
    pool = torch.randn(batch, channels, 4, device="cuda")
    before = pool.clone()
    y = selective_scan_step(pool, *_core(t), **_options(t))
    _close(y, pool, _reference(t, list(range(batch + 1)), before))


def test_without_gate_skip_bias_softplus():
    from stepquant_b200.kernels.scan import selective_scan
    t = _data(50, 96, 16, 1, torch.float32, 1, plain=True)
    t["dt"] = t["dt"].abs() * 0.1
    y, final = selective_scan(*_core(t), dt_softplus=False)
    _close(y, final, _reference(t, [0, 50], None, softplus=False))
    y, none = selective_scan(t["u"][None], t["dt"][None], t["a"], t["b"][None, :, 0], t["c"][None], output_final_state=False)
    assert none is None and y.shape == (1, 50, 96)
    _close(y[0], None, _reference(t, [0, 50], None))


@pytest.mark.parametrize("channels,states,groups,cu", [(256, 16, 1, [0, 3000]), (128, 8, 2, [0, 1, 1500, 1500, 2600]),
                                                       (64, 64, 1, [0, 1111]), (320, 32, 1, [0, 900, 901, 1800])])
def test_long_prompts_of_few_channels(channels, states, groups, cu):
    """Few channels and sequences with many tokens, slow and fast decays."""
    from stepquant_b200.kernels.scan import selective_scan
    t = _data(cu[-1], channels, states, groups, torch.bfloat16, 2)
    t["a"] *= torch.logspace(-3, 0, channels, device="cuda")[:, None]
    initial = torch.randn(len(cu) - 1, channels, states, device="cuda")
    y, final = selective_scan(*_core(t), **_options(t), initial_state=initial, cu_seqlens=torch.tensor(cu, device="cuda"))
    _close(y, final, _reference(t, cu, initial))


@pytest.mark.parametrize("channels,states,groups,cu", [
    (1032, 16, 1, [0, 200]), (70, 4, 2, [0, 500]), (99, 8, 3, [0, 31, 63, 96, 160, 161, 161, 450]),
    (224, 64, 4, [0, 400, 700]), (146, 32, 1, [0, 64, 129, 460]), (36, 16, 4, [0, 32, 64, 600])])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_short_chunks(channels, states, groups, cu, dtype):
    """Prompts of a few hundred tokens, cut into chunks too; into a pool's rows, one request padding."""
    from stepquant_b200.kernels.scan import selective_scan, selective_scan_extend
    t = _data(cu[-1], channels, states, groups, dtype, 11)
    t["a"] *= torch.logspace(-3, 0, channels, device="cuda")[:, None]
    ends = torch.tensor(cu, device="cuda")
    want = _reference(t, cu, None)
    y, final = selective_scan(*_core(t), **_options(t), cu_seqlens=ends)
    _close(y, final, want)
    y2, none = selective_scan(*_core(t), **_options(t), cu_seqlens=ends, output_final_state=False)
    assert none is None and torch.equal(y2, y)
    pool = torch.zeros(len(cu) + 1, channels, states, device="cuda")
    slots = torch.arange(len(cu) - 1, 0, -1, device="cuda")
    slots[0] = 0
    y3 = selective_scan_extend(pool, *_core(t), **_options(t), slots=slots, cu_seqlens=ends)
    assert torch.equal(y3[cu[1]:], y[cu[1]:]) and not y3[:cu[1]].any()
    assert torch.equal(pool[slots[1:]], final[1:]) and not pool[0].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("channels,states,groups,batch", [(1, 4, 1, 1), (33, 8, 1, 5), (128, 16, 2, 300), (60, 32, 4, 3),
                                                          (21, 64, 3, 2), (4096, 16, 1, 9)])
def test_step(channels, states, groups, batch, dtype):
    from stepquant_b200.kernels.scan import selective_scan_step
    t = _data(batch, channels, states, groups, dtype, 3)
    pool = torch.randn(batch + 2, channels, states, device="cuda")
    before = pool.clone()
    slots = torch.randperm(batch, device="cuda") + 1
    y = selective_scan_step(pool, *_core(t), **_options(t), slots=slots)
    _close(y, pool[slots], _reference(t, list(range(batch + 1)), before[slots]))
    assert torch.equal(pool[0], before[0]) and torch.equal(pool[-1], before[-1])
    again = before[1:batch + 1].clone()
    y = selective_scan_step(again, *_core(t), **_options(t))
    _close(y, again, _reference(t, list(range(batch + 1)), before[1:batch + 1]))


def test_strided_inputs():
    """z, B, C as slices of projections, at odd offsets too."""
    from stepquant_b200.kernels.scan import selective_scan, selective_scan_step
    tokens, channels, states = 70, 96, 16
    t = _data(tokens, channels, states, 2, torch.bfloat16, 4)
    for off in (0, 5, 8):
        wide = torch.zeros(tokens, 2 * channels + off, device="cuda", dtype=torch.bfloat16)
        wide[:, off:off + channels] = t["z"]
        wide[:, off + channels:] = t["u"]
        proj = torch.zeros(tokens, off + 4 * states, device="cuda", dtype=torch.bfloat16)
        proj[:, off:off + 2 * states] = t["b"].flatten(1)
        proj[:, off + 2 * states:] = t["c"].flatten(1)
        b, c = proj[:, off:].unflatten(1, (2, 2, states)).unbind(1)
        args = (wide[:, off + channels:], t["dt"], t["a"], b, c)
        options = dict(d=t["d"], z=wide[:, off:off + channels], dt_bias=t["dt_bias"])
        y, final = selective_scan(*args, **options)
        want = _reference(t, [0, tokens], None)
        _close(y, final, want)
        state = torch.zeros(tokens, channels, states, device="cuda")
        y = selective_scan_step(state, *args, **options)
        _close(y, state, _reference(t, list(range(tokens + 1)), None))


def test_pool_prompt_in_parts_and_tokens():
    """SelectiveStatePool: a prompt in parts, then single tokens, against one pass."""
    from stepquant_b200.kernels.scan import SelectiveStatePool, selective_scan
    t = _data(90, 160, 16, 1, torch.bfloat16, 5)
    pool = SelectiveStatePool(4, 160, 16)
    slot = torch.tensor([3], device="cuda")
    part = lambda lo, hi: {k: v[lo:hi] if k in ("u", "dt", "z", "b", "c") else v for k, v in t.items()}  # noqa: E731
    outs = []
    for lo, hi in ((0, 40), (40, 41), (41, 80)):
        p = part(lo, hi)
        outs.append(pool.extend(*_core(p), slot, torch.tensor([0, hi - lo], device="cuda"), **_options(p)))
    for i in range(80, 90):
        p = part(i, i + 1)
        outs.append(pool.step(*_core(p), slot, **_options(p)))
    want = _reference(t, [0, 90], None)
    _close(torch.cat(outs), pool.state[3:4], want)
    y, final = selective_scan(*_core(t), **_options(t))
    _close(y, final, want)
    assert bool((pool.state[:3] == 0).all())
    pool.copy(slot, torch.tensor([1], device="cuda"))
    assert torch.equal(pool.state[1], pool.state[3])
    pool.clear(slot)
    assert bool((pool.state[3] == 0).all())
    pool.check_status()


def test_padding_and_slots_outside():
    from stepquant_b200.kernels.scan import SelectiveStatePool
    t = _data(6, 40, 8, 1, torch.float16, 6)
    pool = SelectiveStatePool(3, 40, 8, dtype=torch.float16)
    pool.state.normal_()
    before = pool.state.clone()
    three = {k: v[:3] if k in ("u", "dt", "z", "b", "c") else v for k, v in t.items()}
    y = pool.step(*_core(three), torch.tensor([0, -5, 1], device="cuda"), **_options(three))
    assert bool((y[:2] == 0).all()) and bool((y[2] != 0).any())
    pool.check_status()
    y = pool.extend(*_core(t), torch.tensor([3, 2], device="cuda"), torch.tensor([0, 4, 6], device="cuda"), **_options(t))
    assert bool((y[:4] == 0).all()) and bool((y[4:] != 0).any())
    assert torch.equal(pool.state[0], before[0])
    with pytest.raises(IndexError):
        pool.check_status()
    pool.check_status()


def test_no_tokens_and_repeatability():
    """Empty batches keep their states; two runs give the same bits."""
    from stepquant_b200.kernels.scan import selective_scan, selective_scan_step
    t = _data(0, 48, 16, 1, torch.bfloat16, 7)
    initial = torch.randn(2, 48, 16, device="cuda")
    y, final = selective_scan(*_core(t), **_options(t), initial_state=initial, cu_seqlens=torch.tensor([0, 0, 0], device="cuda"))
    assert y.shape == (0, 48) and torch.equal(final, initial)
    assert selective_scan_step(initial[:0], *_core(t), **_options(t)).shape == (0, 48)
    t = _data(2000, 48, 16, 1, torch.bfloat16, 8)
    one, two = (selective_scan(*_core(t), **_options(t)) for _ in range(2))
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


def test_nan_stays_in_its_channel_and_sequence():
    from stepquant_b200.kernels.scan import selective_scan
    t = _data(60, 48, 16, 1, torch.float32, 9)
    t["u"][10, 5] = float("nan")
    y, final = selective_scan(*_core(t), **_options(t), cu_seqlens=torch.tensor([0, 30, 60], device="cuda"))
    assert bool(y[10:30, 5].isnan().all()) and bool(final[0, 5].isnan().all())
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[10:30, 5] = False
    assert bool(y[keep].isfinite().all()) and bool(final[1].isfinite().all())


def test_large_steps():
    """softplus beyond its switch (dt > 20) and far below zero; decays that underflow."""
    from stepquant_b200.kernels.scan import selective_scan
    t = _data(40, 48, 16, 1, torch.float32, 10)
    t["dt"][::3] = 25.0
    t["dt"][1::3] = -30.0
    y, final = selective_scan(*_core(t), **_options(t))
    _close(y, final, _reference(t, [0, 40], None))


@pytest.mark.parametrize("tokens", [40, 600])
def test_default_boundaries_under_capture(tokens):
    """One sequence without cu_seqlens, whole and in chunks, captured and replayed on new inputs."""
    from stepquant_b200.kernels.scan import selective_scan
    t = _data(tokens, 64, 16, 1, torch.bfloat16, 14)
    want = selective_scan(*_core(t), **_options(t))
    still = torch.zeros_like(t["u"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = selective_scan(still, *_core(t)[1:], **_options(t))
    still.copy_(t["u"])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("channels", [48, 200])
@pytest.mark.parametrize("cu,tokens", [([0, 30, 41], 41), ([0, 30, 41], 70), ([5, 30, 30, 99], 99), ([131, 131, 402], 1500),
                                       ([0, 700, 1400], 2001), ([0], 50), ([0, 0], 333), ([300, 300, 300], 300), ([77, 78], 79),
                                       ([600, 1600], 1611)])
def test_tokens_of_no_sequence_are_zero(cu, tokens, channels, dtype):
    """Tokens before the first boundary and past the last, whole sequences and chunks, in memory that held NaN."""
    from stepquant_b200.kernels.scan import selective_scan
    t = _data(tokens, channels, 16, 1, dtype, 15)
    for k in ("u", "dt", "z", "b", "c"):
        t[k][:cu[0]] = t[k][cu[-1]:] = float("nan")
    want = torch.zeros(tokens, channels, device="cuda", dtype=torch.float64)
    limit = torch.zeros_like(want)
    states = state_limits = torch.zeros(0, channels, 16, device="cuda", dtype=torch.float64)
    if len(cu) > 1:
        inner = {k: v[cu[0]:cu[-1]] if k in ("u", "dt", "z", "b", "c") else v for k, v in t.items()}
        want[cu[0]:cu[-1]], limit[cu[0]:cu[-1]], states, state_limits = _reference(inner, [at - cu[0] for at in cu], None)
    for _ in range(3):
        torch.full((tokens, channels), float("nan"), device="cuda", dtype=dtype)  # freed at once: the next output's memory
        y, final = selective_scan(*_core(t), **_options(t), cu_seqlens=torch.tensor(cu, device="cuda"))
        outside = torch.ones(tokens, device="cuda", dtype=torch.bool)
        outside[cu[0]:cu[-1]] = False
        assert not bool(y[outside].isnan().any()) and not bool(y[outside].any())
        _close(y, final, (want, limit, states, state_limits))


@pytest.mark.parametrize("single", [False, True])
def test_step_sizes_alone(single):
    """softplus(dt + dt_bias) by itself: u = b = 1, one token from a state of zero, so that the
    state is dt'.  Off by at most 16 * 2^-24 of itself: the exponential 4, the first order
    correction of its argument, its product and the quotient's sum 1 each, the reciprocal 2, the
    quotient, its square, the series and the sum with max(x, 0) 1 each, with room for what the
    argument's own rounding error was rounded to.  Values below 2^-126 may be flushed to zero."""
    from stepquant_b200.kernels.scan import selective_scan, selective_scan_step
    raw = torch.cat([torch.linspace(-80, 30, 100001), torch.linspace(-1, 1, 20001), torch.linspace(-100, -85, 301),
                     torch.tensor([0.0, 1e-30, -1e-30, 1e4, 3e38])])
    raw = torch.nn.functional.pad(raw, (0, -len(raw) % 1000)).cuda().view(-1, 1000)
    for bias in (0.0, -0.03, 0.07, -1.0, -2.7, -4.6, -6.9, 5.3, 40.0, -60.0):
        t = dict(a=torch.zeros(1000, 4, device="cuda"), b=torch.ones(len(raw), 1, 4, device="cuda"), u=torch.ones_like(raw),
                 dt_bias=torch.full((1000,), bias, device="cuda"))
        if single:
            state = torch.zeros(len(raw), 1000, 4, device="cuda")
            selective_scan_step(state, t["u"], raw, t["a"], t["b"], t["b"], dt_bias=t["dt_bias"])
        else:
            state = selective_scan(t["u"], raw, t["a"], t["b"], t["b"], dt_bias=t["dt_bias"],
                                   cu_seqlens=torch.arange(len(raw) + 1, device="cuda", dtype=torch.int32))[1]
        x = raw.double() + t["dt_bias"].double()
        want = torch.clamp_min(x, 0) + torch.log1p(torch.exp(-x.abs()))
        error = (state[:, :, 0].double() - want).abs()
        limit = 16 * E24 * want + torch.where(want < 2.0 ** -125, want, 0.0)
        assert bool((error <= limit).all()), (bias, float((error / want.clamp_min(2.0 ** -125)).max() / E24))
        assert bool((state == state[:, :, :1]).all())
