"""Cases of the operators around the recurrent state: what each is measured on.

A recurrent layer runs residual norm -> 8-bit projection -> short causal
convolution -> state pass -> 8-bit projection.  ``run`` computes one of

  norm       rms_norm / rms_norm_fp8: residual addition, root-mean-square norm,
             e4m3 output with one scale per token and 128 channels
  matmul     matmul_fp8: e4m3 product with a scale per block of 128
  conv       causal_conv1d over concatenated sequences; conv_step one token each
  scan       selective_scan over concatenated sequences; scan_step one token each

in elementary torch operations (``own`` false) or by the package's kernels.
"""
import math
import random

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
SCALE_FLOOR = 1e-30
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
BLOCK = 128


def listed():
    return [
        # One request's token through the residual norm of a 5120-wide layer: latency.
        dict(name="norm one token", op="norm", tokens=1, hidden=5120, dtype="bfloat16", residual=True, fp8=True),
        # An odd batch of a width that no block divides, kept in the input's type.
        dict(name="norm odd rows", op="norm", tokens=777, hidden=4100, dtype="float16", residual=True, fp8=False),
        # 512 prompts of 128 tokens: the prompt pass of the 48-layer stack.
        dict(name="norm prompts", op="norm", tokens=65536, hidden=5120, dtype="bfloat16", residual=True, fp8=True),
        # Input projection (q, k, v, a, b of 16 / 32 heads) of a few requests: the weights' bytes count.
        dict(name="matmul few requests", op="matmul", tokens=8, width=8256, hidden=5120, dtype="bfloat16", residual=False),
        # Output projection of the 48-layer stack's decode step, added to the residual.
        dict(name="matmul decode", op="matmul", tokens=512, width=5120, hidden=4096, dtype="bfloat16", residual=True),
        # Input projection of prompts: the tensor cores' rate counts.
        dict(name="matmul prompts", op="matmul", tokens=16384, width=8256, hidden=5120, dtype="bfloat16", residual=False),
        # q, k, v channels of 16 / 32 heads over 16 ragged prompts.
        dict(name="conv prompts", op="conv", tokens=32768, channels=8192, taps=4, seqs=16, ragged=True, dtype="bfloat16",
             bias=True, initial=False),
        # The same channels, one token of each of 256 requests.
        dict(name="conv decode", op="conv_step", tokens=256, channels=8192, taps=4, dtype="bfloat16", bias=True),
        # Eight ragged prompts through a 4096-channel selective layer, from kept states.
        dict(name="scan prompts", op="scan", tokens=16384, channels=4096, states=16, groups=1, seqs=8, ragged=True,
             dtype="bfloat16", initial=True),
        # One long prompt: the only parallel axes are the channels and the prompt itself.
        dict(name="scan long prompt", op="scan", tokens=8192, channels=2048, states=16, groups=1, seqs=1, ragged=False,
             dtype="bfloat16", initial=False),
        # One token of one request: latency.
        dict(name="scan one token", op="scan_step", tokens=1, channels=4096, states=16, groups=1, dtype="bfloat16"),
        # One token of each of 512 requests: the states' bytes count.
        dict(name="scan decode", op="scan_step", tokens=512, channels=4096, states=16, groups=1, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "matmul", "conv", "conv_step", "scan", "scan_step"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    yes = lambda: rng.random() < 0.5  # noqa: E731
    if op == "norm":
        hidden = _log(rng, 64, 8192)
        hidden -= 0 if yes() else hidden % 8
        most = 65536 * 5120 // hidden // (2 if dtype == "float32" else 1)
        return dict(op=op, tokens=_log(rng, 1, min(65536, most)), hidden=hidden, dtype=dtype, residual=yes(), fp8=yes())
    if op == "matmul":
        hidden, width = 16 * _log(rng, 8, 512), _log(rng, 64, 16384)
        most = 16384 * 8256 * 5120 // (hidden * width)
        return dict(op=op, tokens=_log(rng, 1, min(16384, most)), width=width, hidden=hidden,
                    dtype=rng.choice(["bfloat16", "float16"]), residual=yes())
    if op == "conv":
        channels = _log(rng, 64, 12288)
        tokens = _log(rng, 1, min(65536, 32768 * 8192 // channels // (2 if dtype == "float32" else 1)))
        return dict(op=op, tokens=tokens, channels=channels, taps=rng.choice([2, 3, 4, 4]),
                    seqs=_log(rng, 1, max(1, min(256, tokens))), ragged=yes(), dtype=dtype, bias=yes(), initial=yes())
    if op == "conv_step":
        return dict(op=op, tokens=_log(rng, 1, 1024), channels=_log(rng, 64, 12288), taps=rng.choice([2, 3, 4, 4]),
                    dtype=dtype, bias=yes())
    states, groups = rng.choice([8, 16, 16, 32, 64]), rng.choice([1, 1, 2, 4])
    channels = groups * _log(rng, 32, 2048)
    if op == "scan":
        tokens = _log(rng, 1, min(32768, 16384 * 4096 * 16 // (channels * states)))
        return dict(op=op, tokens=tokens, channels=channels, states=states, groups=groups,
                    seqs=_log(rng, 1, max(1, min(64, tokens))), ragged=yes(), dtype=dtype, initial=yes())
    return dict(op=op, tokens=_log(rng, 1, max(1, min(1024, 512 * 4096 * 16 // (channels * states)))), channels=channels,
                states=states, groups=groups, dtype=dtype)


def _lengths(case):
    """Sequence lengths of a prompt batch: near even, or ragged with empty and one-token ones among them."""
    tokens, seqs = case["tokens"], case["seqs"]
    if not case["ragged"]:
        return [tokens // seqs + (i < tokens % seqs) for i in range(seqs)]
    r = random.Random(tokens * 131 + seqs)
    cuts = sorted(r.randint(0, tokens) for _ in range(seqs - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [tokens])]


def _quantize(x, rows):
    """e4m3 values and fp32 scales of x [R, K] in blocks of `rows` rows and 128 columns."""
    pad = torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK, 0, -x.shape[0] % rows))
    blocks = pad.reshape(pad.shape[0] // rows, rows, pad.shape[1] // BLOCK, BLOCK)
    scale = blocks.abs().amax((1, 3)).clamp_min(SCALE_FLOOR) / E4M3_MAX
    values = (blocks / scale[:, None, :, None]).reshape(pad.shape)[:x.shape[0], :x.shape[1]]
    return values.contiguous().to(torch.float8_e4m3fn), scale


def _cu(case, device):
    ends = [0]
    for n in _lengths(case):
        ends.append(ends[-1] + n)
    return torch.tensor(ends, dtype=torch.int32, device=device)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device=dev)  # noqa: E731
    unit = lambda *shape: torch.rand(*shape, generator=gen, device=dev)  # noqa: E731
    op, tokens = case["op"], case["tokens"]
    dtype = DTYPES[case["dtype"]]
    s = {"case": dict(case)}
    if op == "norm":
        hidden = case["hidden"]
        s["x"] = rand(tokens, hidden).to(dtype)
        s["weight"] = (1 + 0.2 * rand(hidden)).to(dtype)
        # A residual stream carries a few channels that are much larger than the others.
        s["residual"] = (rand(tokens, hidden) * torch.where(unit(hidden) < 0.01, 30.0, 2.0)).to(dtype) if case["residual"] else None
    elif op == "matmul":
        hidden, width = case["hidden"], case["width"]
        s["x"], s["x_scale"] = _quantize(rand(tokens, hidden) * torch.where(unit(hidden) < 0.01, 10.0, 1.0), 1)
        s["w"], s["w_scale"] = _quantize(rand(width, hidden) * hidden ** -0.5, BLOCK)
        s["residual"] = rand(tokens, width).to(dtype) if case["residual"] else None
    elif op in ("conv", "conv_step"):
        channels, taps = case["channels"], case["taps"]
        s["weight"] = rand(channels, taps) * taps ** -0.5
        s["bias"] = 0.1 * rand(channels) if case["bias"] else None
        if op == "conv":
            s["x"] = rand(tokens, channels).to(dtype)
            s["cu"] = _cu(case, dev)
            s["initial"] = rand(case["seqs"], channels, taps - 1).to(dtype) if case["initial"] else None
        else:
            # The projection's output holds the gates behind the convolved channels.
            s["x"] = rand(tokens, channels + 64).to(dtype)[:, :channels]
            s["state"] = rand(tokens + 1, channels, taps - 1).to(dtype)
            s["slots"] = torch.randperm(tokens, generator=gen, device=dev) + 1
    else:
        channels, states, groups = case["channels"], case["states"], case["groups"]
        # u comes from the convolution, z is the second half of the input projection, B and C lie
        # behind the low-rank step size in the second projection's output.
        s["u"] = torch.nn.functional.silu(rand(tokens, channels)).to(dtype)
        s["z"] = rand(tokens, 2 * channels).to(dtype)[:, channels:]
        s["dt"] = (0.5 * rand(tokens, channels)).to(dtype)
        rank = 64
        proj = rand(tokens, rank + 2 * groups * states).to(dtype)
        s["b"] = proj[:, rank:rank + groups * states].unflatten(1, (groups, states))
        s["c"] = proj[:, rank + groups * states:].unflatten(1, (groups, states))
        s["a"] = -torch.arange(1, states + 1, device=dev, dtype=torch.float32) * (0.8 + 0.4 * unit(channels, states))
        s["d"] = rand(channels)
        step = torch.exp(unit(channels) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))  # softplus(dt_bias) = step
        if op == "scan":
            s["cu"] = _cu(case, dev)
            s["initial"] = rand(case["seqs"], channels, states) if case["initial"] else None
        else:
            s["state"] = rand(tokens + 1, channels, states)
            s["slots"] = torch.randperm(tokens, generator=gen, device=dev) + 1
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_norm(s):
    case, dtype = s["case"], s["x"].dtype
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    out = list(_quantize(y, 1)) if case["fp8"] else [y.to(dtype)]
    if s["residual"] is not None:
        out.append(h.to(dtype))
    return out


def _plain_matmul(s):
    hidden, width = s["x"].shape[1], s["w"].shape[0]
    x = s["x"].float() * s["x_scale"].repeat_interleave(BLOCK, 1)[:, :hidden]
    w = s["w"].float() * s["w_scale"].repeat_interleave(BLOCK, 0)[:width].repeat_interleave(BLOCK, 1)[:, :hidden]
    y = x @ w.T
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(DTYPES[s["case"]["dtype"]])


def _silu(x):
    return x / (1 + torch.exp(-x))


def _plain_conv(s):
    """The sequences with their W - 1 earlier inputs before each, then the W taps of every token."""
    x, cu, taps = s["x"].float(), s["cu"].long(), s["case"]["taps"]
    seqs, before = cu.numel() - 1, taps - 1
    first = cu[:-1] + before * torch.arange(seqs, device=x.device)  # of each sequence in the extended rows
    token = torch.arange(x.shape[0], device=x.device)
    at = token + before * (torch.searchsorted(cu[1:], token, right=True) + 1)
    back = torch.arange(before, device=x.device)
    ext = x.new_zeros(x.shape[0] + seqs * before, x.shape[1])
    ext[at] = x
    if s["initial"] is not None:
        ext[first[:, None] + back] = s["initial"].float().transpose(1, 2)
    y = (ext[at[:, None] + torch.arange(-before, 1, device=x.device)] * s["weight"].T).sum(1)
    if s["bias"] is not None:
        y = y + s["bias"]
    last = first + (cu[1:] - cu[:-1])
    return _silu(y).to(s["x"].dtype), ext[last[:, None] + back].transpose(1, 2).to(s["x"].dtype)


def _plain_conv_step(s):
    dtype, slots = s["x"].dtype, s["slots"]
    window = torch.cat([s["state"][slots], s["x"][:, :, None]], 2)
    y = (window.float() * s["weight"]).sum(2)
    if s["bias"] is not None:
        y = y + s["bias"]
    s["state"][slots] = window[:, :, 1:]
    return _silu(y).to(dtype), s["state"]


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(x.clamp_max(20))))


def _scan_terms(s):
    """Decay and input of every (token, channel, state), and C per channel, in 32 bits."""
    per = s["case"]["channels"] // s["case"]["groups"]
    dt = _softplus(s["dt"].float() + s["dt_bias"])
    u = s["u"].float()
    decay = torch.exp(dt[:, :, None] * s["a"])
    put = (dt * u)[:, :, None] * s["b"].float().repeat_interleave(per, 1)
    return decay, put, s["c"].float().repeat_interleave(per, 1), u


def _scan_out(s, h, c, u):
    y = (h * c).sum(2) + s["d"] * u
    return (y * _silu(s["z"].float())).to(s["u"].dtype)


def _plain_scan(s):
    """h_t = decay_t h_{t-1} + put_t by doubling the span that each token's (decay, put) covers."""
    cu = s["cu"].long()
    decay, h, c, u = _scan_terms(s)
    some = cu[1:] > cu[:-1]
    first, last = cu[:-1] * some, (cu[1:] - 1) * some  # an empty sequence points at token 0, a first token too
    some = some[:, None, None]
    if s["initial"] is not None:
        h.index_add_(0, first, torch.where(some, decay[first] * s["initial"], 0.0))
    decay.index_fill_(0, first, 0.0)  # nothing passes from one sequence to the next
    span = 1
    while span < h.shape[0]:
        h[span:] += decay[span:] * h[:-span]
        decay[span:] = decay[span:] * decay[:-span]
        span *= 2
    final = torch.where(some, h[last], 0.0 if s["initial"] is None else s["initial"])
    return _scan_out(s, h, c, u), final


def _plain_scan_step(s):
    decay, put, c, u = _scan_terms(s)
    h = decay * s["state"][s["slots"]] + put
    s["state"][s["slots"]] = h
    return _scan_out(s, h, c, u), s["state"]


_PLAIN = {"norm": _plain_norm, "matmul": _plain_matmul, "conv": _plain_conv, "conv_step": _plain_conv_step,
          "scan": _plain_scan, "scan_step": _plain_scan_step}


# ---------------------------------------------------------------------------
# the package's operators
# ---------------------------------------------------------------------------
def _own_norm(s):
    from stepquant_b200.kernels.norm import rms_norm, rms_norm_fp8
    norm = rms_norm_fp8 if s["case"]["fp8"] else rms_norm
    return norm(s["x"], s["weight"], s["residual"], eps=EPS)


def _own_matmul(s):
    from stepquant_b200.kernels.matmul import matmul_fp8
    return matmul_fp8(s["x"], s["x_scale"], s["w"], s["w_scale"], residual=s["residual"], out_dtype=DTYPES[s["case"]["dtype"]])


def _own_conv(s):
    from stepquant_b200.kernels.conv import causal_conv1d
    return causal_conv1d(s["x"], s["weight"], s["bias"], initial_state=s["initial"], cu_seqlens=s["cu"])


def _own_conv_step(s):
    from stepquant_b200.kernels.conv import causal_conv1d_step
    return causal_conv1d_step(s["x"], s["state"], s["weight"], s["bias"], slots=s["slots"]), s["state"]


def _own_scan(s):
    from stepquant_b200.kernels.scan import selective_scan
    return selective_scan(s["u"], s["dt"], s["a"], s["b"], s["c"], d=s["d"], z=s["z"], dt_bias=s["dt_bias"],
                          initial_state=s["initial"], cu_seqlens=s["cu"])


def _own_scan_step(s):
    from stepquant_b200.kernels.scan import selective_scan_step
    y = selective_scan_step(s["state"], s["u"], s["dt"], s["a"], s["b"], s["c"], d=s["d"], z=s["z"], dt_bias=s["dt_bias"],
                            slots=s["slots"])
    return y, s["state"]


_OWN = {"norm": _own_norm, "matmul": _own_matmul, "conv": _own_conv, "conv_step": _own_conv_step, "scan": _own_scan,
        "scan_step": _own_scan_step}


def run(state):
    out = (_OWN if own else _PLAIN)[state["case"]["op"]](state)
    return list(out) if isinstance(out, (tuple, list)) else [out]


# ---------------------------------------------------------------------------
# floors and 64-bit values
# ---------------------------------------------------------------------------
def work(case):
    op, tokens = case["op"], case["tokens"]
    size = DTYPES[case["dtype"]].itemsize
    if op == "norm":
        values = tokens * case["hidden"]
        wide = values * size * (3 if case["residual"] else 1) + case["hidden"] * size
        out = values + 4 * tokens * -(-case["hidden"] // BLOCK) if case["fp8"] else values * size
        return {"bytes": wide + out, "flops": 6 * values}
    if op == "matmul":
        width, hidden = case["width"], case["hidden"]
        blocks = -(-hidden // BLOCK)
        scales = 4 * blocks * (tokens + -(-width // BLOCK))
        return {"bytes": (tokens + width) * hidden + scales + tokens * width * size * (2 if case["residual"] else 1),
                "flops": 2 * tokens * width * hidden}
    channels = case["channels"]
    if op in ("conv", "conv_step"):
        taps = case["taps"]
        rows = tokens if op == "conv_step" else case["seqs"]
        kept = rows * channels * (taps - 1) * size
        reads = 1 if op == "conv_step" or case["initial"] else 0
        return {"bytes": 2 * tokens * channels * size + (1 + reads) * kept + 4 * channels * (taps + (1 if case["bias"] else 0)),
                "flops": tokens * channels * (2 * taps + 5)}
    states, groups = case["states"], case["groups"]
    kept = 4 * (tokens if op == "scan_step" else case["seqs"]) * channels * states
    reads = 1 if op == "scan_step" or case["initial"] else 0
    return {"bytes": tokens * (4 * channels + 2 * groups * states) * size + (1 + reads) * kept + 4 * channels * (states + 2),
            "flops": tokens * channels * (7 * states + 16)}


def _exact_block_rows(values, scale, rows):
    """values [R, K] times scale per `rows` rows and 128 columns, in 64 bits."""
    r = torch.arange(values.shape[0], device=values.device) // rows
    k = torch.arange(values.shape[1], device=values.device) // BLOCK
    return values.double() * scale.double()[r][:, k]


def _exact_norm(s):
    case = s["case"]
    h = s["x"].double()
    if case["residual"]:
        h = h + s["residual"].double()
    y = h / (h.square().sum(-1, keepdim=True) / h.shape[1] + EPS).sqrt() * s["weight"].double()
    out = [y]
    if case["fp8"]:
        block = torch.arange(h.shape[1], device=h.device) // BLOCK
        scale = torch.zeros(h.shape[0], int(block[-1]) + 1, dtype=torch.float64, device=h.device)
        scale.scatter_reduce_(1, block.expand(h.shape), y.abs(), "amax")
        scale = scale.clamp_min(SCALE_FLOOR) / E4M3_MAX
        out = [y / scale[:, block], scale]
    return out + ([h] if case["residual"] else [])


def _exact_matmul(s):
    y = _exact_block_rows(s["x"], s["x_scale"], 1) @ _exact_block_rows(s["w"], s["w_scale"], BLOCK).T
    return [y if s["residual"] is None else y + s["residual"].double()]


def _exact_conv(s):
    x, taps = s["x"].double(), s["case"]["taps"]
    step = s["case"]["op"] == "conv_step"
    ends = list(range(x.shape[0] + 1)) if step else s["cu"].tolist()
    old = s["state"][s["slots"]] if step else s["initial"]
    y, kept = torch.zeros_like(x), []
    w = s["weight"].double()
    if step:
        window = torch.cat([old.double(), x[:, :, None]], 2)
        y, kept = torch.einsum("bdw,dw->bd", window, w), window[:, :, 1:]
    else:
        for n in range(len(ends) - 1):
            part = x[ends[n]:ends[n + 1]].T
            lead = x.new_zeros(x.shape[1], taps - 1) if old is None else old[n].double()
            window = torch.cat([lead, part], 1)
            kept.append(window[:, window.shape[1] - (taps - 1):])
            for j in range(taps):
                y[ends[n]:ends[n + 1]] += (w[:, j:j + 1] * window[:, j:j + part.shape[1]]).T
        kept = torch.stack(kept)
    if s["bias"] is not None:
        y = y + s["bias"].double()
    y = y * torch.sigmoid(y)
    if step:
        state = s["state"].double()
        state[s["slots"]] = kept
        kept = state
    return [y, kept]


def _exact_scan(s):
    case = s["case"]
    step = case["op"] == "scan_step"
    tokens, channels, states, groups = case["tokens"], case["channels"], case["states"], case["groups"]
    dev = s["u"].device
    lengths = [1] * tokens if step else _lengths(case)
    if step:
        h = s["state"][s["slots"]].double()
    else:
        h = torch.zeros(len(lengths), channels, states, dtype=torch.float64, device=dev)
        h = h if s["initial"] is None else s["initial"].double()
    length = torch.tensor(lengths, device=dev)
    start = length.cumsum(0) - length
    group = torch.arange(channels, device=dev) // (channels // groups)
    y = torch.zeros(tokens, channels, dtype=torch.float64, device=dev)
    a, skip, bias = s["a"].double(), s["d"].double(), s["dt_bias"].double()
    order = sorted(range(len(lengths)), key=lambda n: -lengths[n])
    h, start = h[order], start[order]
    for t in range(max(lengths)):
        live = sum(n > t for n in lengths)
        at = start[:live] + t
        dt = torch.nn.functional.softplus(s["dt"][at].double() + bias, threshold=50.0)
        u, z = s["u"][at].double(), s["z"][at].double()
        h[:live] = torch.exp(dt[..., None] * a) * h[:live] + (dt * u)[..., None] * s["b"][at].double()[:, group]
        y[at] = ((h[:live] * s["c"][at].double()[:, group]).sum(-1) + skip * u) * (z * torch.sigmoid(z))
    back = torch.empty_like(h)
    back[order] = h
    if step:
        state = s["state"].double()
        state[s["slots"]] = back
        back = state
    return [y, back]


def exact(case, seed):
    """run()'s outputs from the definitions in 64 bits; e4m3 values before their rounding."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        return _exact_norm(s)
    if op == "matmul":
        return _exact_matmul(s)
    return _exact_conv(s) if op.startswith("conv") else _exact_scan(s)
