"""Cases of the attention layers between recurrent ones: what each operator is measured on.

Such a layer rotates its queries and keys by their positions, appends keys and
values to a paged cache in 4 bits and attends over it.  ``run`` computes one of

  rotary     rotary: queries rotated by their positions
  append     kv_append, keys rotated on the way, and kv_read of what was written
  attend     kv_attention over the 4-bit cache, single tokens and prompts

in elementary torch operations (``own`` false) or by the package's kernels.

The cache is uint8 [pages, heads, page size / 16, 18 D]: tiles of 16 tokens and
D channels, in groups of 64 channels with a scale s and a minimum m, both
bfloat16, for each token; a code c stands for m + s c.  Page 0 holds nothing.
"""
import math
import random

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
GROUP = 64
TILE = 16
BASE = 1e6


def listed():
    return [
        # One request's token, 32 query heads of 128: latency.
        dict(name="rotary one token", op="rotary", tokens=1, heads=32, dim=128, turned=128, interleaved=False, scaling="none",
             first=5000, pad=0, dtype="bfloat16"),
        # A quarter of each head rotated in interleaved pairs, at positions that a scaled base makes reachable.
        dict(name="rotary part far", op="rotary", tokens=4097, heads=16, dim=256, turned=64, interleaved=True, scaling="bands",
             first=1000003, pad=0, dtype="float16"),
        # 32 prompts of 2048 tokens, the queries being columns of the input projection's output.
        dict(name="rotary prompts", op="rotary", tokens=65536, heads=32, dim=128, turned=128, interleaved=False, scaling="none",
             first=0, pad=16, dtype="bfloat16"),
        # One token of each of 256 requests.
        dict(name="append decode", op="append", seqs=256, new=256, longest=4096, heads=8, dim=128, turned=128, interleaved=False,
             page=64, dtype="bfloat16"),
        # Few wide heads, short pages, ragged prompts of odd lengths.
        dict(name="append wide heads", op="append", seqs=7, new=3001, longest=700, heads=2, dim=256, turned=64, interleaved=True,
             page=16, dtype="float16"),
        # Sixteen ragged prompts, some of which continue an earlier one.
        dict(name="append prompts", op="append", seqs=16, new=32768, longest=2048, heads=8, dim=128, turned=128, interleaved=False,
             page=64, dtype="bfloat16"),
        # One token of one request with a short context: latency.
        dict(name="attend one request", op="attend", seqs=1, new=1, longest=1000, queries=32, heads=8, dim=128, window=0, page=64,
             dtype="bfloat16"),
        # One token over one long document: the only parallel axes are the heads and the document.
        dict(name="attend long document", op="attend", seqs=1, new=1, longest=131072, queries=32, heads=8, dim=128, window=0,
             page=64, dtype="bfloat16"),
        # One token of each of 256 requests with ragged contexts: the cache's bytes count.
        dict(name="attend decode", op="attend", seqs=256, new=256, longest=8192, queries=32, heads=8, dim=128, window=0, page=64,
             dtype="bfloat16"),
        # Few wide heads, a sliding window, short pages.
        dict(name="attend window", op="attend", seqs=37, new=37, longest=20000, queries=16, heads=2, dim=256, window=4096, page=16,
             dtype="float16"),
        # Ragged prompts, each continuing a context of its own.
        dict(name="attend prompts", op="attend", seqs=8, new=8192, longest=4096, queries=32, heads=8, dim=128, window=0, page=64,
             dtype="bfloat16"),
        # The last piece of a long prompt: the tensor cores' rate counts.
        dict(name="attend long prompt", op="attend", seqs=1, new=4096, longest=12288, queries=32, heads=8, dim=128, window=0,
             page=64, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend"])
    dim = rng.choice([64, 128, 128, 256])
    turned = rng.choice([dim, dim, dim // 2, dim // 4])
    yes = lambda: rng.random() < 0.5  # noqa: E731
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    if op == "rotary":
        if yes():
            dim = 2 * _log(rng, 16, 256)
            turned = 2 * _log(rng, 8, dim // 2)
        heads = _log(rng, 1, 64)
        dtype = rng.choice([dtype, "float32"])
        most = 65536 * 32 * 128 // (heads * dim) // (2 if dtype == "float32" else 1)
        return dict(op=op, tokens=_log(rng, 1, min(65536, most)), heads=heads, dim=dim, turned=turned, interleaved=yes(),
                    scaling=rng.choice(["none", "linear", "bands"]), first=rng.choice([0, _log(rng, 1, 10 ** 7)]),
                    pad=rng.choice([0, 1, 8]), dtype=dtype)
    heads, page = _log(rng, 1, 16), rng.choice([16, 32, 64, 64, 128])
    seqs = _log(rng, 1, 256)
    if op == "append":
        new = seqs if yes() else _log(rng, seqs, max(seqs, min(32768, 32768 * 8 * 128 // (heads * dim))))
        return dict(op=op, seqs=seqs, new=new, longest=_log(rng, 1, 8192), heads=heads, dim=dim, turned=turned, interleaved=yes(),
                    page=page, dtype=dtype)
    queries = heads * rng.choice([1, 2, 4, 8, 8, 16])
    window = rng.choice([0, 0, 0, _log(rng, 16, 8192)])
    if yes():  # single tokens
        longest = _log(rng, 1, max(1, min(131072, 256 * 8192 * 8 * 128 // (seqs * heads * dim))))
        return dict(op=op, seqs=seqs, new=seqs, longest=longest, queries=queries, heads=heads, dim=dim, window=window, page=page,
                    dtype=dtype)
    seqs = _log(rng, 1, 32)
    most = 4096 * 14000 * 32 * 128 / (queries * dim)  # pairs of the longest prompt
    new = _log(rng, seqs, int(min(8192.0 if seqs == 1 else 16384.0, 0.4 * most ** 0.5)) + seqs)
    longest = _log(rng, 1, int(min(16384, most / new / 2)) + 1)
    return dict(op=op, seqs=seqs, new=new, longest=longest, queries=queries, heads=heads, dim=dim, window=window, page=page,
                dtype=dtype)


def _lengths(case):
    """(new tokens, all tokens) of each sequence.

    Single tokens: contexts from a tenth of the longest on, every 16th request padding.  Prompts: ragged,
    with one-token ones among them, each after an earlier part of up to `longest` tokens (a lone one: of just that).
    """
    seqs, new, longest = case["seqs"], case["new"], case["longest"]
    r = random.Random(new * 131 + seqs * 17 + longest)
    if new == seqs:
        total = [longest if n == 0 else 0 if n % 16 == 15 else r.randint(max(1, longest // 10), longest) for n in range(seqs)]
        return [1] * seqs, total
    cuts = sorted(r.randint(0, new - seqs) for _ in range(seqs - 1))
    count = [b - a + 1 for a, b in zip([0] + cuts, cuts + [new - seqs])]
    return count, [c + (longest if seqs == 1 else r.choice([0, r.randint(0, longest)])) for c in count]


def _frequencies(turned, scaling, device):
    """Radians a token of each pair, in 64 bits: none, all slowed down, or the slow ones only."""
    f = BASE ** (-torch.arange(0, turned, 2, dtype=torch.float64) / turned)
    if scaling == "linear":
        f = f / 8
    if scaling == "bands":
        turns = 8192 * f / (2 * math.pi)  # over the length that the model was trained on
        keep = ((turns - 1) / (4 - 1)).clamp(0, 1)
        f = f * keep + f / 8 * (1 - keep)
    return f.to(device)


def _pages(case, total, gen, dev):
    """Page table [seqs, most pages] with pages in no order, padded with 0, and the number of pages of the pool."""
    size = case["page"]
    counts = [-(-n // size) for n in total]
    pages = torch.randperm(sum(counts), generator=gen, device=dev).int() + 1
    table = torch.zeros(case["seqs"], max(1, max(counts)), dtype=torch.int32, device=dev)
    held = torch.arange(table.shape[1], device=dev) < torch.tensor(counts, device=dev)[:, None]
    table[held] = pages
    return table, sum(counts) + 1


def _ends(count, dev):
    ends = [0]
    for n in count:
        ends.append(ends[-1] + n)
    return torch.tensor(ends, dtype=torch.int32, device=dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device=dev)  # noqa: E731
    dtype, dim, heads = DTYPES[case["dtype"]], case["dim"], case["heads"]
    s = {"case": dict(case)}
    if case["op"] == "rotary":
        wide = rand(case["tokens"], (heads + case["pad"]) * dim).to(dtype)
        s["x"] = wide[:, :heads * dim].unflatten(1, (heads, dim))
        s["positions"] = torch.arange(case["tokens"], device=dev) % 2048 + case["first"]
        s["frequencies"] = _frequencies(case["turned"], case["scaling"], dev)
        return s
    count, total = _lengths(case)
    s["table"], pages = _pages(case, total, gen, dev)
    s["lengths"] = torch.tensor(total, dtype=torch.int32, device=dev)
    s["cu"] = None if case["new"] == case["seqs"] else _ends(count, dev)
    shape = (pages, heads, case["page"] // TILE, 18 * dim)
    # Keys have a few channels that are larger than the others.
    loud = torch.where(torch.rand(dim, generator=gen, device=dev) < 0.03, 4.0, 1.0)
    if case["op"] == "append":
        s["data"] = torch.zeros(shape, dtype=torch.uint8, device=dev)
        kv = rand(case["new"], 2 * heads * dim).unflatten(1, (2, heads, dim))
        kv[:, 0] *= loud
        s["k"], s["v"] = kv.to(dtype).unbind(1)
        s["frequencies"] = _frequencies(case["turned"], "none", dev)
        return s
    s["data"] = torch.empty(shape, dtype=torch.uint8, device=dev)
    rows = s["data"].permute(0, 2, 1, 3)  # [pages, tiles, heads, 18 D]
    step = max(1, 65536 * 8 * 128 // (case["page"] * heads * dim))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        tiles = n * case["page"] // TILE
        k = (rand(tiles, TILE, heads, dim) * loud).to(dtype).float()
        v = rand(tiles, TILE, heads, dim).to(dtype).float()
        rows[at:at + n] = _tile_bytes(k, v).reshape(n, case["page"] // TILE, heads, 18 * dim)
    s["q"] = (2 * rand(case["new"], case["queries"], dim)).to(dtype)
    return s


# ---------------------------------------------------------------------------
# the cache's form
# ---------------------------------------------------------------------------
# A tile: key codes, their (s, m) pairs, value codes, their pairs.  A 32-bit word holds 8 channels, even ones
# in its low half.  Token u's pairs and key codes are in row 2 (u % 4) + (u / 4) % 2 + 8 (u / 8); a key
# row's words go by (quarter t of each group, group, half of the quarter) in blocks of 128 channels, a value
# row's by (eighth of each group, group) in blocks of 32 bytes.
ROW = [(u & 8) | ((u & 3) << 1) | ((u >> 2) & 1) for u in range(TILE)]


def _down(x):
    """bfloat16 values at most x (64 bits), as floats."""
    f = x.float()
    f = torch.where(f.double() > x, torch.nextafter(f, torch.full_like(f, -math.inf)), f)
    bits = f.view(torch.int32)
    return torch.where(f < 0, bits + 0xFFFF, bits).bitwise_and(-0x10000).view(torch.float32)


def _quantize(x):
    """Codes and (s, m) of x [..., D], which is in 64 bits where the last bit can decide."""
    g = x.unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1), g.amax(-1)
    m = _down(low.double())
    s = -_down(-(high.double() - m.double()) / 15)
    c = torch.round((g - m[..., None]) / torch.where(s > 0, s, 1.0)[..., None])
    return c.to(torch.uint8).flatten(-2), s, m


def _pairs(s, m):
    """(s, m) [..., G] as bytes [..., 4 G]."""
    return torch.stack([s, m], -1).bfloat16().view(torch.uint8).flatten(-2)


def _key_words(c, dim):
    """Key codes [..., D] in the order of their nibbles."""
    per = min(dim, 128) // GROUP
    return c.unflatten(-1, (-1, per, 4, 2, 4, 2)).movedim(-4, -5).movedim(-1, -2).flatten(-6)


def _key_channels(n, dim):
    per = min(dim, 128) // GROUP
    return n.unflatten(-1, (-1, 4, per, 2, 2, 4)).movedim(-5, -4).movedim(-2, -1).flatten(-6)


def _value_words(c, dim):
    return c.unflatten(-1, (-1, 8, 4, 2)).movedim(-3, -4).movedim(-1, -2).flatten(-4)


def _value_channels(n, dim):
    return n.unflatten(-1, (8, -1, 2, 4)).movedim(-3, -4).movedim(-2, -1).flatten(-4)


def _bytes(n):
    """Bytes of nibbles, the first in the low half."""
    return n[..., 0::2] | (n[..., 1::2] << 4)


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _tile_bytes(k, v):
    """Tiles [n, heads, 18 D] of k, v [n, 16, heads, D]."""
    dim = k.shape[-1]
    place = torch.tensor(ROW, device=k.device).argsort()  # the token of each row
    (ck, sk, mk), (cv, sv, mv) = _quantize(k), _quantize(v)
    keys = _bytes(_key_words(ck[:, place], dim)).unflatten(-1, (-1, min(dim, 128) // 2))  # [n, row, heads, block, bytes]
    values = _bytes(_value_words(cv, dim)).unflatten(-1, (-1, 32))
    parts = [keys.permute(0, 2, 3, 1, 4), _pairs(sk, mk)[:, place].transpose(1, 2), values.permute(0, 2, 3, 1, 4),
             _pairs(sv, mv)[:, place].transpose(1, 2)]
    return torch.cat([p.flatten(2) for p in parts], -1)


def _tile_values(tiles, dim):
    """k, v [..., 16, heads, D] in 32 bits of tiles [..., heads, 18 D]."""
    row = torch.tensor(ROW, device=tiles.device)
    keys, kp, values, vp = tiles.split([8 * dim, dim, 8 * dim, dim], -1)

    def unpack(codes, pairs, channels, width):
        c = codes.unflatten(-1, (-1, TILE, width)).transpose(-3, -2).flatten(-2)  # [..., heads, 16, D / 2]
        sm = pairs.contiguous().view(torch.bfloat16).float().unflatten(-1, (TILE, -1, 1, 2))[..., row, :, :, :]
        c = channels(_nibbles(c), dim)
        return c, sm

    ck, pk = unpack(keys, kp, _key_channels, min(dim, 128) // 2)
    ck = ck[..., row, :]
    cv, pv = unpack(values, vp, _value_channels, 32)
    out = [(sm[..., 1] + sm[..., 0] * c.float().unflatten(-1, (-1, GROUP))).flatten(-2) for c, sm in ((ck, pk), (cv, pv))]
    return [x.movedim(-3, -2) for x in out]


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _turn(x, angle, interleaved):
    """x [T, H, D] with its first channels rotated by angle [T, R / 2] (64 bits), in x's precision."""
    turned = 2 * angle.shape[1]
    cos, sin = (f(angle).to(x.dtype)[:, None] for f in (torch.cos, torch.sin))
    a, b = (x[..., 0:turned:2], x[..., 1:turned:2]) if interleaved else x[..., :turned].chunk(2, -1)
    y = [a * cos - b * sin, a * sin + b * cos]
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat([y, x[..., turned:]], -1)


def _plain_rotary(s):
    angle = s["positions"].double()[:, None] * s["frequencies"]
    return _turn(s["x"].float(), angle, s["case"]["interleaved"]).to(s["x"].dtype)


def _places(s):
    """(sequence, position) of each new token."""
    seqs, new = s["case"]["seqs"], s["case"]["new"]
    token = torch.arange(new, device=s["table"].device)
    if s["cu"] is None:
        return token, s["lengths"].long() - 1
    ends = s["cu"].long()
    seq = torch.searchsorted(ends[1:], token, right=True)
    return seq, s["lengths"].long()[seq] - ends[seq + 1] + token


def _plain_append(s):
    case, data = s["case"], s["data"]
    dim, size = case["dim"], case["page"]
    seq, position = _places(s)
    held = position >= 0
    angle = position.double()[:, None] * s["frequencies"]
    (ck, sk, mk), (cv, sv, mv) = _quantize(_turn(s["k"].double(), angle, case["interleaved"])), _quantize(s["v"].double())
    dev = data.device
    row = torch.tensor(ROW, device=dev)
    u = position % TILE
    at = position.clamp_min(0)
    tile = (s["table"][seq, at // size].long(), slice(None), at % size // TILE)
    pairs = torch.arange(dim // 16, device=dev)
    wide = min(dim, 128) // 2
    byte = torch.arange(dim // 2, device=dev)
    parts = [(_bytes(_key_words(ck, dim)), byte // wide * TILE * wide + row[u][:, None] * wide + byte % wide),
             (_pairs(sk, mk), 8 * dim + row[u][:, None] * (dim // 16) + pairs),
             (_bytes(_value_words(cv, dim)), 9 * dim + byte // 32 * TILE * 32 + u[:, None] * 32 + byte % 32),
             (_pairs(sv, mv), 17 * dim + row[u][:, None] * (dim // 16) + pairs)]
    head = torch.arange(case["heads"], device=dev)[None, :, None]
    for value, place in parts:
        data[tile[0][held][:, None, None], head, tile[2][held][:, None, None], place[held][:, None]] = value[held]
    out = []
    for c, scale, low in ((ck, sk, mk), (cv, sv, mv)):
        x = (low[..., None] + scale[..., None] * c.float().unflatten(-1, (-1, GROUP))).flatten(-2)
        out.append(torch.where(held[:, None, None], x, 0.0).to(s["k"].dtype))
    return out


def _plain_attend(s):
    case = s["case"]
    dim, heads, seqs = case["dim"], case["heads"], case["seqs"]
    group = case["queries"] // heads
    k, v = _tile_values(s["data"][s["table"].long()].transpose(2, 3), dim)  # [seqs, pages, tiles, 16, heads, D]
    k, v = (x.flatten(1, 3).permute(0, 2, 1, 3) for x in (k, v))
    seq, position = _places(s)
    first = torch.zeros(seqs, dtype=torch.long, device=k.device) if s["cu"] is None else s["cu"][:-1].long()
    at = torch.arange(case["new"], device=k.device) - (seq if s["cu"] is None else first[seq])
    most = case["new"] // seqs if s["cu"] is None else max(_lengths(case)[0])
    q = k.new_zeros(seqs, most, case["queries"], dim)
    q[seq, at] = s["q"].float()
    limit = torch.full((seqs, most), -1, device=k.device)
    limit[seq, at] = position
    q = q.unflatten(2, (heads, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [seqs, heads, rows, D]
    score = (q @ k.transpose(-1, -2)).mul_(dim ** -0.5).unflatten(2, (most, group))
    key = torch.arange(k.shape[2], device=k.device)
    seen = key <= limit[..., None]
    if case["window"]:
        seen &= key > limit[..., None] - case["window"]
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    out = (score.flatten(2, 3) @ v).unflatten(2, (most, group)) / score.sum(-1, keepdim=True).clamp_min(1e-30)
    return out.permute(0, 2, 1, 3, 4)[seq, at].flatten(1, 2).to(s["q"].dtype)


_PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend}


# ---------------------------------------------------------------------------
# the package's operators
# ---------------------------------------------------------------------------
def _own_rotary(s):
    from stepquant_b200.kernels.rotary import rotary
    return rotary(s["x"], s["positions"], s["frequencies"], interleaved=s["case"]["interleaved"])


def _own_append(s):
    from stepquant_b200.kernels.kv_cache import kv_append, kv_read
    kv_append(s["data"], s["k"], s["v"], s["table"], s["lengths"], cu_seqlens=s["cu"], frequencies=s["frequencies"],
              interleaved=s["case"]["interleaved"])
    return kv_read(s["data"], s["table"], s["lengths"], cu_seqlens=s["cu"], tokens=s["case"]["new"], dtype=s["k"].dtype)


def _own_attend(s):
    from stepquant_b200.kernels.kv_cache import kv_attention
    return kv_attention(s["q"], s["data"], s["table"], s["lengths"], cu_seqlens=s["cu"], window=s["case"]["window"] or None)


_OWN = {"rotary": _own_rotary, "append": _own_append, "attend": _own_attend}


def run(state):
    out = (_OWN if own else _PLAIN)[state["case"]["op"]](state)
    return list(out) if isinstance(out, (tuple, list)) else [out]


# ---------------------------------------------------------------------------
# floors and 64-bit values
# ---------------------------------------------------------------------------
def work(case):
    size, dim, heads = DTYPES[case["dtype"]].itemsize, case["dim"], case["heads"]
    if case["op"] == "rotary":
        values = case["tokens"] * heads * dim
        return {"bytes": 2 * values * size + 8 * case["tokens"], "flops": 3 * case["tokens"] * heads * case["turned"]}
    token = heads * 18 * dim // TILE  # bytes of a token's keys and values
    count, total = _lengths(case)
    if case["op"] == "append":
        values = 2 * case["new"] * heads * dim
        return {"bytes": 2 * values * size + 2 * case["new"] * token, "flops": 12 * values}
    window, group = case["window"], case["queries"] // heads
    read = pairs = 0
    for c, n in zip(count, total):
        start = max(0, n - c + 1 - window) if window else 0
        read += n - min(n, start)
        for a, b in ((n - c, n),) if n >= c else ():
            full = b * (b + 1) // 2 - a * (a + 1) // 2  # a query at position p sees p + 1 keys
            if window:
                far = max(a, window)
                full -= sum(p + 1 - window for p in (far, b - 1)) * (b - far) // 2 if b > far else 0
            pairs += full
    return {"bytes": read * token + 2 * case["new"] * case["queries"] * dim * size, "flops": 4 * pairs * heads * group * dim}


def _exact_turn(x, position, f, interleaved):
    turned = 2 * f.numel()
    phase = torch.remainder(position.double()[:, None] * f, 2 * math.pi)
    z = torch.polar(torch.ones_like(phase), phase)[:, None]
    y = x.double().clone()
    even, odd = ([2 * i for i in range(turned // 2)], [2 * i + 1 for i in range(turned // 2)]) if interleaved else (
        list(range(turned // 2)), list(range(turned // 2, turned)))
    w = torch.complex(y[..., even], y[..., odd]) * z
    y[..., even], y[..., odd] = w.real, w.imag
    return y


def _exact_value(x):
    """What the codes of x [..., D] stand for."""
    y = torch.empty_like(x)
    for g in range(0, x.shape[-1], GROUP):
        part = x[..., g:g + GROUP]
        low, high = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
        m = _exact_border(low, -1)
        s = _exact_border((high - m) / 15, 1)
        y[..., g:g + GROUP] = m + s * torch.round((part - m) / torch.where(s == 0, 1.0, s))
    return y


def _exact_border(x, side):
    """The nearest value of 8 significant bits that is not on the other side of x."""
    mantissa, exponent = torch.frexp(x)
    unit = torch.ldexp(torch.ones_like(x), (exponent - 8).clamp_min(-133))
    return (torch.floor(x / unit) if side < 0 else torch.ceil(x / unit)) * unit


def _exact_places(s):
    count, total = _lengths(s["case"])
    return [(n, t - c + i) for n, (c, t) in enumerate(zip(count, total)) for i in range(c)]


def _exact_append(s):
    position = torch.tensor([p for _, p in _exact_places(s)], device=s["k"].device)
    k = _exact_value(_exact_turn(s["k"], position, s["frequencies"], s["case"]["interleaved"]))
    return [torch.where((position >= 0)[:, None, None], x, 0.0) for x in (k, _exact_value(s["v"].double()))]


def _exact_cached(tiles, dim, keys):
    """Keys or values [16 n, D] in 64 bits of one head's tiles [n, 18 D], by where each channel of a token lies."""
    byte, shift, pair = [], [], []
    for u in range(TILE):
        row = 2 * (u % 4) + u // 4 % 2 + u // 8 * 8
        for c in range(dim):
            group, rest = divmod(c, GROUP)
            nibble = rest % 8 // 2 + 4 * (rest % 2)
            if keys:
                per = min(dim, 128) // GROUP
                word = rest // 16 * 2 * per + group % per * 2 + rest % 16 // 8
                at = group // per * TILE * per * 32 + row * per * 32 + 4 * word
            else:
                word = rest // 8 * (dim // GROUP) + group
                at = 9 * dim + word // 8 * TILE * 32 + u * 32 + word % 8 * 4
            byte.append(at + nibble // 2)
            shift.append(4 * (nibble % 2))
            pair.append((8 if keys else 17) * dim + (row * (dim // GROUP) + group) * 4)
    byte, shift, pair = (torch.tensor(x, device=tiles.device) for x in (byte, shift, pair))
    code = (tiles[:, byte].int() >> shift) & 15

    def wide(at):  # the bfloat16 at a byte offset
        bits = (tiles[:, at].int() << 16) | (tiles[:, at + 1].int() << 24)
        return bits.view(torch.float32).double()

    return (wide(pair + 2) + wide(pair) * code.double()).reshape(-1, dim)


def _exact_attend(s):
    case, q = s["case"], s["q"].double()
    dim, heads, group = case["dim"], case["heads"], case["queries"] // case["heads"]
    out = torch.zeros_like(q)
    count, total = _lengths(case)
    tiles = case["page"] // TILE
    begin = 0
    for n, (c, t) in enumerate(zip(count, total)):
        pages = s["table"][n, :-(-t // case["page"])].long()
        limit = torch.arange(t - c, t, device=q.device)[:, None]
        for h in range(heads if t else 0):
            held = s["data"][pages, h].reshape(len(pages) * tiles, -1)[:-(-t // TILE)]
            k, v = _exact_cached(held, dim, True)[:t], _exact_cached(held, dim, False)[:t]
            key = torch.arange(t, device=q.device)[None]
            hidden = (key > limit) | ((key <= limit - case["window"]) if case["window"] else (key < 0))
            for head in range(h * group, (h + 1) * group):
                score = q[begin:begin + c, head] @ k.T / math.sqrt(dim)
                score[hidden] = -math.inf
                out[begin:begin + c, head] = torch.softmax(score, -1) @ v
        begin += c
    return [torch.nan_to_num(out)]


def exact(case, seed):
    """run()'s outputs from the definitions in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return [_exact_turn(s["x"], s["positions"], s["frequencies"], case["interleaved"])]
    return _exact_append(s) if case["op"] == "append" else _exact_attend(s)
