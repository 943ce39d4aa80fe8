"""The 4-bit cache and attention over it in 64 bits, for tests: values by their
definition, and where a tile's bytes lie by the C header's description."""
import math

import torch

GROUP, TILE = 64, 16


def border(x, up):
    """bfloat16 next to x (64 bits) at or below it, or at or above."""
    mantissa, exponent = torch.frexp(x)
    unit = torch.ldexp(torch.ones_like(x), (exponent - 8).clamp_min(-133))
    return (torch.ceil if up else torch.floor)(x / unit) * unit


def turn(x, positions, frequencies, interleaved=False, magnitude=1.0, inverse=False):
    """x [T, H, D] with its first channels rotated, in 64 bits."""
    y = x.double().clone()
    n = frequencies.numel()
    a = positions.double()[:, None] * frequencies.double()
    cos, sin = magnitude * a.cos()[:, None], (-magnitude if inverse else magnitude) * a.sin()[:, None]
    one, two = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    u, v = y[..., one].clone(), y[..., two].clone()
    y[..., one], y[..., two] = u * cos - v * sin, u * sin + v * cos
    return y


def quantize(x):
    """(codes, s, m) of x [..., D] in 64 bits: [..., G, 64], [..., G, 1] twice; m is NaN where a value is not finite."""
    x = x.double().unflatten(-1, (-1, GROUP))
    bad = ~torch.isfinite(x).all(-1, keepdim=True) | (x.abs() > 3.3895313892515355e38).any(-1, keepdim=True)
    x = torch.where(bad, 0.0, x)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    m = border(low, False)
    s = border((high - m) / 15, True)
    c = torch.round((x - m) / torch.where(s == 0, 1.0, s))
    return c, torch.where(bad, math.nan, s), torch.where(bad, math.nan, m)


def value(x):
    """What the codes of x stand for."""
    c, s, m = quantize(x)
    return (m + s * c).flatten(-2)


def tile_places(dim):
    """byte and shift of each (token, channel)'s code, and byte of its pair, for keys and for values: [2][16, D]."""
    out = []
    for values in (False, True):
        byte, shift, pair = (torch.zeros(TILE, dim, dtype=torch.long) for _ in range(3))
        for u in range(TILE):
            r = 2 * (u % 4) + u // 4 % 2 + u // 8 * 8
            for c in range(dim):
                group, i, e = c // 64, c % 64 // 8, c % 8
                if values:
                    w = dim // 64 * i + group
                    word = 9 * dim + ((w // 8 * 16 + u) * 8 + w % 8) * 4
                else:
                    n = min(2, dim // 64)
                    word = ((group // n * 16 + r) * 8 * n + 2 * n * (i // 2) + 2 * (group % n) + i % 2) * 4
                bit = 2 * e if e % 2 == 0 else 14 + 2 * e
                byte[u, c], shift[u, c] = word + bit // 8, bit % 8
                pair[u, c] = (17 * dim if values else 8 * dim) + (r * (dim // 64) + group) * 4
        out.append((byte, shift, pair))
    return out


def unpack(tiles, dim, parts=False):
    """(k, v) [..., 16, D] in 64 bits of tiles [..., 18 D]; with parts, and sizes |m + 8 s| + s (|c - 8| + 2^-8) of v's."""
    out = []
    for byte, shift, pair in tile_places(dim):
        byte, shift, pair = (x.to(tiles.device) for x in (byte, shift, pair))
        c = (tiles[..., byte].int() >> shift) & 15
        word = lambda at: ((tiles[..., at].int() << 16) | (tiles[..., at + 1].int() << 24)).view(torch.float32).double()  # noqa: E731
        out.append(word(pair + 2) + word(pair) * c)
    return [*out, (word(pair + 2) + 8 * word(pair)).abs() + word(pair) * ((c - 8).abs() + 2.0 ** -8)] if parts else out


def cached(data, pages, page_size, length):
    """(k, v, sizes of v's parts) [H, length, D] of a sequence from the pool's bytes."""
    dim = data.shape[3] // 18
    held = data[torch.as_tensor(pages[:-(-length // page_size)], device=data.device).long()]  # [pages, H, tiles, 18 D]
    return [x.transpose(0, 1).flatten(1, 3)[:, :length] for x in unpack(held, dim, parts=True)]


def attend(q, k, v, sizes, before, scale, window=None, hidden=None):
    """(out, weighted sum of sizes) [c, Hq, D] in 64 bits: q of the tokens at positions before + i, k, v [H, L, D].
    hidden: positions that hold nothing."""
    c, q_heads, dim = q.shape
    heads, length, _ = k.shape
    q = q.double().unflatten(1, (heads, -1)).permute(1, 2, 0, 3)  # [H, G, c, D]
    score = scale * q @ k[:, None].transpose(-1, -2)
    j, p = torch.arange(length, device=q.device), before + torch.arange(c, device=q.device)[:, None]
    seen = j <= p
    if window is not None:
        seen &= j > p - window
    if hidden is not None:
        seen &= ~hidden
    score = score.masked_fill(~seen, -math.inf)
    some = seen.any(-1)[:, None]
    w = torch.where(seen, torch.exp(score - torch.where(some, score.amax(-1, keepdim=True), 0.0)), 0.0)
    w = torch.where(some, w / w.sum(-1, keepdim=True), 0.0)
    clean = lambda x: torch.where(seen.any(0)[:, None], x, 0.0)[:, None]  # noqa: E731
    back = lambda x: x.permute(2, 0, 1, 3).flatten(1, 2)  # noqa: E731
    return back(w @ clean(v)), back(w @ clean(sizes))
