"""Paged cache of keys and values in 4 bits, and attention over it (csrc/sq_kv.cu, sq_attention.cu).

``kv_append``         keys, rotated on the way, and values of new tokens into their pages.
``kv_attention``      the new tokens' queries over their sequences: prompts, or one token each.
``kv_read``           the values that the new tokens' codes stand for.
``QuantizedKVPool``   the pages that an attention layer keeps, with these as methods.

For each token, kv head and group of 64 channels x: minimum m = min x rounded
down to bfloat16, scale s = (max x - m) / 15 rounded up to bfloat16, codes
c = rint((x - m) / s); c stands for m + s c, no further than s / 2 from x: 4.5
bits a channel.  ``data`` is uint8 [pages, heads, page size / 16, 18 D], tiles of
16 tokens whose bytes include/stepquant_b200.h describes.

Sequence n holds lengths[n] tokens, position p in page page_table[n][p // page
size].  Its new tokens, those of [cu_seqlens[n], cu_seqlens[n + 1]) or just one,
are the last of them.  A page <= 0 holds nothing (padding; a window's freed
pages): nothing is written there or attended to, and zeros are read.  The same
goes for positions past the table and pages past the pool, which set a bit in
``status``.  Asynchronous on the current stream.
"""
import functools

import torch

from .. import _native as N
from .rotary import MOST_FLOAT, check_magnitude, checked_frequencies, checked_positions

HEAD_DIMS = (64, 128, 256)
TILE = 16

_pack = N.packer(N.SqKvArgs)
_pack_attention = N.packer(N.SqKvAttentionArgs)


_WIDTHS = {18 * d: d for d in HEAD_DIMS}


def _int32(x, index, device):
    """int32 tensor with a contiguous last axis on ``device``; what int32 does not hold becomes its ends, and so stays outside."""
    if x.dtype is torch.int32 and x.get_device() == index and (x.stride(-1) == 1 or x.shape[-1] < 2):
        return x
    if x.dtype is torch.int64:
        x = x.clamp(-2 ** 31, 2 ** 31 - 1)
    return x.to(device=device, dtype=torch.int32).contiguous()


class _Call:
    """Checked pool and sequences of one call."""

    __slots__ = ("data", "table", "lengths", "cu", "seqs", "width", "dim", "heads", "pages", "page_size", "index")

    def __init__(self, data, page_table, lengths, cu_seqlens, tokens):
        shape = data.shape
        if len(shape) != 4 or data.dtype is not torch.uint8 or shape[3] not in _WIDTHS or not data.is_contiguous():
            raise ValueError("data: expected contiguous uint8 [pages, heads, page size / 16, 18 D] with D in (64, 128, 256), got "
                             f"{data.dtype} {list(shape)}")
        self.pages, self.heads, tiles, width = shape
        if data.data_ptr() % 16 or self.heads < 1 or tiles < 1:
            raise ValueError("data: expected a 16-byte aligned pool of at least one head and one tile a page")
        self.data, self.page_size, self.dim, self.index = data, TILE * tiles, _WIDTHS[width], data.get_device()
        device = data.device
        if lengths.dim() != 1:
            raise ValueError(f"lengths: expected [sequences], got {list(lengths.shape)}")
        self.lengths, self.seqs = _int32(lengths, self.index, device), lengths.shape[0]
        rows = page_table.shape
        if len(rows) != 2 or rows[0] != self.seqs:
            raise ValueError(f"page_table: expected [{self.seqs}, pages], got {list(rows)}")
        self.table, self.width = _int32(page_table, self.index, device), rows[1]
        if cu_seqlens is None:
            if tokens != self.seqs:
                raise ValueError(f"expected one token of each of {self.seqs} sequences without cu_seqlens, got {tokens}")
            self.cu = None
        elif cu_seqlens.shape != (self.seqs + 1,):
            raise ValueError(f"cu_seqlens: expected [{self.seqs + 1}], got {list(cu_seqlens.shape)}")
        else:
            self.cu = _int32(cu_seqlens, self.index, device)


def _rows(x, shape, dtype, name):
    if x.shape != shape or x.dtype is not dtype:
        raise ValueError(f"{name}: expected {dtype} {list(shape)}, got {x.dtype} {list(x.shape)}")
    return x if x.stride(2) == 1 else x.contiguous()


def _launch(entry, call, k, v, frequencies, positions, interleaved, magnitude, status):
    p, table, (ks, kh, _), (vs, vh, _) = N.address, call.table, k.stride(), v.stride()
    index = N.device_index(call.data, k, v, frequencies, positions, N.status_word(status))
    N.launch(entry, _pack(k.data_ptr(), v.data_ptr(), call.data.data_ptr(), table.data_ptr(), call.lengths.data_ptr(), p(call.cu),
                          p(positions), p(frequencies), p(status), ks, kh, vs, vh, table.stride(0), call.pages, k.shape[0], call.seqs,
                          call.width, call.heads, call.dim, call.page_size, N.dtype_code(k.dtype),
                          0 if frequencies is None else 2 * frequencies.numel(),
                          positions is not None and positions.dtype is torch.int64, bool(interleaved), magnitude), index)


def kv_append(data, k, v, page_table, lengths, *, cu_seqlens=None, frequencies=None, interleaved=False, magnitude=1.0,
              positions=None, status=None):
    """Write k and v [T, H, D] of the new tokens into their pages.

    data: the pool, updated in place; k, v: float32, bfloat16 or float16, alike,
    tokens and heads any stride apart; page_table: [S, pages] and lengths: [S],
    the new tokens counted, int32 (others are converted on every call);
    cu_seqlens: [S + 1] boundaries of the sequences' new tokens, None for one
    each (T = S).  No two new tokens share a place: pages that sequences have in
    common hold earlier tokens.  With ``frequencies`` keys are rotated as by ``rotary.rotary``,
    by ``positions`` [T] or their position in the sequence, and quantized without
    a rounding between.
    """
    if k.dim() != 3:
        raise ValueError("k: expected [tokens, heads, dim]")
    call = _Call(data, page_table, lengths, cu_seqlens, k.shape[0])
    N.dtype_code(k.dtype)
    shape = (k.shape[0], call.heads, call.dim)
    k = _rows(k, shape, k.dtype, "k")
    v = _rows(v, shape, k.dtype, "v")
    frequencies = checked_frequencies(frequencies, call.dim)
    if positions is not None:
        positions = checked_positions(positions, k.shape[0])
    check_magnitude(magnitude)
    _launch(N.lib().sq_kv_append, call, k, v, frequencies, positions, interleaved, magnitude, status)


def kv_read(data, page_table, lengths, *, cu_seqlens=None, tokens=None, dtype=torch.bfloat16, status=None):
    """(k, v), [T, H, D] in ``dtype``: what the new tokens' codes stand for,
    addressed as in ``kv_append``; zeros where nothing is held.  ``tokens`` is T,
    needed with cu_seqlens (which stays on the device)."""
    if tokens is None:
        if cu_seqlens is not None:
            raise ValueError("tokens: required with cu_seqlens")
        tokens = lengths.numel()
    if tokens < 0:
        raise ValueError("tokens must not be negative")
    call = _Call(data, page_table, lengths, cu_seqlens, tokens)
    N.dtype_code(dtype)
    k, v = data.new_empty((2, tokens, call.heads, call.dim), dtype=dtype).unbind(0)
    _launch(N.lib().sq_kv_read, call, k, v, None, None, False, 1.0, status)
    return k, v


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*sizes):
    return N.lib().sq_kv_attention_workspace_bytes(*sizes)


def kv_attention(q, data, page_table, lengths, *, cu_seqlens=None, scale=None, window=None, status=None):
    """Softmax attention of the new tokens over their sequences: [T, Hq, D] like q.

    q: [T, Hq, D] bfloat16 or float16, Hq a multiple of the pool's heads, tokens and
    heads any stride apart; data, page_table, lengths, cu_seqlens as in
    ``kv_append``, which comes first: a token sees its sequence up to itself and,
    with ``window``, the last ``window`` positions of that.  scale: D^-1/2.  A
    token that sees nothing, and tokens of no sequence, get zeros.  In sequences of
    more than 32 rows (new tokens times query heads of a kv head) weights below 2^-32
    of a row's largest count for nothing.  Should a bounded
    device wait give up, outputs left undone are NaN and ``status`` has SQ_STATUS_TIMEOUT.
    """
    if q.dim() != 3:
        raise ValueError("q: expected [tokens, heads, dim]")
    tokens, q_heads, dim = q.shape
    call = _Call(data, page_table, lengths, cu_seqlens, tokens)
    if q.dtype is not torch.bfloat16 and q.dtype is not torch.float16:
        raise NotImplementedError(f"attention is built for bfloat16 and float16 queries, got {q.dtype}")
    if dim != call.dim or q_heads < 1 or q_heads % call.heads:
        raise ValueError(f"q: expected [{tokens}, a multiple of {call.heads}, {call.dim}], got {list(q.shape)}")
    if scale is None:
        scale = dim ** -0.5
    if not 0 < scale <= MOST_FLOAT:
        raise ValueError("scale must be above zero and finite")
    if window is not None and window < 1:
        raise ValueError("window must be at least 1")
    index = N.device_index(data, q, N.status_word(status))
    (rows, heads, last), table = q.stride(), call.table
    # The stride of an axis of one is nobody's (contiguous() leaves it too).
    rows, heads = rows if tokens > 1 else 0, heads if q_heads > 1 else 0
    if last != 1 or rows % 8 or heads % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        rows, heads, _ = q.stride()
    out = data.new_empty((tokens, q_heads, dim), dtype=q.dtype)
    if not call.seqs:
        return out.zero_()
    p, size = N.address, _workspace_bytes(tokens, call.seqs, q_heads, call.heads, dim)
    workspace = data.new_empty(size) if size > 0 else None
    N.launch(N.lib().sq_kv_attention, _pack_attention(
        q.data_ptr(), data.data_ptr(), out.data_ptr(), table.data_ptr(), call.lengths.data_ptr(), p(call.cu), p(status), p(workspace),
        size, rows, heads, table.stride(0), call.pages, tokens, call.seqs, call.width, q_heads, call.heads, dim,
        call.page_size, N.dtype_code(q.dtype), 0 if window is None else min(window, 2 ** 31 - 1), scale, 0), index)
    return out


class QuantizedKVPool:
    """The pages of an attention layer: ``data``, uint8 [pages, heads, page_size / 16,
    18 head_dim], zeroed.  Page 0 is the padding sentinel."""

    def __init__(self, pages, heads, head_dim, page_size=64, device="cuda"):
        if pages < 1 or heads < 1 or page_size < TILE or page_size % TILE:
            raise ValueError(f"invalid cache: {pages} pages of {page_size} tokens, {heads} heads (page sizes are multiples of {TILE})")
        if head_dim not in HEAD_DIMS:
            raise NotImplementedError(f"the cache is built for heads of {HEAD_DIMS} channels, got {head_dim}")
        self.heads, self.head_dim, self.page_size = heads, head_dim, page_size
        self.data = torch.zeros(pages, heads, page_size // TILE, 18 * head_dim, device=device, dtype=torch.uint8)
        self.status = torch.zeros(1, device=device, dtype=torch.int32)

    def append(self, k, v, page_table, lengths, **options):
        kv_append(self.data, k, v, page_table, lengths, status=self.status, **options)

    def read(self, page_table, lengths, **options):
        return kv_read(self.data, page_table, lengths, status=self.status, **options)

    def attend(self, q, page_table, lengths, **options):
        return kv_attention(q, self.data, page_table, lengths, status=self.status, **options)

    def clear(self, pages):
        self.data[pages] = 0

    def copy(self, source, destination):
        self.data[destination] = self.data[source]

    def check_status(self):
        """Raise if a kernel met a page or position outside the pool or table, or gave up waiting (synchronizes)."""
        value = int(self.status.item())
        if value:
            self.status.zero_()
        if value & N.SQ_STATUS_TIMEOUT:
            raise RuntimeError("a bounded device wait of the attention gave up; its outputs are NaN")
        if value & N.SQ_STATUS_SLOT_RANGE:
            raise IndexError("a page was outside the pool, or a position past its page table; those tokens were skipped")
