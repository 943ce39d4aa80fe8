"""Short causal convolution of recurrent layers (csrc/sq_conv.cu).

``causal_conv1d``       concatenated prompts, keyword names of
                        ``prefill.chunk_gated_delta_rule``.
``causal_conv1d_step``  one token of each request, the state updated in place.

y[t, d] = act(bias[d] + sum_j weight[d, j] x[t - W + 1 + j, d]) with W = 2 to 4
taps.  A state row [channels, W - 1] holds the inputs before the next token,
oldest first, in x's dtype.  Asynchronous on the current stream.
"""
import torch

from .. import _native as N

_pack = N.packer(N.SqConvArgs)


def sequence_ends(cu_seqlens, tokens, device):
    """int32 boundaries on ``device`` (default: one sequence of all tokens, written
    there: a copy from the host could not be captured)."""
    if cu_seqlens is None:
        return torch.arange(0, 2 * tokens, tokens, dtype=torch.int32, device=device) if tokens else torch.zeros(
            2, dtype=torch.int32, device=device)
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError("cu_seqlens: expected [sequences + 1]")
    if cu_seqlens.dtype == torch.int32 and cu_seqlens.device == device and cu_seqlens.is_contiguous():
        return cu_seqlens
    return cu_seqlens.to(device=device, dtype=torch.int32).contiguous()


def slot_rows(slots, count, device):
    """int64 state rows of ``count`` requests, or None."""
    if slots is None:
        return None
    if slots.shape != (count,):
        raise ValueError(f"slots: expected [{count}]")
    return slots if slots.dtype == torch.int64 and slots.device == device and slots.stride(0) == 1 else slots.to(device=device, dtype=torch.int64).contiguous()


def _filter(weight, bias, channels):
    if weight.dim() == 3 and weight.shape[1] == 1:
        weight = weight[:, 0]
    if weight.dim() != 2 or weight.shape[0] != channels:
        raise ValueError(f"weight: expected [{channels}, taps]")
    if not 2 <= weight.shape[1] <= 4:
        raise NotImplementedError("the convolution is built for 2 to 4 taps")
    if bias is not None and bias.shape != (channels,):
        raise ValueError(f"bias: expected [{channels}]")
    return weight.float().contiguous(), None if bias is None else bias.float().contiguous()


def _activation(name):
    if name not in (None, "silu"):
        raise ValueError("activation: expected 'silu' or None")
    return 1 if name == "silu" else 0


def _state(state, rows, channels, taps, dtype, name):
    if state.dim() != 3 or state.shape[1:] != (channels, taps - 1) or (rows is not None and state.shape[0] != rows):
        raise ValueError(f"{name}: expected [{'rows' if rows is None else rows}, {channels}, {taps - 1}]")
    if state.dtype != dtype:
        raise ValueError(f"{name}: expected dtype {dtype}, got {state.dtype}")
    return state


def _launch(entry, rows, y, weight, bias, initial, final, slots, cu, status, seqs, activation, index):
    p = N.address
    N.launch(entry, _pack(p(rows), p(weight), p(bias), p(y), p(initial), p(final), p(slots), p(cu), p(status),
                          rows.stride(0), 0 if final is None else final.shape[0], rows.shape[0], seqs, rows.shape[1],
                          weight.shape[1], N.dtype_code(rows.dtype), activation), index)


def outputs(x, seqs):
    """y of concatenated sequences; without any there is no launch that writes its zeros."""
    return x.new_empty(x.shape) if seqs else x.new_zeros(x.shape)


def _token_rows(x):
    """[tokens, channels] of concatenated sequences."""
    if x.dim() == 3 and x.shape[0] != 1:
        raise ValueError("x: expected a leading batch of 1 (concatenated sequences)")
    if x.dim() not in (2, 3) or x.shape[-1] < 1:
        raise ValueError("x: expected [tokens, channels]")
    return N.rows_of(x, "x")


def causal_conv1d(x, weight, bias=None, *, initial_state=None, output_final_state=True, activation="silu",
                  cu_seqlens=None):
    """Convolution of concatenated sequences: (y, final_state).

    x: [T, D] or [1, T, D] float32, bfloat16 or float16, rows any stride apart;
    weight: [D, W] (or [D, 1, W]), bias: [D], both used in fp32; cu_seqlens:
    [N + 1] boundaries (default: one sequence); initial_state: [N, D, W - 1] in
    x's dtype, or None (zeros).  y has x's shape and dtype, zero for tokens of no
    sequence; final_state [N, D, W - 1] or None when ``output_final_state`` is false.
    """
    rows = _token_rows(x)
    tokens, channels = rows.shape
    weight, bias = _filter(weight, bias, channels)
    activation = _activation(activation)
    index = N.device_index(x, weight, bias, initial_state)
    cu = sequence_ends(cu_seqlens, tokens, x.device)
    seqs, taps = cu.numel() - 1, weight.shape[1]
    if initial_state is not None:
        initial_state = _state(initial_state, seqs, channels, taps, x.dtype, "initial_state").contiguous()
    final = x.new_empty((seqs, channels, taps - 1)) if output_final_state else None
    y = outputs(x, seqs)
    _launch(N.lib().sq_causal_conv, rows, y, weight, bias, initial_state, final, None, cu, None, seqs, activation, index)
    return y, final


def causal_conv1d_extend(x, state, weight, bias=None, *, slots, cu_seqlens=None, activation="silu", status=None):
    """``causal_conv1d`` on a pool of states [S, D, W - 1]: sequence n continues
    from, and updates in place, row slots[n].  A slot <= 0 (padding) or outside
    the pool (flagged in ``status``, an int32 word) gives zero outputs."""
    if slots is None:
        raise ValueError("slots: required, the pool's row of each sequence")
    rows = _token_rows(x)
    tokens, channels = rows.shape
    weight, bias = _filter(weight, bias, channels)
    activation = _activation(activation)
    index = N.device_index(x, weight, bias, state, N.status_word(status))
    cu = sequence_ends(cu_seqlens, tokens, x.device)
    seqs = cu.numel() - 1
    state = _pool_state(state, channels, weight.shape[1], x.dtype)
    y = outputs(x, seqs)
    _launch(N.lib().sq_causal_conv, rows, y, weight, bias, state, state, slot_rows(slots, seqs, x.device), cu, status, seqs,
            activation, index)
    return y


def _pool_state(state, channels, taps, dtype):
    _state(state, None, channels, taps, dtype, "state")
    if not state.is_contiguous():
        raise ValueError("state: updated in place, expected a contiguous tensor")
    return state


def causal_conv1d_step(x, state, weight, bias=None, *, slots=None, activation="silu", status=None):
    """One token of each request: x [B, D] -> y [B, D]; ``state`` [S, D, W - 1]
    (x's dtype, contiguous) is updated in place at rows ``slots`` [B] (None: row
    i for request i, S = B).  Slots are distinct; padding and slots outside the
    pool as in ``causal_conv1d_extend``."""
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError("x: expected [batch, channels]")
    rows = N.rows_of(x, "x")
    batch, channels = rows.shape
    weight, bias = _filter(weight, bias, channels)
    activation = _activation(activation)
    index = N.device_index(x, weight, bias, state, N.status_word(status))
    state = _pool_state(state, channels, weight.shape[1], x.dtype)
    if slots is None and state.shape[0] != batch:
        raise ValueError(f"state: expected {batch} rows without slots")
    y = x.new_empty((batch, channels))
    _launch(N.lib().sq_causal_conv_step, rows, y, weight, bias, None, state, slot_rows(slots, batch, x.device), None, status,
            batch, activation, index)
    return y
