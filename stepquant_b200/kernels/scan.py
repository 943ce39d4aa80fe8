"""Selective state space scan (csrc/sq_scan.cu) and its pool of request states.

``selective_scan``       concatenated prompts, keyword names of
                         ``prefill.chunk_gated_delta_rule``.
``selective_scan_step``  one token of each request, the state updated in place.
``SelectiveStatePool``   the states a selective layer keeps per request slot, its
                         convolution's and its scan's, with the ``extend`` /
                         ``step`` / ``clear`` / ``copy`` of ``PackedStatePool``.

For channel d of group g and state n:

    dt' = softplus(dt + dt_bias);  h[d, n] <- exp(dt' a[d, n]) h[d, n] + dt' u b[g, n]
    y[d] = (sum_n c[g, n] h[d, n] + d[d] u) silu(z)

States are fp32.  Asynchronous on the current stream.
"""
import torch

from .. import _native as N
from .conv import causal_conv1d_extend, causal_conv1d_step, outputs, sequence_ends, slot_rows

STATES = (4, 8, 16, 32, 64)


_pack = N.packer(N.SqScanArgs)


def _token_groups(x, tokens, states, dtype, name):
    """b or c as [tokens, groups, states] with a token's groups contiguous."""
    shape = x.shape
    if len(shape) != 3 or shape[0] != tokens:
        if len(shape) == 2:  # one group
            x = x.unsqueeze(1)
        elif len(shape) == 4 and shape[0] == 1:
            x = x[0]
        elif len(shape) == 3 and shape[0] == 1 and shape[1] == tokens:  # a leading batch of 1, one group
            x = x[0].unsqueeze(1)
        shape = x.shape
    if len(shape) != 3 or shape[0] != tokens or shape[2] != states or x.dtype != dtype:
        raise ValueError(f"{name}: expected {dtype} [{tokens}, groups, {states}]")
    stride = x.stride()
    return x if stride[2] == 1 and (shape[1] == 1 or stride[1] == states) else x.contiguous()


def _row_input(x, u, name):
    if x.shape != u.shape or x.dtype != u.dtype:
        raise ValueError(f"{name}: expected u's shape and dtype")
    return N.rows_of(x, name)


def _channel_vector(x, channels, name):
    if x is None:
        return None
    if x.shape != (channels,):
        raise ValueError(f"{name}: expected [{channels}]")
    return x if x.dtype == torch.float32 and x.is_contiguous() else x.float().contiguous()


class _Call:
    """Checked operands of one call, and the launch of an entry point on them."""

    __slots__ = ("tokens", "channels", "states", "groups", "index", "kept", "pointers", "strides", "tail")

    def __init__(self, u, dt, a, b, c, d, z, dt_bias, softplus):
        rows = N.rows_of(u, "u")
        tokens, channels = rows.shape
        if a.dim() != 2 or a.shape[0] != channels or a.dtype != torch.float32:
            raise ValueError(f"a: expected float32 [{channels}, states]")
        states = a.shape[1]
        if states not in STATES:
            raise NotImplementedError(f"the scan is built for {STATES} states, got {states}")
        a, dtype = N.aligned(a), u.dtype
        dt = _row_input(dt, u, "dt")
        z = None if z is None else _row_input(z, u, "z")
        b, c = _token_groups(b, tokens, states, dtype, "b"), _token_groups(c, tokens, states, dtype, "c")
        groups = b.shape[1]
        if c.shape[1] != groups or groups < 1 or channels < 1 or channels % groups:
            raise ValueError("b and c need the same groups, a divisor of the channels")
        d, dt_bias = _channel_vector(d, channels, "d"), _channel_vector(dt_bias, channels, "dt_bias")
        self.index = N.device_index(rows, a, dt, z, b, c, d, dt_bias)
        self.tokens, self.channels, self.states, self.groups = tokens, channels, states, groups
        p = N.address
        self.kept = (rows, dt, z, b, c, a, d, dt_bias)  # copies made above live until the launch
        self.pointers = (rows.data_ptr(), dt.data_ptr(), p(z), b.data_ptr(), c.data_ptr(), a.data_ptr(), p(d), p(dt_bias))
        self.strides = (rows.stride(0), dt.stride(0), 0 if z is None else z.stride(0), b.stride(0), c.stride(0))
        self.tail = (channels, states, groups, N.dtype_code(dtype), bool(softplus))

    def launch(self, entry, y, initial, final, slots, cu, status, workspace, seqs):
        p = N.address
        N.launch(entry, _pack(*self.pointers, y.data_ptr(), p(initial), p(final), p(slots), p(cu), p(status), p(workspace),
                              0 if workspace is None else workspace.numel(), *self.strides,
                              0 if final is None else final.shape[0], self.tokens, seqs, *self.tail), self.index)


def _state(state, rows, channels, states, name):
    if state.dim() != 3 or state.shape[1:] != (channels, states) or (rows is not None and state.shape[0] != rows):
        raise ValueError(f"{name}: expected [{'rows' if rows is None else rows}, {channels}, {states}]")
    if state.dtype != torch.float32:
        raise ValueError(f"{name}: expected float32, got {state.dtype}")
    return state


def _pool_state(state, channels, states):
    _state(state, None, channels, states, "state")
    if not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError("state: updated in place, expected a contiguous, 16-byte aligned tensor")
    return state


def _prompts(u, dt, a, b, c, d, z, dt_bias, dt_softplus, cu_seqlens, initial, final, slots, status):
    """The scan of concatenated prompts; ``final``: with slots their pool, else whether to return the states."""
    if u.dim() == 3 and u.shape[0] != 1:
        raise ValueError("u: expected a leading batch of 1 (concatenated sequences)")
    if u.dim() not in (2, 3):
        raise ValueError("u: expected [tokens, channels]")
    call = _Call(u, dt, a, b, c, d, z, dt_bias, dt_softplus)
    device = u.device
    cu = sequence_ends(cu_seqlens, call.tokens, device)
    seqs = cu.numel() - 1
    if slots is not None:
        initial = final = _pool_state(final, call.channels, call.states)
        slots = slot_rows(slots, seqs, device)
        N.device_index(u, final, N.status_word(status))
    else:
        if initial is not None:
            initial = N.aligned(_state(initial, seqs, call.channels, call.states, "initial_state"))
            N.device_index(u, initial)
        final = u.new_empty((seqs, call.channels, call.states), dtype=torch.float32) if final else None
    y = outputs(u, seqs)
    size = N.lib().sq_selective_scan_workspace_bytes(call.tokens, seqs, call.channels, call.states, call.groups)
    workspace = u.new_empty(size, dtype=torch.uint8) if size > 0 else None
    call.launch(N.lib().sq_selective_scan, y, initial, final, slots, cu, status, workspace, seqs)
    return y, final


def selective_scan(u, dt, a, b, c, *, d=None, z=None, dt_bias=None, dt_softplus=True, initial_state=None,
                   output_final_state=True, cu_seqlens=None):
    """Scan of concatenated sequences: (y, final_state).

    u, dt, z: [T, D] or [1, T, D] float32, bfloat16 or float16, alike; a: [D, N]
    float32 (negative), N in {4, 8, 16, 32, 64}; b, c: [T, G, N] (or [T, N] for
    one group) in u's dtype; d, dt_bias: [D] or None, used in fp32; rows any
    stride apart.  cu_seqlens: [S + 1] boundaries (default: one sequence);
    initial_state: [S, D, N] float32 or None (zeros).  y has u's shape and
    dtype, zero for tokens of no sequence; final_state [S, D, N] float32, None
    when ``output_final_state`` is false.
    """
    return _prompts(u, dt, a, b, c, d, z, dt_bias, dt_softplus, cu_seqlens, initial_state, bool(output_final_state), None, None)


def selective_scan_extend(state, u, dt, a, b, c, *, slots, d=None, z=None, dt_bias=None, dt_softplus=True, cu_seqlens=None,
                          status=None):
    """``selective_scan`` on a pool of states [S, D, N]: sequence n continues
    from, and updates in place, row slots[n].  A slot <= 0 (padding) or outside
    the pool (flagged in ``status``, an int32 word) gives zero outputs."""
    if slots is None:
        raise ValueError("slots: required, the pool's row of each sequence")
    return _prompts(u, dt, a, b, c, d, z, dt_bias, dt_softplus, cu_seqlens, None, state, slots, status)[0]


def selective_scan_step(state, u, dt, a, b, c, *, d=None, z=None, dt_bias=None, dt_softplus=True, slots=None, status=None):
    """One token of each request: u, dt, z [B, D], b, c [B, G, N] -> y [B, D];
    ``state`` [S, D, N] float32 (contiguous) is updated in place at rows
    ``slots`` [B] (None: row i for request i, S = B).  Slots are distinct;
    padding and slots outside the pool as in ``selective_scan_extend``."""
    if u.dim() != 2:
        raise ValueError("u: expected [batch, channels]")
    call = _Call(u, dt, a, b, c, d, z, dt_bias, dt_softplus)
    batch = call.tokens
    state = _pool_state(state, call.channels, call.states)
    N.device_index(u, state, N.status_word(status))
    if slots is None and state.shape[0] != batch:
        raise ValueError(f"state: expected {batch} rows without slots")
    y = u.new_empty((batch, call.channels))
    call.launch(N.lib().sq_selective_scan_step, y, None, state, slot_rows(slots, batch, u.device), None, status, None, batch)
    return y


class SelectiveStatePool:
    """Per-request states of a selective layer: ``conv`` [slots, D, W - 1] in the
    activations' dtype and ``state`` [slots, D, N] fp32, zeroed.  Slot 0 is the
    padding sentinel: requests on it get zero outputs and keep nothing."""

    def __init__(self, slots, channels, states, taps=4, dtype=torch.bfloat16, device="cuda"):
        if slots < 1 or channels < 1 or states not in STATES or not 2 <= taps <= 4:
            raise ValueError(f"invalid selective state pool: {slots} slots, {channels} channels, {states} states, {taps} taps")
        N.dtype_code(dtype)
        self.conv = torch.zeros(slots, channels, taps - 1, device=device, dtype=dtype)
        self.state = torch.zeros(slots, channels, states, device=device, dtype=torch.float32)
        self.status = torch.zeros(1, device=device, dtype=torch.int32)

    def convolve(self, x, weight, bias=None, *, slots, cu_seqlens=None, activation="silu"):
        """The convolution of prompts (with ``cu_seqlens``) or of one token each."""
        if cu_seqlens is None:
            return causal_conv1d_step(x, self.conv, weight, bias, slots=slots, activation=activation, status=self.status)
        return causal_conv1d_extend(x, self.conv, weight, bias, slots=slots, cu_seqlens=cu_seqlens, activation=activation,
                                    status=self.status)

    def extend(self, u, dt, a, b, c, slots, cu_seqlens, **options):
        """Prompts of concatenated sequences, each continuing its slot's state."""
        return selective_scan_extend(self.state, u, dt, a, b, c, slots=slots, cu_seqlens=cu_seqlens, status=self.status,
                                     **options)

    def step(self, u, dt, a, b, c, slots, **options):
        """One token of each request."""
        return selective_scan_step(self.state, u, dt, a, b, c, slots=slots, status=self.status, **options)

    def clear(self, slots):
        self.conv[slots] = 0
        self.state[slots] = 0

    def copy(self, source, destination):
        self.conv[destination] = self.conv[source]
        self.state[destination] = self.state[source]

    def check_status(self):
        """Raise if a kernel skipped a request whose slot index was outside the pool (synchronizes)."""
        value = int(self.status.item())
        if value & N.SQ_STATUS_SLOT_RANGE:
            self.status.zero_()
            raise IndexError("a request slot index was outside the state pool; that request was skipped")
