"""Linear attention with a decay per head over resident states, for prompts and
single tokens of many sequences.

``LinearState`` keeps the recurrent states of a layer for several sequences in
HBM and runs the gated recurrence of the reference's recurrent layers
(gated_deltanet.py:264-402), with the delta rule (``beta`` given) or without:

    S <- e^gate S;  u = beta (v - S k)  or  v;  S <- S + u k^T;  out = S q

``step`` takes one token of every sequence, ``prefill`` whole prompts of
different lengths.  ``native_expert.DeltaState`` is the single-sequence state
whose step has the reference kernel's summation order bit for bit; its
``prefill`` runs the same prompt kernels.

Everything is enqueued on the current stream of the state's device (or on
``stream``); nothing synchronizes.  There is no backward.
"""
from __future__ import annotations

import functools
import struct

from . import _lib
from .kv_cache import OnStream, _device_name, _types, check_index, check_rows

_STEP_WORDS = struct.Struct("23q")
_PREFILL_WORDS = struct.Struct("27q")
KEY_DIM_MAX, VALUE_DIM_MAX = 256, 1024
CHUNK_STRIDE_MAX = 1 << 22   # a prompt's offsets within a chunk of tokens are 32-bit


@functools.lru_cache(maxsize=512)
def _prefill_bytes(lib, tokens, seqs, heads, key_dim, value_dim, delta):
    return int(lib.mqh_linear_prefill_workspace_bytes(tokens, seqs, heads, key_dim, value_dim, delta))


def check_dims(key_dim: int, value_dim: int):
    if key_dim < 4 or key_dim > KEY_DIM_MAX or key_dim % 4 or value_dim < 4 or value_dim > VALUE_DIM_MAX or value_dim % 4:
        raise ValueError(f"key_dim must be a multiple of 4 up to {KEY_DIM_MAX}, value_dim one up to {VALUE_DIM_MAX}; "
                         f"got {key_dim} and {value_dim}")


def check_state(state, shape, index):
    """The state a call is about to update in place is still the one its object was made
    for: FP32 of its shape, contiguous, on CUDA device `index` (-1: the CPU)."""
    if state.shape == shape and state.dtype is _FP32()[0] and state.is_contiguous() and not state.requires_grad:
        if state.get_device() != index:
            raise ValueError(f"the state is on {state.device}, expected {_device_name(index)}")
        return
    raise ValueError(f"the state must be a contiguous FP32 tensor of shape {tuple(shape)} without grad")


def _inputs(state, n, q, k, v, beta, gate, out, prompt):
    """Check one call's rows against the states' shape; the shared argument words."""
    _, heads, dv, dk = state.shape
    index, types = state.get_device(), _types()
    key_heads = q.shape[1] if q.dim() == 3 else -1
    if key_heads < 1 or heads % key_heads:
        raise ValueError(f"q must be [tokens, key_heads, key_dim] with key_heads a divisor of {heads}")
    rows = (n, heads, dv)
    vt, vh, _ = check_rows(v, rows, types, index, "v")
    like = (v.dtype,)
    qt, qh, _ = check_rows(q, (n, key_heads, dk), like, index, "q")
    kt, kh, _ = check_rows(k, (n, key_heads, dk), like, index, "k")
    if prompt and n > 1 and max(qt, kt, vt) > CHUNK_STRIDE_MAX:
        name, stride = max(("q", qt), ("k", kt), ("v", vt), key=lambda t: t[1])
        raise ValueError(f"{name} has a token stride of {stride} elements; a prompt takes up to {CHUNK_STRIDE_MAX}")
    gt, _ = check_rows(gate, (n, heads), _FP32(), index, "gate")
    bp = bt = 0
    if beta is not None:
        bt, _ = check_rows(beta, (n, heads), _FP32(), index, "beta")
        bp = beta.data_ptr()
    if out is not None:
        check_rows(out, rows, like, index, "out")
        if not out.is_contiguous():
            raise ValueError("out must be contiguous")
    return (q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, types[v.dtype], bp, bt, gate.data_ptr(), gt,
            state.data_ptr()), key_heads


@functools.lru_cache(maxsize=None)
def _FP32():
    import torch

    return (torch.float32,)


def prefill_states(lib, run, flags, state, q, k, v, beta, gate, starts, out, stream):
    """mqh_linear_prefill over states [sequences, heads, value_dim, key_dim]."""
    import torch

    seqs, heads, dv, dk = state.shape
    n = v.shape[0]
    words, key_heads = _inputs(state, n, q, k, v, beta, gate, out, True)
    if starts is not None:
        check_index(starts, (seqs + 1,), torch.int32, state.get_device(), "starts")
    elif seqs != 1:
        raise ValueError("prompts of several sequences need starts")
    need = 0
    if n:
        need = _prefill_bytes(lib, n, seqs, heads, dk, dv, int(beta is not None))
        if need < 0:
            _lib.check(need, "mqh_linear_prefill_workspace_bytes")

    def call(handle):
        y = torch.empty((n, heads, dv), dtype=v.dtype, device=state.device) if out is None else out
        if n:
            ws = torch.empty(need, dtype=torch.uint8, device=state.device)
            _lib.check(lib.mqh_linear_prefill_words(_PREFILL_WORDS.pack(
                *words, y.data_ptr(), starts.data_ptr() if starts is not None else 0, n, seqs, heads, key_heads, dk, dv,
                ws.data_ptr(), need, flags.data_ptr(), handle)), "mqh_linear_prefill")
        return y

    return run(stream, call)


class LinearState:
    """States of `sequences` sequences of one layer, [sequences, heads, value_dim,
    key_dim] FP32 in HBM (`state`: kept as it is where it is such a tensor)."""

    def __init__(self, sequences: int, heads: int, value_dim: int, key_dim: int, device=None, state=None):
        import torch

        self.shape = (int(sequences), int(heads), int(value_dim), int(key_dim))
        if min(self.shape) < 1:
            raise ValueError(f"a state's sizes are at least 1, got {self.shape}")
        check_dims(self.shape[3], self.shape[2])
        if state is None:
            self.state = torch.zeros(self.shape, dtype=torch.float32, device=device or "cuda")
        else:
            if tuple(state.shape) != self.shape:
                raise ValueError("state shape mismatch")
            if torch.is_tensor(state) and state.requires_grad:
                raise ValueError("the state requires grad; these calls have no backward")
            if device is None:
                device = state.device if torch.is_tensor(state) else "cuda"
            self.state = torch.as_tensor(state, dtype=torch.float32).to(device).contiguous()
        if self.state.device.type != "cuda":
            raise ValueError(f"expected a CUDA device, got {self.state.device}")
        self.lib = _lib.load()
        self._run, self._empty, self._index = OnStream(self.state.device), torch.empty, self.state.get_device()
        self._flags = torch.zeros(64, dtype=torch.int32, device=self.state.device)

    def reset(self):
        self.state.zero_()

    def step(self, q, k, v, beta, gate, *, out=None, stream=None):
        """One token of every sequence: q, k [sequences, key_heads, key_dim], v
        [sequences, heads, value_dim] (FP32, FP16 or BF16, any token and head
        strides; value head h uses key head h // (heads // key_heads)), beta (None:
        no delta rule) and gate [sequences, heads] FP32.  Returns out [sequences,
        heads, value_dim] of v's type."""
        seqs, heads, dv, dk = self.shape
        check_state(self.state, self.shape, self._index)
        words, key_heads = _inputs(self.state, seqs, q, k, v, beta, gate, out, False)
        return self._run(stream, self._step, v, out, words, (seqs, heads, key_heads, dk, dv))

    def _step(self, handle, v, out, words, sizes):
        if out is None:
            out = self._empty(v.shape, dtype=v.dtype, device=self.state.device)
        rc = self.lib.mqh_linear_step_words(_STEP_WORDS.pack(*words, out.data_ptr(), *sizes, self._flags.data_ptr(), handle))
        if rc:
            _lib.check(rc, "mqh_linear_step")
        return out

    def prefill(self, q, k, v, beta, gate, *, starts=None, out=None, stream=None):
        """Prompts: the arguments of ``step`` with [tokens, ...] rows (token strides of
        q, k and v up to 2^22 elements); sequence b's are rows starts[b] ..
        starts[b + 1] - 1 (int32 [sequences + 1] on the device; may be omitted for one
        sequence).  The same states and outputs as ``step`` token by token up to FP32
        rounding; rows of no sequence are left as they were.  A value that is not
        finite also reaches earlier tokens of its 64-token chunk."""
        check_state(self.state, self.shape, self._index)
        return prefill_states(self.lib, self._run, self._flags, self.state, q, k, v, beta, gate, starts, out, stream)

    def status(self, stream=None) -> int:
        """Synchronizes; 0, -4 (an output was not finite) or -9 (starts out of
        range) since the last call."""
        return int(self._run(stream, lambda handle: self.lib.mqh_status(self._flags.data_ptr(), handle)))
