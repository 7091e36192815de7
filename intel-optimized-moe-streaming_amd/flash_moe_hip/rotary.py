"""Rotary positions of queries and keys in HBM.

``Rotary`` holds a layer's frequencies and turns the first channels of every head's
row by the angles of its position, after the norm of each head's row where weights
are given (the reference's attention layers norm and rotate on the host,
rope.py, attention.py:220-306).

Everything is enqueued on the current stream of the frequencies' device (or on
``stream``); nothing synchronizes.  ``status()`` synchronizes and reports what the
kernels latched.  There is no backward: tensors that require grad are refused.
"""
from __future__ import annotations

import math
import struct

from . import _lib
from .kv_cache import HEAD_DIMS, OnStream, _types, check_index, check_rows

LAYOUTS = ("half", "interleaved")
_WORDS = struct.Struct("15qd2qd8q")


def frequencies(rotary_dim: int, base: float = 10000.0, scaling=None):
    """Radians a position of each of the rotary_dim / 2 pairs, base^(-2 i / rotary_dim),
    and the factor of the turned channels, as (list of float, float).  ``scaling``
    stretches them for contexts longer than the trained one:

      {"kind": "linear", "factor": s}              frequencies / s
      {"kind": "yarn", "factor": s, "original": n, "fast": 32, "slow": 1, "amplitude": a}
          by parts: pairs that turn more than `fast` times over the n trained positions
          stay, those that turn less than `slow` times are divided by s, a ramp over the
          pairs' numbers between; the factor is a, 0.1 ln s + 1 without it
      {"kind": "bands", "factor": s, "original": n, "low": 1, "high": 4}
          the same by turns over the n positions: `high` and more stay, `low` and fewer are
          divided, a ramp over the turns between
    """
    if not 1 < base < math.inf:
        raise ValueError(f"base must be above 1 and finite, got {base}")
    f = [float(base) ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling is None:
        return f, 1.0
    known = {"linear": ("factor",), "yarn": ("factor", "original", "fast", "slow", "amplitude"),
             "bands": ("factor", "original", "low", "high")}
    sc = dict(scaling)
    kind = sc.pop("kind", None)
    if kind not in known:
        raise ValueError(f"a scaling's kind is one of {tuple(known)}, got {kind!r}")
    if any(name not in known[kind] for name in sc) or any(name not in sc for name in known[kind][:2]):
        raise ValueError(f"a {kind} scaling has {known[kind]}, got {tuple(sc)}")
    if not all(0 < x < math.inf for x in sc.values()) or sc["factor"] < 1:
        raise ValueError(f"a scaling's numbers are positive and finite and its factor at least 1, got {sc}")
    if not 2.0 ** -149 <= sc.get("amplitude", 1.0) < 2.0 ** 128 - 2.0 ** 103:
        raise ValueError(f"amplitude must be an FP32 number, got {sc['amplitude']}")
    s = sc["factor"]
    if kind == "linear":
        return [x / s for x in f], 1.0
    if kind == "yarn":
        fast, slow = sc.get("fast", 32.0), sc.get("slow", 1.0)
        if fast <= slow:
            raise ValueError(f"fast must be above slow, got {fast} and {slow}")
        # the pair's number whose frequency turns so many times over the trained positions
        first, last = (rotary_dim * math.log(sc["original"] / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (fast, slow))
        first, last = max(math.floor(first), 0), min(math.ceil(last), rotary_dim - 1)
        span = max(last - first, 0.001)
        ramp = [min(max((i - first) / span, 0.0), 1.0) for i in range(len(f))]
        return [x / s * r + x * (1 - r) for x, r in zip(f, ramp)], sc.get("amplitude", 0.1 * math.log(s) + 1.0)
    low, high = sc.get("low", 1.0), sc.get("high", 4.0)
    if high <= low:
        raise ValueError(f"high must be above low, got {high} and {low}")
    keep = [min(max((sc["original"] * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for x in f]
    return [x / s * (1 - r) + x * r for x, r in zip(f, keep)], 1.0


class Rotary:
    """Rotary positions for heads of head_dim (64, 128 or 256) channels, of which the
    first rotary_dim (all without it; a multiple of 16) are turned in pairs: "half"
    (i, i + rotary_dim / 2) or "interleaved" (2 i, 2 i + 1).  base and scaling as in
    ``frequencies``."""

    def __init__(self, head_dim: int, rotary_dim: int | None = None, *, base: float = 10000.0, layout: str = "half",
                 scaling=None, device="cuda"):
        import torch

        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if not 16 <= rotary_dim <= head_dim or rotary_dim % 16:
            raise ValueError(f"rotary_dim must be a multiple of 16 up to head_dim, got {rotary_dim}")
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
        self.head_dim, self.rotary_dim, self.layout = head_dim, rotary_dim, layout
        self.frequencies, self.amplitude = frequencies(rotary_dim, base, scaling)
        # turns a position as whole numbers of 2^-64 (below 2^62: a frequency is at most 1)
        turns = [round(x / (2 * math.pi) * 2.0 ** 64) for x in self.frequencies]
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"expected a CUDA device, got {device}")
        self._turns = torch.tensor(turns, dtype=torch.int64, device=device)
        self.device = self._turns.device
        self.lib = _lib.load()
        self._run, self._index = OnStream(self.device), self._turns.get_device()
        self._types, self._int32, self._float = _types(), torch.int32, (torch.float32,)
        self._empty_like, self._format = torch.empty_like, torch.contiguous_format  # half of empty's host time
        self._flags = torch.zeros(64, dtype=torch.int32, device=self.device)
        self._flag = self._flags.data_ptr()

    def apply(self, q, k, positions, *, q_weight=None, k_weight=None, eps: float = 1e-6, out=None, stream=None):
        """(q, k) turned: q [tokens, heads, head_dim], k [tokens, kv_heads, head_dim] of one
        type (FP32, FP16 or BF16; any token and head strides), positions int32 [tokens].
        Channels from rotary_dim on stay as they are.  q_weight, k_weight (FP32 [head_dim],
        either or both): the row first goes through x / sqrt(mean x^2 + eps) * weight.
        FP32 inside, rounded once.  A negative position turns the other way; rows of position
        -1, a batch's padding, are turned by one position back and never reported.  out: two tensors like q and k to write
        to, of any token and head strides; q and k themselves turn them in place, other
        overlaps are not allowed.  An output of another row that its type cannot hold latches
        -4."""
        if q.dim() != 3 or k.dim() != 3:
            raise ValueError("q and k must be [tokens, heads, head_dim]")
        index, dim = self._index, self.head_dim
        n, heads, _ = q.shape
        kv_heads = k.shape[1]
        if not 1 <= heads <= 4096 or not 1 <= kv_heads <= 4096:
            raise ValueError(f"heads must be 1 to 4096, got {heads} and {kv_heads}")
        if n > 1 << 24:
            raise ValueError(f"at most 2^24 tokens a call, got {n}")
        qt, qh, _ = check_rows(q, (n, heads, dim), self._types, index, "q")
        like = (q.dtype,)
        kt, kh, _ = check_rows(k, (n, kv_heads, dim), like, index, "k")
        check_index(positions, (n,), self._int32, index, "positions")
        weights = []
        for w, what in ((q_weight, "q_weight"), (k_weight, "k_weight")):
            if w is not None:
                check_rows(w, (dim,), self._float, index, what)
            weights.append(0 if w is None else w.data_ptr())
        eps = float(eps)
        if not 1e-30 <= eps <= 1e30:
            raise ValueError(f"eps must be from 1e-30 to 1e30, got {eps}")
        if out is not None:
            check_rows(out[0], q.shape, like, index, "out[0]")
            check_rows(out[1], k.shape, like, index, "out[1]")
        return self._run(stream, self._apply, q, k, out, (
            q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, self._types[q.dtype], positions.data_ptr(), n, heads, kv_heads, dim,
            self._turns.data_ptr(), self.rotary_dim, int(self.layout == "interleaved"), self.amplitude, *weights, eps))

    def _apply(self, handle, q, k, out, words):
        if out is None:
            qo, ko = self._empty_like(q, memory_format=self._format), self._empty_like(k, memory_format=self._format)
        else:
            qo, ko = out
        if words[8]:
            rc = self.lib.mqh_rotary_words(_WORDS.pack(
                *words, qo.data_ptr(), *qo.stride()[:2], ko.data_ptr(), *ko.stride()[:2], self._flag, handle))
            if rc:
                _lib.check(rc, "mqh_rotary")
        return qo, ko

    def status(self, stream=None) -> int:
        """Synchronizes; 0, or -4 (an output was not finite) since the last call."""
        return int(self._run(stream, lambda handle: self.lib.mqh_status(self._flag, handle)))
