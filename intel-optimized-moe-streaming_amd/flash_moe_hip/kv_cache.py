"""Paged key/value cache of an attention layer in HBM, and attention over it.

``PagedCache`` holds one layer's keys and values as pages [pages, kv_heads,
page_size, head_dim] in FP16, BF16 or as 8-bit codes with one FP32 scale per
token and head.  ``write`` stores new tokens' rows (quantizing them for an 8-bit
cache), ``read`` gives rows back as values, ``attend`` is attention of new
tokens over what the sequences hold: chunks of prompts, drafts, or one token a
sequence.  (The reference keeps a preallocated FP16 cache per sequence and
attends on the host, attention.py:144-306.)

Everything is enqueued on the current stream of the cache's device (or on
``stream``); nothing synchronizes.  ``status()`` synchronizes and reports what
the kernels latched.  There is no backward: tensors that require grad are
refused.
"""
from __future__ import annotations

import functools
import struct

from . import _lib

HEAD_DIMS = (64, 128, 256)
F32, F16, BF16, Q8 = 0, 1, 2, 3   # the library's element types (MQH_MIX_*)

_WRITE_WORDS = struct.Struct("20q")
_READ_WORDS = struct.Struct("16q")
_ATTEND_WORDS = struct.Struct("21qd5q")


@functools.lru_cache(maxsize=None)
def _types():
    import torch

    return {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


@functools.lru_cache(maxsize=512)
def _attend_bytes(lib, tokens, seqs, single, heads, kv_heads, dim, most):
    return int(lib.mqh_attend_workspace_bytes(tokens, seqs, single, heads, kv_heads, dim, most))


def check_rows(t, shape, types, index, what):
    """The strides of a tensor of rows as the kernels take it: of `shape` and a type
    of `types`, on CUDA device `index`, its last dimension contiguous (other strides
    are free).  (A small call's time is the host's: one test where all is well.)"""
    strides = t.stride()
    if t.shape == shape and t.dtype in types and t.get_device() == index and not t.requires_grad and (
            strides[-1] == 1 or shape[-1] == 1):
        return strides
    if t.shape != shape:
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype not in types:
        raise ValueError(f"{what} is {t.dtype}, expected one of {[str(d) for d in types]}")
    if strides[-1] != 1 and shape[-1] != 1:
        raise ValueError(f"{what} must be contiguous in its last dimension")
    if t.get_device() != index:
        raise ValueError(f"{what} is on {t.device}, expected {_device_name(index)}")
    raise ValueError(f"{what} requires grad; these calls have no backward")


def _device_name(index):
    return f"cuda:{index}" if index >= 0 else "cpu"


def check_index(t, shape, dtype, index, what):
    """An index tensor: exact shape and type, contiguous, on CUDA device `index`."""
    if t.shape == shape and t.dtype == dtype and t.get_device() == index and t.is_contiguous():
        return
    if t.shape != shape or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of shape {tuple(shape)}")
    raise ValueError(f"{what} is on {t.device}, expected {_device_name(index)}")


class OnStream:
    """Runs a call on a device: with it current and the handle of its current
    stream, or of the stream given (of the same device), which the call's tensors
    are then allocated on."""

    def __init__(self, device):
        import torch

        self.index = device.index
        self._torch = torch
        self._current = torch.cuda.current_device
        self._stream_of = _lib.stream_accessor()

    def __call__(self, stream, call, *args):
        if stream is not None:
            if stream.device.index != self.index:
                raise ValueError(f"the stream is on {stream.device}, expected {_device_name(self.index)}")
            with self._torch.cuda.stream(stream):
                return call(stream.cuda_stream, *args)
        if self._current() != self.index:
            with self._torch.cuda.device(self.index):
                return call(self._stream_of(self.index), *args)
        return call(self._stream_of(self.index), *args)


class PagedCache:
    """One layer's paged cache over tensors the caller keeps: k and v [pages,
    kv_heads, page_size, head_dim], FP16, BF16 or int8 (then k_scale and v_scale
    [pages, kv_heads, page_size] FP32), contiguous.  head_dim 64, 128 or 256,
    page_size a power of two from 16 to 1024.  Scales are those that ``write``
    stores: 0, NaN, or 2^-100 and more.

    A *slot* is page * page_size + offset; a sequence's page table lists its
    pages in order."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        import torch

        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must be [pages, kv_heads, page_size, head_dim] of one type")
        pages, kv_heads, page_size, dim = k.shape
        if dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {dim}")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        if pages < 1 or kv_heads < 1 or kv_heads > 1024:
            raise ValueError("a cache has at least one page and 1 to 1024 kv heads")
        types = {torch.float16: F16, torch.bfloat16: BF16, torch.int8: Q8}
        if k.dtype not in types:
            raise ValueError(f"a cache is FP16, BF16 or int8, got {k.dtype}")
        held = [k, v]
        if k.dtype == torch.int8:
            if k_scale is None or v_scale is None:
                raise ValueError("an int8 cache needs k_scale and v_scale")
            for s in (k_scale, v_scale):
                if s.dtype != torch.float32 or tuple(s.shape) != (pages, kv_heads, page_size):
                    raise ValueError("scales must be FP32 [pages, kv_heads, page_size]")
            held += [k_scale, v_scale]
        elif k_scale is not None or v_scale is not None:
            raise ValueError("only int8 caches have scales")
        if any(t.device != k.device or not t.is_contiguous() for t in held):
            raise ValueError("a cache's tensors must be contiguous and on one device")
        if any(t.requires_grad for t in held):
            raise ValueError("a tensor of the cache requires grad; these calls have no backward")
        if k.device.type != "cuda":
            raise ValueError(f"expected a CUDA device, got {k.device}")
        self._held = (k, v, k_scale, v_scale)
        self._like = [None if t is None else (t.shape, t.dtype, t.device) for t in self._held]
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, kv_heads, page_size, dim
        self.device = k.device
        self.lib = _lib.load()
        self._run = OnStream(k.device)
        self._index = k.device.index
        self._types = _types()
        self._empty, self._int32, self._int64, self._uint8 = torch.empty, torch.int32, torch.int64, torch.uint8
        int8 = k.dtype == torch.int8
        self._q_types = (torch.float16, torch.bfloat16) if int8 else (k.dtype,)
        self._read_type = torch.float32 if int8 else k.dtype
        self._flags = torch.zeros(64, dtype=torch.int32, device=k.device)
        self._fixed = (*self._addresses(), types[k.dtype], pages, kv_heads, page_size, dim)

    # (a call's addresses and sizes are those of the tensors checked here: no others can be put in their place)
    k = property(lambda self: self._held[0], doc="The keys [pages, kv_heads, page_size, head_dim].")
    v = property(lambda self: self._held[1], doc="The values, as the keys.")
    k_scale = property(lambda self: self._held[2], doc="An int8 cache's scales [pages, kv_heads, page_size], or None.")
    v_scale = property(lambda self: self._held[3], doc="The values' scales.")

    def _addresses(self):
        return tuple(0 if t is None else t.data_ptr() for t in self._held)

    def _words(self):
        """The cache's share of a call's words, at the addresses its tensors have now
        (their storage may have moved)."""
        k, v, ks, vs = self._held
        w = self._fixed
        if k.data_ptr() != w[0] or v.data_ptr() != w[1] or (
                ks is not None and (ks.data_ptr() != w[2] or vs.data_ptr() != w[3])):
            for t, like in zip(self._held, self._like):
                if t is not None and ((t.shape, t.dtype, t.device) != like or not t.is_contiguous() or (
                        t.untyped_storage().nbytes() < (t.storage_offset() + t.numel()) * t.element_size())):
                    shape, dtype, device = like
                    raise ValueError(f"a tensor of the cache is no longer {dtype} {tuple(shape)}, contiguous, on {device}")
            self._fixed = w = (*self._addresses(), *w[4:])
        return w

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, dtype=None, device="cuda"):
        """A cache of zeros; dtype torch.float16 (default), torch.bfloat16 or torch.int8."""
        import torch

        dtype = torch.float16 if dtype is None else dtype
        shape = (pages, kv_heads, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        if dtype != torch.int8:
            return cls(k, v)
        return cls(k, v, *(torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))

    def slots(self, page_table, seq, position):
        """Slots of positions of sequences: page_table [sequences, columns], seq
        and position index tensors of one shape.  A negative position gives -1,
        which write and read skip; one past the table gives a slot past the cache,
        which they report."""
        column, last = position // self.page_size, page_table.shape[1] - 1
        page = page_table[seq, column.clamp(0, max(last, 0))].long()
        slot = page * self.page_size + position % self.page_size
        slot = slot.masked_fill(column > last, self.pages * self.page_size)
        return slot.masked_fill(position < 0, -1)

    def write(self, k, v, slots, *, stream=None):
        """Store rows k, v [tokens, kv_heads, head_dim] (FP32, FP16 or BF16, any
        token and head strides) at `slots` [tokens] int64; a negative slot is
        skipped, one past the cache is skipped and latched (-9).  Each slot may
        occur once in a call, of at most 2^30 tokens.  16-bit caches round once; an
        int8 cache stores round(x / s), s = max|x| / 127 of the row.  A value that is
        not finite (or that an FP16 cache cannot hold) latches -4; in an int8 cache
        its row then reads back as NaN."""
        n = self._tokens(slots)
        shape = (n, self.kv_heads, self.head_dim)
        kt, kh, _ = check_rows(k, shape, self._types, self._index, "k")
        vt, vh, _ = check_rows(v, shape, (k.dtype,), self._index, "v")
        if n:
            self._run(stream, self._write, (k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, self._types[k.dtype],
                                            slots.data_ptr(), n, *self._words(), self._flags.data_ptr()))

    def _write(self, handle, words):
        rc = self.lib.mqh_kv_write_words(_WRITE_WORDS.pack(*words, handle))
        if rc:
            _lib.check(rc, "mqh_kv_write")

    def _tokens(self, slots):
        n = slots.shape[0] if slots.dim() == 1 else -1
        check_index(slots, (n,), self._int64, self._index, "slots")
        return n

    def read(self, slots, dtype=None, *, stream=None):
        """(k, v) [tokens, kv_heads, head_dim] at `slots` [tokens] int64 as `dtype`
        (the cache's own, FP32 for int8); rows of negative slots are zeros, so are
        those past the cache, which latch -9.  A number that `dtype` cannot hold
        becomes infinite and latches -4."""
        n = self._tokens(slots)
        if dtype is None:
            dtype = self._read_type
        if dtype not in self._types:
            raise ValueError(f"rows are read as FP32, FP16 or BF16, not {dtype}")
        return self._run(stream, self._read, slots, n, dtype)

    def _read(self, handle, slots, n, dtype):
        rows = self._empty((2, n, self.kv_heads, self.head_dim), dtype=dtype, device=self.device)
        k, v = rows.unbind()
        if n:
            rc = self.lib.mqh_kv_read_words(_READ_WORDS.pack(
                slots.data_ptr(), n, *self._words(), k.data_ptr(), v.data_ptr(), self._types[dtype],
                self._flags.data_ptr(), handle))
            if rc:
                _lib.check(rc, "mqh_kv_read")
        return k, v

    def attend(self, q, page_table, lengths, starts=None, *, scale=None, out=None, stream=None):
        """Attention of new tokens, whose rows are already written, over the cache.

        q [tokens, heads, head_dim] (heads a multiple of kv_heads, at most 128
        times; the cache's type, FP16 or BF16 for int8 caches; any token and head
        strides); page_table [sequences, columns] int32; lengths [sequences] int32:
        tokens a sequence holds, the new ones included.  starts [sequences + 1]
        int32: sequence b's queries are rows starts[b] .. starts[b + 1] - 1, the
        last of its tokens; without it every sequence has one.  Query head h reads
        kv head h // (heads // kv_heads).  Each query sees the keys up to its own
        position; a row that sees none (a length below its queries) is zeros; rows
        of `out` that belong to no sequence are left as they were (without `out`
        they hold anything).  scale > 0
        (default head_dim ** -0.5).  Returns out [tokens, heads, head_dim] of q's
        type.  Probabilities are rounded once to the cache's 16-bit type (FP16 for
        int8), sums are FP32; BF16 queries of an int8 cache are multiplied as FP16
        times a power of two of their row (exact down to 2^-17 of its largest).  Page
        numbers, lengths and starts out of range latch -9 (the rows concerned are
        then undefined), outputs that are not finite -4."""
        if q.dim() != 3 or page_table.dim() != 2:
            raise ValueError("q must be [tokens, heads, head_dim] and page_table [sequences, columns]")
        tokens, heads, _ = shape = q.shape
        seqs, cols = page_table.shape
        index = self._index
        qt, qh, _ = check_rows(q, (tokens, heads, self.head_dim), self._q_types, index, "q")
        group = heads // self.kv_heads
        if group * self.kv_heads != heads or not 1 <= group <= 128:
            raise ValueError(f"heads must be 1 to 128 times the cache's {self.kv_heads}, got {heads}")
        row, step = page_table.stride()
        if page_table.dtype != self._int32 or page_table.get_device() != index or (step != 1 and cols > 1) or (
                row < cols and seqs > 1):
            raise ValueError(f"page_table must be int32 rows on {self.device}")
        check_index(lengths, (seqs,), self._int32, index, "lengths")
        if starts is not None:
            check_index(starts, (seqs + 1,), self._int32, index, "starts")
        elif tokens != seqs:
            raise ValueError("without starts there is one query a sequence")
        scale = self.head_dim ** -0.5 if scale is None else float(scale)
        if not 0 < scale < float("inf"):
            raise ValueError("scale must be positive and finite")
        if out is not None:
            check_rows(out, shape, (q.dtype,), index, "out")
            if not out.is_contiguous() or out.data_ptr() % 16:
                raise ValueError("out must be contiguous and 16-byte aligned")
        need = 0
        if tokens and seqs:
            if cols == 0:
                raise ValueError("page_table has no columns")
            need = _attend_bytes(self.lib, tokens, seqs, int(starts is None), heads, self.kv_heads, self.head_dim,
                                 cols * self.page_size)
            if need < 0:
                _lib.check(need, "mqh_attend_workspace_bytes")
        return self._run(stream, self._attend, q, out, need, (
            q.data_ptr(), qt, qh, self._types[q.dtype], tokens, starts.data_ptr() if starts is not None else 0, seqs,
            heads, *self._words(), page_table.data_ptr(), row if seqs > 1 else cols, cols, lengths.data_ptr(), scale))

    def _attend(self, handle, q, out, need, words):
        if out is None:
            out = self._empty(q.shape, dtype=q.dtype, device=self.device)
        if words[4] and words[6]:
            ws = self._empty(need, dtype=self._uint8, device=self.device) if need else None
            rc = self.lib.mqh_attend_words(_ATTEND_WORDS.pack(
                *words, out.data_ptr(), ws.data_ptr() if need else 0, need, self._flags.data_ptr(), handle))
            if rc:
                _lib.check(rc, "mqh_attend")
        return out

    def status(self, stream=None) -> int:
        """Synchronizes; 0, -4 (a value that is not finite) or -9 (a slot, page,
        length or start out of range) since the last call."""
        return int(self._run(stream, lambda handle: self.lib.mqh_status(self._flags.data_ptr(), handle)))
