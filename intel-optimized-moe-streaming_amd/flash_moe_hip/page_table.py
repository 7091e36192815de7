"""Page tables of a batch's sequences, kept and extended in HBM.

``PageTable`` holds which pages of a ``PagedCache`` each sequence has, how many
tokens it holds, and the pages that are free.  ``extend`` gives new tokens their
pages, slots and positions from the number each sequence gets, ``trim`` takes
tokens back (rejected drafts, finished sequences).  (The reference preallocates a
cache per sequence, attention.py:144-206.)

Everything is enqueued on the current stream of the table's device (or on
``stream``); nothing synchronizes and no size depends on device data, so a
captured step replays with other numbers.  ``status()`` synchronizes and reports
what the kernels latched.
"""
from __future__ import annotations

import struct

from . import _lib
from .kv_cache import OnStream, check_index

SEQUENCES_MAX = 8192
_EXTEND_WORDS = struct.Struct("15q")
_TRIM_WORDS = struct.Struct("11q")


class PageTable:
    """Tables over tensors the caller keeps: table [sequences, columns], lengths
    [sequences], free [pages] and count [1], all int32: free[:count] are the pages that
    no sequence has, the last of them goes first.  A page is in one sequence's columns
    or among the free ones; columns past a sequence's tokens hold anything.

    page_size is the cache's; at most 8192 sequences, columns * page_size at most
    2^30.  One table serves the caches of all layers.  Its calls have to be in order
    (on one stream, or ordered by events)."""

    def __init__(self, table, lengths, free, count, page_size: int = 64):
        import torch

        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        if table.dim() != 2 or free.dim() != 1:
            raise ValueError("table must be [sequences, columns] and free [pages]")
        sequences, columns = table.shape
        if not 1 <= sequences <= SEQUENCES_MAX or columns < 1 or columns * page_size > 1 << 30 or free.shape[0] < 1:
            raise ValueError(f"a table has 1 to {SEQUENCES_MAX} sequences, at least one page and 2^30 / page_size columns "
                             f"at most; got {sequences} x {columns} and {free.shape[0]} pages")
        index = table.get_device()
        for t, shape, what in ((table, table.shape, "table"), (lengths, (sequences,), "lengths"),
                               (free, free.shape, "free"), (count, (1,), "count")):
            check_index(t, shape, torch.int32, index, what)
        if index < 0:
            raise ValueError(f"expected a CUDA device, got {table.device}")
        self._held, self._fixed = (table, lengths, free, count), None
        self.sequences, self.columns, self.pages, self.page_size = sequences, columns, free.shape[0], page_size
        self.device = table.device
        self.lib = _lib.load()
        self._run, self._index = OnStream(table.device), index
        self._empty, self._int32, self._int64 = torch.empty, torch.int32, torch.int64
        self._flags = torch.zeros(64, dtype=torch.int32, device=table.device)

    table = property(lambda self: self._held[0], doc="Pages of each sequence in order [sequences, columns].")
    lengths = property(lambda self: self._held[1], doc="Tokens each sequence holds [sequences].")
    free = property(lambda self: self._held[2], doc="The free pages: the first `count` of [pages].")
    count = property(lambda self: self._held[3], doc="How many pages are free [1].")

    @classmethod
    def empty(cls, sequences: int, columns: int, pages: int, page_size: int = 64, device="cuda"):
        """A table of sequences without tokens, all pages free (page 0 goes first)."""
        import torch

        as_int = dict(dtype=torch.int32, device=device)
        return cls(torch.zeros((sequences, columns), **as_int), torch.zeros(sequences, **as_int),
                   torch.arange(pages - 1, -1, -1, **as_int), torch.full((1,), pages, **as_int), page_size)

    def _words(self):
        """The table's share of a call's words, at the addresses its tensors have now
        (their storage may have moved)."""
        table, lengths, free, count = self._held
        w = self._fixed
        if w and table.data_ptr() == w[0] and lengths.data_ptr() == w[2] and free.data_ptr() == w[3] and (
                count.data_ptr() == w[4]):
            return w
        for t, shape in ((table, (self.sequences, self.columns)), (lengths, (self.sequences,)), (free, (self.pages,)),
                         (count, (1,))):
            if t.shape != shape or t.dtype != self._int32 or t.get_device() != self._index or not t.is_contiguous() or (
                    t.untyped_storage().nbytes() < (t.storage_offset() + t.numel()) * 4):
                raise ValueError(f"a tensor of the table is no longer int32 {tuple(shape)}, contiguous, on {self.device}")
        self._fixed = w = (table.data_ptr(), self.columns, lengths.data_ptr(), free.data_ptr(), count.data_ptr(),
                           self.sequences, self.pages, self.page_size)
        return w

    def extend(self, new, tokens: int, *, stream=None):
        """Room for new[b] >= 0 more tokens of each sequence (int32 [sequences]), in a
        batch of `tokens` rows.  Returns (starts, slots, positions): starts int32
        [sequences + 1], sequence b's rows are starts[b] .. starts[b + 1] - 1; slots int64
        and positions int32 [tokens], -1 in the rows behind the last sequence.  They are
        what ``PagedCache.write`` and ``attend`` and ``Rotary.apply`` take, with this
        table's ``table`` and ``lengths``, which count the new tokens from then on.

        A call that cannot be served changes nothing and gives no rows (starts of 0, slots
        and positions of -1): -10 latches where pages are lacking, -9 where a number is
        negative, a sequence outgrows its columns, or the new tokens are more than
        `tokens`, or a length or the count is out of range.  Numbers in ``free`` and ``table``
        that are no pages are found as they are handed out: the call is carried out, rows of
        such a page get the slot pages * page_size, past a cache of as many pages (``write``
        skips and reports it), and -9 latches."""
        check_index(new, (self.sequences,), self._int32, self._index, "new")
        if isinstance(tokens, bool) or not isinstance(tokens, int) or not 0 <= tokens <= 1 << 30:
            raise ValueError(f"tokens must be a whole number from 0 to 2^30, got {tokens!r}")
        return self._run(stream, self._extend, new, tokens)

    def _extend(self, handle, new, tokens):
        device = self.device
        starts = self._empty(self.sequences + 1, dtype=self._int32, device=device)
        slots = self._empty(tokens, dtype=self._int64, device=device)
        positions = self._empty(tokens, dtype=self._int32, device=device)
        rc = self.lib.mqh_pages_extend_words(_EXTEND_WORDS.pack(
            new.data_ptr(), *self._words(), tokens, starts.data_ptr(), slots.data_ptr(), positions.data_ptr(),
            self._flags.data_ptr(), handle))
        if rc:
            _lib.check(rc, "mqh_pages_extend")
        return starts, slots, positions

    def trim(self, keep, *, stream=None):
        """Sequence b keeps its first min(lengths[b], keep[b]) tokens (int32 [sequences]);
        0 ends it.  Pages behind them become free: those that the last ``extend`` took
        lie among the free ones where they were.  A negative number, or a length or count
        out of range, changes nothing and latches -9; a number that is no page goes back
        like the others and latches -9."""
        check_index(keep, (self.sequences,), self._int32, self._index, "keep")
        self._run(stream, self._trim, keep)

    def _trim(self, handle, keep):
        rc = self.lib.mqh_pages_trim_words(_TRIM_WORDS.pack(keep.data_ptr(), *self._words(), self._flags.data_ptr(), handle))
        if rc:
            _lib.check(rc, "mqh_pages_trim")

    def status(self, stream=None) -> int:
        """Synchronizes; 0, -9 (a number, length, page or count out of range) or -10 (no
        free pages left) since the last call."""
        return int(self._run(stream, lambda handle: self.lib.mqh_status(self._flags.data_ptr(), handle)))
