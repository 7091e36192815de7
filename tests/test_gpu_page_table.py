"""Page tables on the GPU against the same kept in Python."""
from __future__ import annotations

import random

import pytest
import torch

pytestmark = pytest.mark.gpu


class Plain:
    def __init__(self, t):
        self.size, self.cols, self.pages = t.page_size, t.columns, t.pages
        self.table, self.lengths = t.table.tolist(), t.lengths.tolist()
        self.free, self.count = t.free.tolist(), int(t.count)

    def extend(self, new, rows):
        starts, slots, positions = [0], [], []
        for b, n in enumerate(new):
            for p in range(self.lengths[b], self.lengths[b] + n):
                if p % self.size == 0:
                    self.count -= 1
                    self.table[b][p // self.size] = self.free[self.count]
                slots.append(self.table[b][p // self.size] * self.size + p % self.size)
                positions.append(p)
            self.lengths[b] += n
            starts.append(starts[-1] + n)
        fill = [-1] * (rows - len(slots))
        return starts, slots + fill, positions + fill

    def trim(self, keep):
        back = []
        for b, n in enumerate(keep):
            n = min(n, self.lengths[b])
            back += self.table[b][-(-n // self.size):-(-self.lengths[b] // self.size)]
            self.lengths[b] = n
        self.free[self.count:self.count + len(back)] = back[::-1]
        self.count += len(back)

    def check(self, t):
        assert t.table.tolist() == self.table and t.lengths.tolist() == self.lengths
        assert int(t.count) == self.count and t.free.tolist() == self.free
        mine = [p for row, n in zip(self.table, self.lengths) for p in row[:-(-n // self.size)]]
        assert sorted(mine + self.free[:self.count]) == list(range(self.pages))


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def extend(t, new, rows, **kw):
    return [x.tolist() for x in t.extend(ints(new), rows, **kw)]


def state(t):
    return [x.tolist() for x in (t.table, t.lengths, t.free, t.count)]


@pytest.mark.parametrize("sequences,columns,page,steps", [(1, 40, 16, 30), (7, 9, 64, 40), (64, 20, 16, 25), (300, 6, 32, 12),
                                                          (1000, 12, 128, 6)])
def test_batches_in_turn(sequences, columns, page, steps):
    """Tokens given and taken back at random, in batches of one row to many workgroups' rows."""
    from flash_moe_hip.page_table import PageTable

    r = random.Random(sequences)
    t = PageTable.empty(sequences, columns, sequences * columns + 3, page)
    order = list(range(t.pages))
    r.shuffle(order)
    t.free.copy_(ints(order))
    want = Plain(t)
    most = columns * page
    for step in range(steps):
        print(sequences, step, flush=True)
        room = [most - n for n in want.lengths]
        kind = step % 4
        new = [min(x, 1 if kind == 0 else r.choice([0, 0, 1, page, r.randint(0, most)]) if kind == 1 else r.randint(0, 5))
               for x in room]
        rows = sum(new) + r.choice([0, 0, 1, 255, 5000])
        assert extend(t, new, rows) == list(want.extend(new, rows))
        want.check(t)
        keep = [r.choice([n, 2 ** 31 - 1, n - min(n, r.randint(0, 6)), 0 if r.random() < 0.2 else n]) for n in want.lengths]
        t.trim(ints(keep))
        want.trim(keep)
        want.check(t)
    assert t.status() == 0


def test_the_most_sequences():
    from flash_moe_hip.page_table import PageTable

    t = PageTable.empty(8192, 3, 8192 * 3, 16)
    want = Plain(t)
    r = random.Random(3)
    for _ in range(3):
        new = [r.randint(0, 15) for _ in range(8192)]
        assert extend(t, new, sum(new)) == list(want.extend(new, sum(new)))
        want.check(t)
    t.trim(ints([17] * 8192))
    want.trim([17] * 8192)
    want.check(t)
    assert t.status() == 0


def test_a_long_sequence():
    """Many pages at once: several workgroups fill the table's columns and give pages back."""
    from flash_moe_hip.page_table import PageTable

    t = PageTable.empty(2, 20000, 30000, 16)
    want = Plain(t)
    for new in ([5, 200000], [3, 100001], [0, 0]):
        assert extend(t, new, sum(new) + 2) == list(want.extend(new, sum(new) + 2))
    want.check(t)
    before = state(t)
    t.extend(ints([100000, 3]), 100003)
    t.trim(ints(before[1]))
    assert [state(t)[i] for i in (1, 2, 3)] == before[1:]      # (columns past the tokens hold anything)
    t.trim(ints([0, 0]))
    want.trim([0, 0])
    assert int(t.count) == 30000 and t.free.tolist() == want.free
    assert t.status() == 0


@pytest.mark.parametrize("rows", [40, 40000])
def test_calls_that_cannot_be_served_change_nothing(rows):
    from flash_moe_hip.page_table import PageTable

    def fresh(free=10):
        t = PageTable.empty(3, 50, free, 16)
        t.extend(ints([20, 0, 30]), 50)    # four pages
        return t

    none = [[0] * 4, [-1] * rows, [-1] * rows]
    t = fresh()
    before = state(t)
    for new, why in (([1, -1, 0], -9), ([0, 49 * 16 + 17, 0], -9), ([rows + 1 - 7, 7, 0], -9), ([2 ** 31 - 1] * 3, -9),
                     ([12, 16 * 6 + 1, 0], -10)):
        if sum(new) > rows and why == -10:
            continue
        assert extend(t, new, rows) == none and state(t) == before, new
        assert t.status() == why and t.status() == 0, new
    t.trim(ints([1, 1, -1]))
    assert t.status() == -9 and state(t) == before
    if rows > 100:   # and the last free page is given
        assert extend(t, [12, 16 * 6, 2], rows)[0] == [0, 12, 108, 110] and int(t.count) == 0
        assert extend(t, [0, 0, 0], rows)[0] == [0] * 4 and t.status() == 0
    for which, value in ((1, -1), (1, 50 * 16 + 1), (3, -1), (3, 11)):   # lengths and counts out of range
        t = fresh()
        state_of = (t.table, t.lengths, t.free, t.count)
        state_of[which][0] = value
        before = state(t)
        assert extend(t, [0, 1, 0], rows) == none and t.status() == -9
        t.trim(ints([0, 0, 0]))
        assert t.status() == -9 and state(t) == before


def test_pages_that_are_none_are_reported():
    from flash_moe_hip.page_table import PageTable

    t = PageTable.empty(2, 4, 8, 16)
    t.extend(ints([3, 0]), 3)
    t.table[0, 0] = 1000
    _, slots, positions = t.extend(ints([1, 1]), 2)
    assert slots.tolist() == [8 * 16, 16] and positions.tolist() == [3, 0] and t.status() == -9
    t.free[5] = -3
    _, slots, _ = t.extend(ints([0, 16]), 16)
    assert slots.tolist()[-1] == 8 * 16 and t.status() == -9


def test_no_rows():
    from flash_moe_hip.page_table import PageTable

    t = PageTable.empty(5, 2, 9, 16)
    starts, slots, positions = t.extend(ints([0] * 5), 0)
    assert starts.tolist() == [0] * 6 and slots.numel() == positions.numel() == 0 and t.status() == 0
    assert t.extend(ints([0, 0, 1, 0, 0]), 0)[0].tolist() == [0] * 6 and t.status() == -9


def test_captured_replayed_and_other_streams():
    """A captured step replays with other numbers, with eager work between; a side stream."""
    from flash_moe_hip.page_table import PageTable

    t = PageTable.empty(40, 30, 900, 16)
    want = Plain(t)
    new, keep = ints([1] * 40), ints([2 ** 31 - 1] * 40)
    for _ in range(2):   # (what a first call loads)
        t.extend(new, 3000)
        t.trim(ints([0] * 40))
    want.free = t.free.tolist()
    want.table = t.table.tolist()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = t.extend(new, 3000)
        t.trim(keep)
    r = random.Random(1)
    for _ in range(6):
        n = [r.randint(0, 20) for _ in range(40)]
        k = [r.randint(0, 60) for _ in range(40)]
        new.copy_(ints(n))
        keep.copy_(ints(k))
        graph.replay()
        assert [x.tolist() for x in out] == list(want.extend(n, 3000))
        want.trim(k)
        want.check(t)
        assert extend(t, [1] * 40, 40) == list(want.extend([1] * 40, 40))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = t.extend(new, 3000, stream=side)
    t.trim(keep, stream=side)
    side.synchronize()
    assert [x.tolist() for x in got] == list(want.extend(new.tolist(), 3000))
    want.trim(keep.tolist())
    want.check(t)
    assert t.status() == 0


def test_refusals():
    from flash_moe_hip.page_table import PageTable

    t = PageTable.empty(3, 4, 8, 16)
    new = ints([1, 1, 1])
    for args, why in (((new.long(), 3), "new must be"), ((new[:2], 3), "new must be"), ((new.cpu(), 3), "is on cpu"),
                      ((new, -1), "whole number"), ((new, 2 ** 30 + 1), "whole number"), ((new, 3.0), "whole number"),
                      ((new, True), "whole number")):
        with pytest.raises(ValueError, match=why):
            t.extend(*args)
    with pytest.raises(ValueError, match="keep must be"):
        t.trim(new.long())
    with pytest.raises(AttributeError):
        t.table = t.table
    kept = t.lengths.data
    t.lengths.data = kept.long()
    with pytest.raises(ValueError, match="no longer"):
        t.extend(new, 3)
    t.lengths.data = torch.zeros(3, dtype=torch.int32, device="cuda")   # (another place: calls follow)
    assert extend(t, [1, 0, 0], 1)[1] == [0] and not kept.any() and t.lengths.tolist() == [1, 0, 0]


def test_pages_that_are_none_are_reported_by_a_trim():
    """A number in a sequence's columns that is no page goes back where it would, and is reported."""
    from flash_moe_hip.page_table import PageTable

    for tokens in (40, 40000):   # one workgroup's pages, several's
        for bad in (-3, 10 ** 6, 4001):
            t = PageTable.empty(2, 4000, 4001, 16)
            t.extend(ints([tokens, 5]), tokens + 5)
            t.table[0, 1] = bad
            t.trim(ints([2 ** 31 - 1, 0]))
            assert t.status() == 0                       # (no page of that sequence moved)
            t.trim(ints([20, 0]))
            assert t.status() == 0                       # (the column is still the sequence's)
            t.trim(ints([1, 0]))
            assert t.status() == -9 and t.lengths.tolist() == [1, 0] and int(t.count) == 4000
            assert bad in t.free.tolist()


def test_pages_that_are_none_lengths_grow_all_the_same():
    """What a call does that hands out such a number: rows past the cache, the rest as ever."""
    from flash_moe_hip.page_table import PageTable

    t = PageTable.empty(2, 4, 8, 16)
    t.free[6] = 99
    starts, slots, positions = t.extend(ints([20, 3]), 24)
    assert starts.tolist() == [0, 20, 23] and positions.tolist() == [*range(20), 0, 1, 2, -1]
    assert slots.tolist() == [*range(16)] + [8 * 16] * 4 + [32, 33, 34, -1]
    assert t.lengths.tolist() == [20, 3] and int(t.count) == 5 and t.table[0, 1] == 99 and t.status() == -9
