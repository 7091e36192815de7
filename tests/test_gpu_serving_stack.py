"""An attention layer as a serving program runs it: page tables extended on the device, queries and keys normed and
rotated, rows written into the paged cache, attention over it; batches of prompts, drafts and single tokens, padded, with
drafts taken back, sequences that end and others that take their pages."""
from __future__ import annotations

import pytest
import torch

import f4_reference as f4
import mixer_reference as ref

pytestmark = pytest.mark.gpu

SEQS, HEADS, KV_HEADS, DIM, PAGE = 5, 8, 2, 128, 16
CACHES = [f4.CODES, torch.bfloat16, torch.int8]


class Layer:
    def __init__(self, cache_type, pages=120, columns=40):
        from flash_moe_hip.kv_cache import PagedCache
        from flash_moe_hip.page_table import PageTable
        from flash_moe_hip.rotary import Rotary

        g = torch.Generator(device="cuda").manual_seed(1)
        self.table = PageTable.empty(SEQS, columns, pages, PAGE)
        self.table.free.copy_(torch.randperm(pages, generator=g, device="cuda"))
        self.cache = PagedCache.empty(pages, KV_HEADS, DIM, PAGE, cache_type)
        self.rotary = Rotary(DIM, 64, base=1e6, scaling=dict(kind="yarn", factor=8.0, original=4096))
        self.weights = [1 + 0.2 * torch.randn(DIM, generator=g, device="cuda") for _ in range(2)]

    def run(self, qkv, new):
        """qkv [rows, HEADS + 2 KV_HEADS, DIM], a projection's rows, `new` int32 new tokens of each sequence."""
        q, k, v = qkv.split([HEADS, KV_HEADS, KV_HEADS], 1)
        starts, slots, positions = self.table.extend(new, qkv.shape[0])
        q, k = self.rotary.apply(q, k, positions, q_weight=self.weights[0], k_weight=self.weights[1])
        self.cache.write(k, v, slots)
        out = self.cache.attend(q, self.table.table, self.table.lengths, starts)
        return out, (q, k, v, starts, slots, positions)

    def check(self):
        assert self.table.status() == 0 and self.rotary.status() == 0 and self.cache.status() == 0


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def rows(n, seed):
    return torch.randn(n, HEADS + 2 * KV_HEADS, DIM, generator=torch.Generator(device="cuda").manual_seed(seed),
                       device="cuda").bfloat16()


def stored(x, cache_type):
    """What a cache of this type gives back of rows [tokens, heads, dim], float64."""
    x = x.cpu()
    if cache_type == f4.CODES:
        return f4.quantized(x)[2]
    if cache_type == torch.int8:
        codes, scale = ref.quantized(x)
        return codes.double() * scale.double().unsqueeze(-1)
    return x.to(cache_type).double()


@pytest.mark.parametrize("cache_type", CACHES, ids=str)
def test_batches_of_all_kinds(cache_type):
    layer = Layer(cache_type)
    keys = [torch.zeros(0, KV_HEADS, DIM, dtype=torch.float64) for _ in range(SEQS)]
    values = [t.clone() for t in keys]
    steps = [   # new tokens of each sequence, rows of padding, tokens taken back afterwards
        ([70, 0, 3, 33, 0], 6, [0] * 5),       # prompts
        ([1, 1, 1, 1, 0], 0, [0] * 5),
        ([5, 5, 5, 5, 0], 12, [2, 4, 5, 0, 0]),   # drafts, some of them kept
        ([1, 300, 1, 1, 1], 0, [0] * 5),       # a prompt beside single tokens
        ([0, 0, 1, 0, 0], 7, [500, 0, 0, 0, 0]),   # one sequence ends
        ([200, 3, 1, 90, 40], 1, [0] * 5),     # and another takes its place
        ([1, 1, 1, 1, 1], 0, [0] * 5),
    ]
    for i, (new, padded, back) in enumerate(steps):
        print(i, new, padded, back, flush=True)
        n = sum(new)
        out, (q, k, v, starts, slots, positions) = layer.run(rows(n + padded, i), ints(new))
        layer.check()
        assert starts.tolist() == torch.tensor([0] + new).cumsum(0).tolist() and (slots[n:] == -1).all()
        got_k, got_v = (t[:n].cpu().double() for t in layer.cache.read(slots))
        new_k, new_v = stored(k[:n], cache_type), stored(v[:n], cache_type)
        exact = 0.0 if cache_type != torch.int8 else 2.0 ** -24   # (a code times its scale, rounded to FP32)
        assert ((got_k - new_k).abs() <= exact * new_k.abs()).all() and ((got_v - new_v).abs() <= exact * new_v.abs()).all()
        at = 0
        for b, a in enumerate(new):
            assert positions[at:at + a].tolist() == list(range(len(keys[b]), len(keys[b]) + a))
            keys[b] = torch.cat([keys[b], new_k[at:at + a]])
            values[b] = torch.cat([values[b], new_v[at:at + a]])
            want, bound = ref.attend(q[at:at + a].cpu(), keys[b], values[b], DIM ** -0.5,
                                     torch.bfloat16 if cache_type == torch.bfloat16 else torch.int8)
            assert ((out[at:at + a].cpu().double() - want).abs() <= bound).all(), (i, b)
            at += a
        keep = [max(len(t) - x, 0) for t, x in zip(keys, back)]
        layer.table.trim(ints(keep))
        keys, values = [[t[:m] for t, m in zip(x, keep)] for x in (keys, values)]
        assert layer.table.lengths.tolist() == keep
    layer.check()


@pytest.mark.parametrize("cache_type", [f4.CODES, torch.bfloat16], ids=str)
def test_a_captured_step_replays(cache_type):
    """One captured step, drafts taken back within it, against eager ones: the same bits, tables and free pages."""
    layers = [Layer(cache_type) for _ in range(2)]
    for layer in layers:
        layer.run(rows(100, 1), ints([40, 20, 0, 7, 33]))
    eager, other = layers
    new, keep, qkv = ints([1] * 5), ints([2 ** 31 - 1] * 5), rows(20, 2)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y, _ = other.run(qkv, new)
        other.table.trim(keep)
    for step, (n, m) in enumerate([([1] * 5, [1000] * 5), ([4] * 5, [44, 23, 5, 11, 36]), ([0, 0, 16, 0, 4], [0, 1000, 12, 9, 38]),
                                   ([5, 0, 1, 0, 1], [1000] * 5), ([1] * 5, [1000] * 5)]):
        x = rows(20, 10 + step)
        new.copy_(ints(n))
        keep.copy_(ints(m))
        qkv.copy_(x)
        y.zero_()
        graph.replay()
        want, (_, _, _, starts, slots, _) = eager.run(x, ints(n))
        eager.table.trim(ints(m))
        assert torch.equal(y[:sum(n)], want[:sum(n)]), step
        assert eager.table.lengths.tolist() == other.table.lengths.tolist() and torch.equal(eager.table.free, other.table.free)
        assert int(eager.table.count) == int(other.table.count)
        assert all(torch.equal(a, b) for a, b in zip(eager.cache.read(slots), other.cache.read(slots)))
    eager.check()
    other.check()


def test_a_step_without_free_pages_leaves_everything():
    """The tables refuse the batch on the device, its rows go nowhere, and the layer goes on."""
    layer = Layer(f4.CODES, pages=8)
    layer.run(rows(60, 1), ints([16, 16, 16, 0, 12]))
    layer.check()
    before = [t.view(torch.uint8).clone() for t in (layer.cache.k, layer.cache.v_scale)]
    _, (_, _, _, starts, slots, _) = layer.run(rows(90, 2), ints([1, 1, 0, 80, 0]))
    assert not starts.any() and (slots == -1).all() and layer.table.status() == -10 and layer.cache.status() == 0
    assert all(torch.equal(a, t.view(torch.uint8)) for a, t in zip(before, (layer.cache.k, layer.cache.v_scale)))
    assert layer.table.lengths.tolist() == [16, 16, 16, 0, 12]
    layer.run(rows(2, 3), ints([1, 1, 0, 0, 0]))
    layer.check()


@pytest.mark.parametrize("cache_type", CACHES, ids=str)
def test_rows_of_padding_hold_anything(cache_type):
    """Rows behind the last sequence that a layer before left unwritten: real rows are the same, nothing is reported."""
    clean, other = Layer(cache_type), Layer(cache_type)
    for i, new in enumerate(([30, 0, 7, 200, 1], [1, 1, 1, 1, 1], [4, 0, 5, 3, 0])):
        n = sum(new)
        x, y = rows(n + 19, i), rows(n + 19, i)
        y[n:n + 7], y[n + 7:] = float("nan"), float("inf")
        want, got = clean.run(x, ints(new))[0], other.run(y, ints(new))[0]
        assert torch.equal(got[:n], want[:n])
        other.check()
    # a row of a sequence is still reported
    x = rows(5, 9)
    x[2, 1, 70] = float("inf")
    other.run(x, ints([1] * 5))
    assert other.rotary.status() == -4 and other.table.status() == 0
