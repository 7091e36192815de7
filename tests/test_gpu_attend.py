"""Attention over the paged cache on the GPU against a plain form in 64 bits,
with the bounds of mixer_reference.attend."""
from __future__ import annotations

import math

import pytest
import torch

import mixer_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.int8, torch.bfloat16),
         (torch.int8, torch.float16)]


def problem(new, lengths, heads, kv_heads, dim, page, cache, qt, seed=0, k_scale=1.0, v_scale=1.0):
    """Queries, a shuffled paged cache with stale places, its tables, and the values it stands for."""
    g = torch.Generator().manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g)

    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=g).to(torch.int32)
    cols = max(max(counts), 1) + 1
    table, used = torch.full((len(lengths), cols), -7, dtype=torch.int32), 0   # (columns past a sequence's end hold anything)
    for b, c in enumerate(counts):
        table[b, :c] = order[used:used + c]
        used += c
    k = [randn(n, kv_heads, dim) * k_scale for n in lengths]
    v = [randn(n, kv_heads, dim) * torch.exp(randn(n, kv_heads, 1)) * v_scale for n in lengths]
    kc, ks, kv = ref.paged(k, table, page, pages, cache)
    vc, vs, vv = ref.paged(v, table, page, pages, cache)
    q = randn(sum(new), heads, dim).to(qt)
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    return dict(q=q, table=table, lengths=torch.tensor(lengths, dtype=torch.int32), starts=starts, k=kv, v=vv,
                cache=[None if t is None else t.cuda() for t in (kc, vc, ks, vs)], new=new)


def cache_of(p):
    from flash_moe_hip.kv_cache import PagedCache

    return PagedCache(*p["cache"])


def call(c, p, single=False, **kw):
    return c.attend(p["q"].cuda(), p["table"].cuda(), p["lengths"].cuda(),
                    starts=None if single else p["starts"].cuda(), **kw)


def check(got, p, scale, cache):
    at = 0
    for b, n in enumerate(p["new"]):
        want, bound = ref.attend(p["q"][at:at + n], p["k"][b], p["v"][b], scale, cache)
        err = (got[at:at + n].cpu().double() - want).abs()
        assert (err <= bound).all(), f"sequence {b}: {float((err / bound).max()):.3g} of the bound"
        at += n


SHAPES = [   # new, lengths, heads, kv_heads, dim, page
    ([1], [1], 1, 1, 64, 16),
    ([5], [5], 4, 2, 128, 16),
    ([3, 0, 17, 1], [3, 0, 40, 65], 8, 2, 64, 32),
    ([70, 33], [70, 161], 5, 1, 128, 16),
    ([40], [300], 6, 6, 64, 1024),
    ([129, 2, 31], [129, 1027, 500], 16, 2, 256, 64),
    ([9, 9], [777, 64], 128, 1, 64, 64),
    ([300], [2300], 4, 1, 128, 128),
]


@pytest.mark.parametrize("cache,qt", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_chunks(shape, cache, qt):
    print(shape, cache, qt, flush=True)
    p = problem(*shape, cache, qt, seed=sum(shape[1]))
    c = cache_of(p)
    check(call(c, p), p, shape[4] ** -0.5, cache)
    assert c.status() == 0


SINGLE = [   # lengths, heads, kv_heads, dim, page
    ([1], 1, 1, 64, 16),
    ([31, 32, 33], 8, 8, 128, 16),
    ([0, 5, 1000], 16, 2, 256, 64),
    ([4099], 16, 1, 128, 64),
    ([2049, 129], 6, 2, 64, 32),
    ([100, 515], 40, 2, 128, 16),       # 20 heads a kv head
    ([20000, 3], 8, 4, 64, 128),
    ([70000], 4, 2, 256, 16),
]


@pytest.mark.parametrize("cache,qt", TYPES, ids=str)
@pytest.mark.parametrize("shape", SINGLE, ids=str)
def test_single_tokens(shape, cache, qt):
    print(shape, cache, qt, flush=True)
    lengths, heads, kv_heads, dim, page = shape
    p = problem([1] * len(lengths), lengths, heads, kv_heads, dim, page, cache, qt, seed=sum(lengths))
    c = cache_of(p)
    got = call(c, p, single=True)
    check(got, p, dim ** -0.5, cache)
    # the same through starts
    check(call(c, p), p, dim ** -0.5, cache)
    assert c.status() == 0


@pytest.mark.parametrize("cache,qt", TYPES, ids=str)
def test_queries_before_the_first_key_are_zeros(cache, qt):
    """More new tokens than cached ones: the first see nothing."""
    p = problem([6, 200], [4, 0], 4, 2, 64, 16, cache, qt)
    c = cache_of(p)
    got = call(c, p).cpu()
    assert not got[:2].any() and not got[6:].any() and c.status() == 0
    p["q"], p["new"] = p["q"][2:6], [4]
    check(got[2:6], p, 64 ** -0.5, cache)


@pytest.mark.parametrize("cache,qt", TYPES, ids=str)
@pytest.mark.parametrize("single", [False, True])
def test_scales_far_from_one(cache, qt, single):
    """Sharp and flat softmaxes, large and small values."""
    n = 1 if single else 37
    for k_scale, v_scale, scale in ((8.0, 1.0, 0.3), (1.0, 200.0, 0.125), (0.01, 2e-3, 0.05), (1.0, 1.0, 1e-6)):
        p = problem([n], [700], 4, 2, 128, 32, cache, qt, seed=5, k_scale=k_scale, v_scale=v_scale)
        c = cache_of(p)
        check(call(c, p, single=single, scale=scale), p, scale, cache)
        assert c.status() == 0


@pytest.mark.parametrize("single", [False, True])
def test_long_rows_and_growing_scores(single):
    """Scores that grow with the position move the reference exponent at every step."""
    n = 1 if single else 20
    p = problem([n], [3000], 2, 1, 64, 64, torch.float16, torch.float16, seed=8)
    ramp = torch.linspace(0.01, 4, 3000).view(-1, 1, 1)
    k = [torch.sign(p["q"][-1:, :1].float()) * ramp]
    kc, _, kv = ref.paged(k, p["table"], 64, p["cache"][0].shape[0], torch.float16)
    p["cache"][0], p["k"] = kc.cuda(), kv
    c = cache_of(p)
    check(call(c, p, single=single), p, 64 ** -0.5, torch.float16)


@pytest.mark.parametrize("cache,qt", TYPES, ids=str)
def test_values_of_later_tokens_do_not_matter(cache, qt):
    """Infinities and NaN in keys and values reach the rows that see them, and no other."""
    lengths, new, page = [150], [100], 16
    p = problem(new, lengths, 4, 2, 64, page, cache, qt, seed=3)
    clean = call(cache_of(p), p).cpu()
    at = {60: math.nan, 90: math.inf, 120: -math.inf}

    def put(t, s, i, x):
        page_, off = int(p["table"][0, i // page]), i % page
        if cache == torch.int8:
            s[page_, 1, off] = math.nan
        else:
            t[page_, 1, off, 11] = x

    for what in (1, 0):   # values, then keys as well
        for i, x in at.items():
            put(p["cache"][what], p["cache"][2 + (what == 1)], i, x)
        c = cache_of(p)
        got = call(c, p).cpu()
        assert c.status() == -4
        first = 60 - 50   # the row of position 60
        torch.testing.assert_close(got[:first], clean[:first], rtol=0, atol=0)
        torch.testing.assert_close(got[:, :2], clean[:, :2], rtol=0, atol=0)   # the other kv head
        assert got[first:, 2:, 11].isnan().all()
        if what == 1 and cache != torch.int8:
            others = [d for d in range(64) if d != 11]
            torch.testing.assert_close(got[:, :, others], clean[:, :, others], rtol=0, atol=0)


def test_an_infinite_value_that_is_seen_is_infinite():
    p = problem([100], [100], 2, 2, 64, 16, torch.bfloat16, torch.bfloat16, seed=3)
    page_, off = int(p["table"][0, 70 // 16]), 70 % 16
    p["cache"][1][page_, 0, off, 5] = -math.inf
    got = call(cache_of(p), p).cpu()
    assert got[:70].isfinite().all() and (got[70:, 0, 5] == -math.inf).all() and got[70:, 1].isfinite().all()


@pytest.mark.parametrize("cache,qt", TYPES, ids=str)
def test_strided_queries_and_tables_rows_of_no_sequence(cache, qt):
    new, lengths = [7, 20], [90, 33]
    p = problem(new, lengths, 4, 2, 128, 16, cache, qt, seed=6)
    c = cache_of(p)
    wide = torch.zeros(40, 4 * 128 + 9, dtype=qt)
    wide[3:30, 5:5 + 512] = p["q"].flatten(1)
    q = wide.cuda()[:, 5:5 + 512].unflatten(1, (4, 128))
    starts = (p["starts"] + 3).cuda()
    table = torch.nn.functional.pad(p["table"], (0, 5)).cuda()[:, :p["table"].shape[1]]
    out = torch.full((40, 4, 128), 7.0, dtype=qt, device="cuda")
    got = c.attend(q, table, p["lengths"].cuda(), starts=starts, out=out)
    assert got is out and (out[:3] == 7).all() and (out[30:] == 7).all()
    check(out[3:30], p, 128 ** -0.5, cache)
    # the same with the keys split over workgroups
    p = problem([5, 2], [9000, 4000], 4, 2, 128, 16, cache, qt, seed=6)
    c = cache_of(p)
    q = torch.zeros(12, 4, 128, dtype=qt)
    q[2:9] = p["q"]
    out = torch.full((12, 4, 128), 7.0, dtype=qt, device="cuda")
    c.attend(q.cuda(), p["table"].cuda(), p["lengths"].cuda(), starts=(p["starts"] + 2).cuda(), out=out)
    assert (out[:2] == 7).all() and (out[9:] == 7).all()
    check(out[2:9], p, 128 ** -0.5, cache)
    assert c.status() == 0


@pytest.mark.parametrize("single", [False, True])
def test_bad_pages_lengths_and_starts_are_reported(single):
    def fresh():
        return problem([1, 1], [300, 40], 4, 2, 64, 16, torch.float16, torch.float16)

    p = fresh()
    p["table"][0, 3] = 10 ** 6
    c = cache_of(p)
    call(c, p, single=single)
    assert c.status() == -9
    p = fresh()
    p["lengths"][1] = 10 ** 6
    p["table"].clamp_(min=0)
    c = cache_of(p)
    call(c, p, single=single)
    assert c.status() in (-9, -4)
    if not single:
        for starts in ([0, 5, 2], [-3, 1, 2], [0, 1, 9], [2, 0, 1]):
            p = fresh()
            p["starts"] = torch.tensor(starts, dtype=torch.int32)
            c = cache_of(p)
            call(c, p)
            assert c.status() == -9, starts


def test_many_sequences():
    """More sequences than a wavefront has lanes, some without queries, some without keys."""
    new = [i % 4 for i in range(150)]
    lengths = [n + (i * 37) % 200 if i % 7 else n for i, n in enumerate(new)]
    p = problem(new, lengths, 2, 1, 64, 16, torch.bfloat16, torch.bfloat16, seed=2)
    c = cache_of(p)
    check(call(c, p), p, 64 ** -0.5, torch.bfloat16)
    p = problem([1] * 150, [n + 1 for n in lengths], 2, 1, 64, 16, torch.bfloat16, torch.bfloat16, seed=2)
    c = cache_of(p)
    check(call(c, p, single=True), p, 64 ** -0.5, torch.bfloat16)
    assert c.status() == 0


def test_no_queries():
    p = problem([0], [30], 4, 2, 64, 16, torch.float16, torch.float16)
    c = cache_of(p)
    assert call(c, p).shape == (0, 4, 64)
    assert c.status() == 0


@pytest.mark.parametrize("single", [False, True])
def test_captured_replayed_and_other_streams(single):
    """Two captured calls on one cache, replayed in turn with eager work between, and a side stream."""
    n = 1 if single else 6
    p = problem([n, n], [5000, 700], 8, 2, 128, 64, torch.int8, torch.bfloat16, seed=4)
    c = cache_of(p)
    q, table, lengths, starts = (t.cuda() for t in (p["q"], p["table"], p["lengths"], p["starts"]))
    kw = dict(starts=None if single else starts)
    other = torch.randn_like(q.float()).to(q.dtype)
    want, want2 = c.attend(q, table, lengths, **kw), c.attend(other, table, lengths, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = c.attend(q, table, lengths, stream=side, **kw)
    side.synchronize()
    assert torch.equal(got, want)
    graphs = []
    for x in (q, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = c.attend(x, table, lengths, **kw)
        graphs.append((graph, y))
    for _ in range(4):
        for (graph, y), w in zip(graphs, (want, want2)):
            y.zero_()
            graph.replay()
            assert torch.equal(c.attend(other, table, lengths, **kw), want2)
            assert torch.equal(y, w)
    assert c.status() == 0


@pytest.mark.parametrize("cache,qt,heads,kv_heads,dim", [
    (torch.float16, torch.float16, 32, 4, 64), (torch.int8, torch.bfloat16, 32, 4, 64),
    (torch.bfloat16, torch.bfloat16, 24, 8, 128), (torch.int8, torch.float16, 32, 4, 256)], ids=str)
def test_a_prompt_of_thousands_of_keys_a_workgroup(cache, qt, heads, kv_heads, dim):
    """Enough rows that the keys are not split: a workgroup goes through more pages than a wavefront has lanes."""
    p = problem([2311], [2400], heads, kv_heads, dim, 16, cache, qt, seed=1)
    c = cache_of(p)
    got = call(c, p)
    assert c.status() == 0
    # some of the rows, the first and the last among them
    keep = torch.tensor([0, 1, 700, 1023, 1024, 1500, 2048, 2309, 2310])
    for i in keep.tolist():
        n = 2400 - 2310 + i
        want, bound = ref.attend(p["q"][i:i + 1], p["k"][0][:n], p["v"][0][:n], dim ** -0.5, cache)
        assert ((got[i:i + 1].cpu().double() - want).abs() <= bound).all(), i


@pytest.mark.parametrize("cache,qt", TYPES, ids=str)
def test_single_tokens_of_thousands_of_keys_a_workgroup(cache, qt):
    """Enough sequences that the keys are not split (they share pages): a wavefront goes through more blocks than it has
    lanes."""
    p = problem([1], [9001], 8, 8, 64, 16, cache, qt, seed=2)
    c = cache_of(p)
    seqs = 600
    g = torch.Generator().manual_seed(4)
    q = torch.randn(seqs, 8, 64, generator=g).to(qt)
    lengths = torch.full((seqs,), 9001, dtype=torch.int32)
    lengths[5], lengths[77], lengths[599] = 8193, 0, 8190
    table = p["table"].expand(seqs, -1).contiguous()
    got = c.attend(q.cuda(), table.cuda(), lengths.cuda()).cpu()
    assert c.status() == 0 and not got[77].any()
    for b in (0, 5, 300, 599):
        n = int(lengths[b])
        want, bound = ref.attend(q[b:b + 1], p["k"][0][:n], p["v"][0][:n], 64 ** -0.5, cache)
        assert ((got[b:b + 1].double() - want).abs() <= bound).all(), b


@pytest.mark.parametrize("single", [False, True])
def test_pages_past_32_bits_of_offset(single):
    from flash_moe_hip.kv_cache import PagedCache

    pages = 2 ** 32 // (64 * 128) + 9   # elements past 2^32
    n = 1 if single else 7
    p = problem([n], [200], 2, 1, 128, 64, torch.int8, torch.bfloat16, seed=3)
    k = torch.empty(pages, 1, 64, 128, dtype=torch.int8, device="cuda")
    scale = torch.empty(pages, 1, 64, device="cuda")
    big = PagedCache(k, torch.empty_like(k), scale, torch.empty_like(scale))
    far = torch.tensor([[pages - 1, pages - 3, 0, pages // 2]], dtype=torch.int32)
    for b in range(4):
        for t, s in zip((big.k, big.v, big.k_scale, big.v_scale), p["cache"]):
            t[int(far[0, b])] = s[int(p["table"][0, b])]
    p["table"] = far
    check(call(big, p, single=single), p, 128 ** -0.5, torch.int8)
    assert big.status() == 0


def test_refusals():
    """Arguments the Python call refuses before anything is enqueued."""
    p = problem([2, 3], [30, 40], 4, 2, 64, 16, torch.float16, torch.float16)
    c = cache_of(p)
    q, table, lengths, starts = (t.cuda() for t in (p["q"], p["table"], p["lengths"], p["starts"]))
    bad = [
        ((q.float(), table, lengths, starts), {}, "expected one of"),
        ((q.bfloat16(), table, lengths, starts), {}, "expected one of"),
        ((q[:, :3], table, lengths, starts), {}, "times the cache"),
        ((q[:, :, :32], table, lengths, starts), {}, "shape"),
        ((q.cpu(), table, lengths, starts), {}, "is on cpu"),
        ((q, table.long(), lengths, starts), {}, "page_table"),
        ((q, table.cpu(), lengths, starts), {}, "page_table"),
        ((q, table[:, :0], lengths, starts), {}, "no columns"),
        ((q, table, lengths.long(), starts), {}, "lengths"),
        ((q, table, lengths, starts[:2]), {}, "starts"),
        ((q, table, lengths, None), {}, "one query a sequence"),
        ((q, table, lengths, starts), dict(scale=0.0), "scale"),
        ((q, table, lengths, starts), dict(scale=math.nan), "scale"),
        ((q, table, lengths, starts), dict(out=torch.empty_like(q).float()), "expected one of"),
        ((q, table, lengths, starts), dict(out=torch.empty(5, 4, 128, dtype=q.dtype, device="cuda")[:, :, :64]),
         "contiguous"),
        ((q.clone().requires_grad_(), table, lengths, starts), {}, "no backward"),
    ]
    for args, kw, why in bad:
        with pytest.raises(ValueError, match=why):
            c.attend(*args, **kw)
    rows, slots = torch.zeros(3, 2, 64, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for args, why in (((rows, rows.half(), slots), "expected one of"), ((rows, rows[:2], slots), "shape"),
                      ((rows, rows, slots.int()), "slots"), ((rows.double(), rows.double(), slots), "expected one of"),
                      ((rows.transpose(0, 2), rows, slots), "shape"), ((rows, rows, slots.cpu()), "is on cpu")):
        with pytest.raises(ValueError, match=why):
            c.write(*args)
    with pytest.raises(ValueError, match="rows are read"):
        c.read(slots, dtype=torch.int8)
    assert c.status() == 0


def with_zero_rows(p, rows, lead, zeros, scale, page):
    """The problem's int8 cache anew from `rows` (keys and values of one sequence), the value rows `zeros` all
    zero and their keys ahead of the others by `lead` in every score: channel 0 of every query is 8, and of
    these keys alone it is not 0."""
    k, v = rows
    k[:, :, 0] = 0
    k[zeros], v[zeros] = 0, 0
    k[zeros, :, 0] = lead / (8 * scale)
    p["q"][:, :, 0] = 8
    pages = p["cache"][0].shape[0]
    kc, ks, p["k"] = ref.paged([k], p["table"], page, pages, torch.int8)
    vc, vs, p["v"] = ref.paged([v], p["table"], page, pages, torch.int8)
    p["cache"] = [t.cuda() for t in (kc, vc, ks, vs)]


@pytest.mark.parametrize("qt", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("new,length,dim", [(1, 700, 64), (1, 5000, 128), (1, 300, 256), (37, 700, 64), (20, 1024, 128),
                                            (3, 5000, 256)])
def test_zero_value_rows_weigh_in_the_softmax_only(new, length, dim, qt):
    """Value rows of zeros in an int8 cache, with scores level with the others' and ahead of them, beside small and
    large values: the other rows' products keep their bits."""
    scale = dim ** -0.5
    g = torch.Generator().manual_seed(length)
    for v_scale in (1.0, 0.05, 1e-3, 1e-5, 1e-8, 1e-12, 1e3):
        for lead in (0.0, 5.0, 15.0):
            print(new, length, dim, qt, v_scale, lead, flush=True)
            p = problem([new], [length], 4, 2, dim, 32, torch.int8, qt, seed=length)
            k, v = (torch.randn(length, 2, dim, generator=g) for _ in range(2))
            zeros = torch.tensor([0, 1, length // 2, length - new])
            with_zero_rows(p, (k, v * v_scale), lead, zeros, scale, 32)
            c = cache_of(p)
            got = call(c, p, single=new == 1)
            if qt == torch.float16 and v_scale < 1e-6:   # (FP16 outputs are zeros then: nothing to see)
                continue
            check(got, p, scale, torch.int8)
            assert c.status() == 0


@pytest.mark.parametrize("new", [1, 9])
def test_values_of_zero_alone(new):
    p = problem([new], [3000], 4, 2, 64, 32, torch.int8, torch.bfloat16, seed=1)
    g = torch.Generator().manual_seed(1)
    with_zero_rows(p, [torch.randn(3000, 2, 64, generator=g) for _ in range(2)], 1.0, torch.arange(3000), 0.125, 32)
    c = cache_of(p)
    assert not call(c, p, single=new == 1).any() and c.status() == 0


@pytest.mark.parametrize("new,length", [(1, 40), (1, 5000), (9, 40), (9, 5000)])
@pytest.mark.parametrize("qt,value", [(torch.float16, 1e5), (torch.bfloat16, 3.399e38)], ids=str)
def test_outputs_their_type_cannot_hold_are_reported(new, length, qt, value):
    """FP32 sums that are finite and round to infinity, whole and joined from splits."""
    p = problem([new], [length], 2, 1, 64, 32, torch.int8, qt, seed=2)
    vc, vs = p["cache"][1], p["cache"][3]
    vc.fill_(100)
    vc[..., 3] = 127   # channel 3 alone is the value
    vs.fill_(value / 127)
    c = cache_of(p)
    got = call(c, p, single=new == 1)
    assert got[..., 3].isinf().all() and c.status() == -4
    vs.fill_(6e4 / 127)
    assert call(c, p, single=new == 1).isfinite().all() and c.status() == 0


@pytest.mark.parametrize("what", [math.inf, math.nan])
@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("length", [330, 9000])
def test_a_seen_value_that_is_not_finite_is_not_lost_where_its_weight_underflows(length, new, what):
    """Keys far below the others in score, in one workgroup's share with them or in shares of their own."""
    p = problem([new], [length], 2, 1, 64, 64, torch.bfloat16, torch.bfloat16, seed=4)
    p["q"][:, :, 0] = 64
    kc, vc = p["cache"][:2]
    kc[..., 0] = 0
    for page_ in p["table"][0, :length // 320].tolist():   # the first fifth of the keys: scores of -4096 or so
        kc[page_, 0, :, 0] = -64
    vc[int(p["table"][0, 0]), 0, 3, 5] = what
    c = cache_of(p)
    got = call(c, p, single=new == 1, scale=1.0)
    assert not got[..., 5].isfinite().any() and c.status() == -4
    others = [d for d in range(64) if d != 5]
    assert got[..., others].isfinite().all()
