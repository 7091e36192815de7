"""The 4-bit paged cache on the GPU: rows quantized and read back, attention over it against 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import f4_reference as f4
import mixer_reference as ref

pytestmark = pytest.mark.gpu

ROWS = [torch.float32, torch.float16, torch.bfloat16]
QUERIES = [torch.bfloat16, torch.float16]


def rows(tokens, heads, dim, dtype, seed, strided=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, dim, generator=g) * torch.exp(2 * torch.randn(tokens, heads, dim // 16, 1, generator=g)).expand(
        tokens, heads, dim // 16, 16).flatten(2)
    x = x.to(dtype)
    if strided:   # part of a wider row, off the 16-byte grid
        wide = torch.zeros(tokens, heads * dim + 7, dtype=dtype)
        wide[:, 3:3 + heads * dim] = x.flatten(1)
        return wide.cuda()[:, 3:3 + heads * dim].unflatten(1, (heads, dim))
    return x.cuda()


def flat(t):
    """Of a cache's tensor, the rows of each slot as bytes [slots, kv_heads, ...]."""
    return t.view(torch.uint8).cpu().transpose(1, 2).flatten(0, 1)


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("dtype", ROWS, ids=str)
@pytest.mark.parametrize("tokens,heads,dim,page", [(1, 1, 64, 16), (37, 3, 128, 16), (130, 2, 256, 64), (65, 8, 64, 1024)])
def test_write_and_read(tokens, heads, dim, page, dtype, strided):
    from flash_moe_hip.kv_cache import PagedCache

    print(tokens, heads, dim, page, dtype, strided, flush=True)
    pages = -(-tokens // page) + 2
    c = PagedCache.empty(pages, heads, dim, page, f4.CODES)
    assert c.head_dim == dim and not c.read(torch.arange(pages * page).cuda())[0].any()
    k, v = rows(tokens, heads, dim, dtype, 1, strided), rows(tokens, heads, dim, dtype, 2, strided)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(3))[:tokens]
    slots[::5] = -1
    c.write(k, v, slots.cuda())
    assert c.status() == 0
    kept = slots >= 0
    untouched = torch.ones(pages * page, dtype=torch.bool)
    untouched[slots[kept]] = False
    for t, s, x in ((c.k, c.k_scale, k), (c.v, c.v_scale, v)):
        codes, scale, _ = f4.quantized(x.cpu()[kept])
        assert torch.equal(flat(t)[slots[kept]], codes) and torch.equal(flat(s)[slots[kept]], scale)
        assert not flat(t)[untouched].any() and not flat(s)[untouched].any()
    for out in ROWS:
        for got, x in zip(c.read(slots.cuda(), dtype=out), (k, v)):
            assert got.dtype == out and not got.cpu()[~kept].any()
            assert torch.equal(got.cpu()[kept], f4.quantized(x.cpu()[kept])[2].to(out))   # (exact in every type)
    assert c.status() == 0 and c.read(slots.cuda())[0].dtype == torch.float32


@pytest.mark.parametrize("tokens,heads,dim", [(8195, 8, 128), (32773, 4, 64), (4101, 8, 256)])
def test_many_rows(tokens, heads, dim):
    """Enough rows that a lane takes several, and a ragged end."""
    from flash_moe_hip.kv_cache import PagedCache

    c = PagedCache.empty(-(-tokens // 32) + 1, heads, dim, 32, f4.CODES)
    k, v = rows(tokens, heads, dim, torch.bfloat16, 1), rows(tokens, heads, dim, torch.bfloat16, 2)
    slots = torch.randperm(c.pages * 32, generator=torch.Generator().manual_seed(5))[:tokens]
    slots[-5:-1] = -1
    kept = slots >= 0
    c.write(k, v, slots.cuda())
    past = False   # (so many draws of such sizes pass 57344 here and there)
    for got, x in zip(c.read(slots.cuda(), torch.bfloat16), (k, v)):
        want = f4.quantized(x.cpu()[kept])[2]
        torch.testing.assert_close(got.cpu()[kept].double(), want, rtol=0, atol=0, equal_nan=True)
        assert not got.cpu()[~kept].any()
        past |= bool(want.isnan().any())
    assert c.status() == (-4 if past else 0)
    free = torch.ones(c.pages * 32, dtype=torch.bool)
    free[slots[kept]] = False
    assert not flat(c.k)[free].any() and not flat(c.v_scale)[free].any()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_edge_blocks(dim):
    """Ties, the borders of scales, the smallest and the largest, blocks that are not finite."""
    from flash_moe_hip.kv_cache import PagedCache

    x = torch.zeros(12, 1, dim)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    x[1, 0, :16] = torch.cat([ties, -ties])
    x[2, 0, :24] = torch.cat([torch.nextafter(ties, torch.tensor(0.0)), torch.nextafter(ties, torch.tensor(9.0)), ties])
    x[3, 0, :2] = torch.tensor([7.0, 0.5])                                     # the next scale: 8, 0
    x[4, 0, :2] = torch.tensor([float(torch.nextafter(torch.tensor(7.0), torch.tensor(0.0))), 0.5])
    x[5, 0, :4] = torch.tensor([2.0 ** -24, -2.0 ** -25, 3 * 2.0 ** -25, 1e-40])   # the least numbers
    x[6, 0, 32:] = 2.0 ** -150
    x[7, 0, :3] = torch.tensor([57343.99, -1.0, 4096.0])
    x[8, 0, 5] = 57344.0                    # past the largest scale
    x[9, 0, 40] = math.inf
    x[10, 0, 1], x[10, 0, 2] = math.nan, -math.inf
    x[11, 0] = torch.linspace(-3e38, 3e38, dim)
    c = PagedCache.empty(2, 1, dim, 16, f4.CODES)
    slots = torch.arange(12).cuda()
    c.write(x.cuda(), -x.cuda(), slots)
    assert c.status() == -4 and c.status() == 0
    k, v = (t.cpu().double() for t in c.read(slots))
    for got, x in ((k, x), (v, -x)):
        torch.testing.assert_close(got, f4.quantized(x)[2], rtol=0, atol=0, equal_nan=True)
    assert k[8, 0, :32].isnan().all() and not k[8, 0, 32:].any() and k[9, 0, 32:64].isnan().all()
    assert k[3, 0, 0] == 8 and k[4, 0, 0] == 6 and k[5, 0, 0] == 2.0 ** -24
    c.read(slots, torch.float16)
    assert c.status() == 0                  # (what is stored so is no fault of a read)


def test_slots_past_the_cache_are_skipped_and_reported():
    from flash_moe_hip.kv_cache import PagedCache

    c = PagedCache.empty(2, 2, 64, 16, f4.CODES)
    x = rows(3, 2, 64, torch.bfloat16, 1)
    slots = torch.tensor([32, 5, 2 ** 40]).cuda()
    c.write(x, x, slots)
    assert c.status() == -9 and c.status() == 0
    k, v = c.read(slots, torch.bfloat16)
    assert c.status() == -9 and not k[0].any() and not v[2].any() and k[1].any()


def problem(new, lengths, heads, kv_heads, dim, page, qt, seed=0, k_scale=1.0, v_scale=1.0):
    """Queries, a shuffled paged cache with stale places, its tables, and the values it stands for."""
    g = torch.Generator().manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g)

    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table, used = torch.full((len(lengths), max(max(counts), 1) + 1), -7, dtype=torch.int32), 0
    for b, c in enumerate(counts):
        table[b, :c] = order[used:used + c]
        used += c
    k = [randn(n, kv_heads, dim) * k_scale for n in lengths]
    v = [randn(n, kv_heads, dim) * torch.exp(randn(n, kv_heads, 1)) * v_scale for n in lengths]
    kc, ks, kv = f4.paged(k, table, page, pages)
    vc, vs, vv = f4.paged(v, table, page, pages)
    return dict(q=randn(sum(new), heads, dim).to(qt), table=table, lengths=torch.tensor(lengths, dtype=torch.int32),
                starts=torch.tensor([0] + new).cumsum(0).to(torch.int32), k=kv, v=vv, held=[kc, vc, ks, vs], new=new)


def call(c, p, single=False, **kw):
    return c.attend(p["q"].cuda(), p["table"].cuda(), p["lengths"].cuda(),
                    starts=None if single else p["starts"].cuda(), **kw)


def check(got, p, scale):
    """Within the bounds of attention over an 8-bit cache: FP16 products of exact operands, FP16 probabilities."""
    at = 0
    for b, n in enumerate(p["new"]):
        want, bound = ref.attend(p["q"][at:at + n], p["k"][b], p["v"][b], scale, torch.int8)
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
    ([7, 3], [9000, 4000], 4, 2, 128, 16),   # keys split over workgroups
    ([200, 90], [5000, 700], 4, 2, 64, 64),
    ([130, 131, 7], [2000, 3100, 900], 8, 1, 256, 16),
]


@pytest.mark.parametrize("qt", QUERIES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_chunks(shape, qt):
    print(shape, qt, flush=True)
    p = problem(*shape, qt, seed=sum(shape[1]))
    c = f4.cache(*p["held"])
    check(call(c, p), p, shape[4] ** -0.5)
    assert c.status() == 0


SINGLE = [   # lengths, heads, kv_heads, dim, page
    ([1], 1, 1, 64, 16),
    ([31, 32, 33], 8, 8, 128, 16),
    ([15, 16, 17, 48], 4, 2, 64, 16),
    ([0, 5, 1000], 16, 2, 256, 64),
    ([4099], 16, 1, 128, 64),
    ([2049, 129], 6, 2, 64, 32),
    ([100, 515], 40, 2, 128, 16),       # 20 heads a kv head
    ([20000, 3], 8, 4, 64, 128),
    ([70000], 4, 2, 256, 16),
]


@pytest.mark.parametrize("qt", QUERIES, ids=str)
@pytest.mark.parametrize("shape", SINGLE, ids=str)
def test_single_tokens(shape, qt):
    print(shape, qt, flush=True)
    lengths, heads, kv_heads, dim, page = shape
    p = problem([1] * len(lengths), lengths, heads, kv_heads, dim, page, qt, seed=sum(lengths))
    c = f4.cache(*p["held"])
    check(call(c, p, single=True), p, dim ** -0.5)
    check(call(c, p), p, dim ** -0.5)   # the same through starts
    assert c.status() == 0


@pytest.mark.parametrize("qt", QUERIES, ids=str)
def test_queries_before_the_first_key_are_zeros(qt):
    p = problem([6, 200], [4, 0], 4, 2, 64, 16, qt)
    c = f4.cache(*p["held"])
    got = call(c, p).cpu()
    assert not got[:2].any() and not got[6:].any() and c.status() == 0
    p["q"], p["new"] = p["q"][2:6], [4]
    check(got[2:6], p, 64 ** -0.5)


@pytest.mark.parametrize("qt", QUERIES, ids=str)
@pytest.mark.parametrize("single", [False, True])
def test_scales_far_from_one(qt, single):
    """Sharp and flat softmaxes, values from FP16's least to its largest numbers, queries of zeros."""
    n = 1 if single else 37
    for k_scale, v_scale, scale in ((8.0, 1.0, 0.3), (1.0, 200.0, 0.125), (0.01, 2e-3, 0.05), (1.0, 1.0, 1e-6),
                                    (1.0, 1e-5, 0.1), (1e-4, 1.0, 30.0), (1.0, 1.0, 1e-30)):
        p = problem([n], [700], 4, 2, 128, 32, qt, seed=5, k_scale=k_scale, v_scale=v_scale)
        p["q"][:, 1] = 0
        c = f4.cache(*p["held"])
        check(call(c, p, single=single, scale=scale), p, scale)
        assert c.status() == 0


@pytest.mark.parametrize("single", [False, True])
def test_scores_that_grow(single):
    """Scores that grow with the position move the reference exponent at every step."""
    p = problem([1 if single else 20], [3000], 2, 1, 64, 64, torch.float16, seed=8)
    k = [torch.sign(p["q"][-1:, :1].float()) * torch.linspace(0.01, 4, 3000).view(-1, 1, 1)]
    p["held"][0], p["held"][2], p["k"] = f4.paged(k, p["table"], 64, p["held"][0].shape[0])
    check(call(f4.cache(*p["held"]), p, single=single), p, 64 ** -0.5)


@pytest.mark.parametrize("qt", QUERIES, ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_values_of_later_tokens_do_not_matter(dim, qt):
    """Blocks that are not finite, in keys and values, reach the rows that see them, and no other."""
    page = 16
    p = problem([100], [150], 4, 2, dim, page, qt, seed=3)
    clean = call(f4.cache(*p["held"]), p).cpu()
    for what in (1, 0):   # values, then keys as well
        for i in (60, 90, 120):
            p["held"][2 + what][int(p["table"][0, i // page]), 1, i % page, 1] = 255
        c = f4.cache(*p["held"])
        got = call(c, p).cpu()
        assert c.status() == -4
        first = 60 - 50   # the row of position 60
        torch.testing.assert_close(got[:first], clean[:first], rtol=0, atol=0)
        torch.testing.assert_close(got[:, :2], clean[:, :2], rtol=0, atol=0)   # the other kv head
        assert got[first:, 2:, 32:64].isnan().all()
        if what == 1:
            others = [d for d in range(dim) if not 32 <= d < 64]
            torch.testing.assert_close(got[:, :, others], clean[:, :, others], rtol=0, atol=0)


@pytest.mark.parametrize("new,length", [(1, 330), (3, 330), (1, 9000), (3, 9000)])
def test_a_seen_block_that_is_not_finite_is_not_lost_where_its_weight_underflows(new, length):
    p = problem([new], [length], 2, 1, 64, 64, torch.bfloat16, seed=4)
    p["q"][:, :, 0] = 64
    kc, vc, ks, vs = p["held"]
    kc[..., 0] &= 0xf0                                     # channel 0 of every key is 0
    for page_ in p["table"][0, :length // 320].tolist():   # and of the first fifth of them far below
        kc[page_, 0, :, 0] |= 0xf
        ks[page_, 0, :, 0] = 127 + 4
    vs[int(p["table"][0, 0]), 0, 3, 1] = 255
    c = f4.cache(kc, vc, ks, vs)
    got = call(c, p, single=new == 1, scale=1.0)
    assert not got[..., 32:].isfinite().any() and c.status() == -4 and got[..., :32].isfinite().all()


@pytest.mark.parametrize("qt", QUERIES, ids=str)
def test_strided_queries_and_tables_rows_of_no_sequence(qt):
    for lengths in ([90, 33], [9000, 4000]):   # (and keys split over workgroups)
        p = problem([7, 20], lengths, 4, 2, 128, 16, qt, seed=6)
        c = f4.cache(*p["held"])
        wide = torch.zeros(40, 4 * 128 + 9, dtype=qt)
        wide[3:30, 5:5 + 512] = p["q"].flatten(1)
        q = wide.cuda()[:, 5:5 + 512].unflatten(1, (4, 128))
        table = torch.nn.functional.pad(p["table"], (0, 5)).cuda()[:, :p["table"].shape[1]]
        out = torch.full((40, 4, 128), 7.0, dtype=qt, device="cuda")
        got = c.attend(q, table, p["lengths"].cuda(), starts=(p["starts"] + 3).cuda(), out=out)
        assert got is out and (out[:3] == 7).all() and (out[30:] == 7).all()
        check(out[3:30], p, 128 ** -0.5)
        assert c.status() == 0


@pytest.mark.parametrize("new", [[1, 1], [4, 2], [150, 70]], ids=str)
def test_results_lie_row_by_row(new):
    """Queries of other orders (heads outermost, one for all heads) give results in order."""
    p = problem(new, [390, 133], 4, 2, 128, 16, torch.bfloat16, seed=8)
    c = f4.cache(*p["held"])
    table, lengths, starts = p["table"].cuda(), p["lengths"].cuda(), p["starts"].cuda()
    for q in (p["q"].cuda().transpose(0, 1).contiguous().transpose(0, 1), p["q"][:, :1].cuda().expand(-1, 4, -1)):
        got = c.attend(q, table, lengths, starts=starts)
        assert got.is_contiguous() and torch.equal(got, c.attend(q.contiguous(), table, lengths, starts=starts))
    assert c.status() == 0


@pytest.mark.parametrize("single", [False, True])
def test_bad_pages_and_lengths_are_reported(single):
    p = problem([1, 1], [300, 40], 4, 2, 64, 16, torch.float16)
    p["table"][0, 3] = 10 ** 6
    c = f4.cache(*p["held"])
    call(c, p, single=single)
    assert c.status() == -9
    p = problem([1, 1], [300, 40], 4, 2, 64, 16, torch.float16)
    p["lengths"][1] = -5
    c = f4.cache(*p["held"])
    got = call(c, p, single=single)
    assert c.status() == -9 and not got[1].any()


@pytest.mark.parametrize("new,lengths", [([2, 1], [300, 40]), ([2, 1], [3000, 4000]), ([150, 200], [300, 400])])
def test_bad_starts_are_reported(new, lengths):
    """Starts out of range or out of order, in calls of few rows and of many."""
    total = sum(new)
    for starts in ([0, total + 5, 2], [-3, 1, total], [0, 1, total + 9], [total, 0, 1], [1, total, 0]):
        print(new, lengths, starts, flush=True)
        p = problem(new, lengths, 4, 2, 64, 16, torch.float16)
        p["starts"] = torch.tensor(starts, dtype=torch.int32)
        c = f4.cache(*p["held"])
        assert call(c, p).shape == (total, 4, 64) and c.status() in (-9, -4), starts   # (rows concerned: undefined)


def test_rows_a_tile_and_one_more():
    """Tiles of 16 rows, full and with one token more, of groups that do not divide 16; keys split and not."""
    for heads, kv_heads in ((3, 1), (10, 2), (32, 2), (7, 7)):
        group = heads // kv_heads
        a = 16 // group
        for lengths in ([5 + a, 77, 200], [1500, 5000, 2 * a + 1]):
            new = [a, a + 1, 2 * a + 1]
            print(heads, kv_heads, lengths, flush=True)
            p = problem(new, lengths, heads, kv_heads, 128, 16, torch.bfloat16, seed=heads)
            c = f4.cache(*p["held"])
            check(call(c, p), p, 128 ** -0.5)
            assert c.status() == 0


def test_many_sequences():
    new = [i % 4 for i in range(150)]
    lengths = [n + (i * 37) % 200 if i % 7 else n for i, n in enumerate(new)]
    p = problem(new, lengths, 2, 1, 64, 16, torch.bfloat16, seed=2)
    check(call(f4.cache(*p["held"]), p), p, 64 ** -0.5)
    p = problem([1] * 150, [n + 1 for n in lengths], 2, 1, 64, 16, torch.bfloat16, seed=2)
    check(call(f4.cache(*p["held"]), p, single=True), p, 64 ** -0.5)


@pytest.mark.parametrize("qt,heads,kv_heads,dim", [(torch.float16, 32, 4, 64), (torch.bfloat16, 24, 8, 128),
                                                   (torch.bfloat16, 32, 4, 256)], ids=str)
def test_a_prompt_of_thousands_of_keys_a_workgroup(qt, heads, kv_heads, dim):
    p = problem([2311], [2400], heads, kv_heads, dim, 16, qt, seed=1)
    c = f4.cache(*p["held"])
    got = call(c, p)
    assert c.status() == 0
    for i in (0, 1, 700, 1023, 1024, 1500, 2048, 2309, 2310):
        n = 2400 - 2310 + i
        want, bound = ref.attend(p["q"][i:i + 1], p["k"][0][:n], p["v"][0][:n], dim ** -0.5, torch.int8)
        assert ((got[i:i + 1].cpu().double() - want).abs() <= bound).all(), i


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_single_tokens_of_thousands_of_keys_a_workgroup(dim):
    """Enough sequences that the keys are not split (they share pages): a wavefront goes through more blocks than it has
    lanes."""
    p = problem([1], [9001], 8, 8, dim, 16, torch.bfloat16, seed=2)
    c = f4.cache(*p["held"])
    seqs = 600
    q = torch.randn(seqs, 8, dim, generator=torch.Generator().manual_seed(4)).bfloat16()
    lengths = torch.full((seqs,), 9001, dtype=torch.int32)
    lengths[5], lengths[77], lengths[599] = 8193, 0, 8190
    got = c.attend(q.cuda(), p["table"].expand(seqs, -1).contiguous().cuda(), lengths.cuda()).cpu()
    assert c.status() == 0 and not got[77].any()
    for b in (0, 5, 300, 599):
        n = int(lengths[b])
        want, bound = ref.attend(q[b:b + 1], p["k"][0][:n], p["v"][0][:n], dim ** -0.5, torch.int8)
        assert ((got[b:b + 1].double() - want).abs() <= bound).all(), b


@pytest.mark.parametrize("single", [False, True])
def test_pages_past_32_bits_of_offset(single):
    from flash_moe_hip.kv_cache import PagedCache

    pages = 2 ** 32 // (64 * 64) + 9   # bytes past 2^32, elements past 2^33
    n = 1 if single else 7
    p = problem([n], [200], 2, 1, 128, 64, torch.bfloat16, seed=3)
    shape = (pages, 1, 64, 64)
    held = [torch.empty(shape, dtype=torch.uint8, device="cuda") for _ in range(2)]
    held += [torch.empty((*shape[:3], 4), dtype=torch.uint8, device="cuda") for _ in range(2)]
    far = torch.tensor([[pages - 1, pages - 3, 0, pages // 2]], dtype=torch.int32)
    for b in range(4):
        for t, s in zip(held, p["held"]):
            t[int(far[0, b])] = s[int(p["table"][0, b])].cuda()
    big = f4.cache(*held)
    p["table"] = far
    check(call(big, p, single=single), p, 128 ** -0.5)
    x = rows(3, 1, 128, torch.float32, 4)
    slots = torch.tensor([pages * 64 - 1, 1, (pages - 2) * 64 + 5]).cuda()
    big.write(x, x, slots)
    assert torch.equal(big.read(slots)[1].cpu(), f4.quantized(x.cpu())[2].float()) and big.status() == 0


@pytest.mark.parametrize("single", [False, True])
def test_captured_replayed_and_other_streams(single):
    n = 1 if single else 6
    p = problem([n, n], [5000, 700], 8, 2, 128, 64, torch.bfloat16, seed=4)
    c = f4.cache(*p["held"])
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


@pytest.mark.parametrize("kind", ["single", "few", "many"])
def test_more_sequences_than_keys_are_shared_out_for(kind):
    """Past 1,024 sequences every tile is one piece: single tokens, a few of each, tiles of many rows."""
    seqs = 1100
    new = [1] * seqs if kind == "single" else [(i * 7) % 4 for i in range(seqs)] if kind == "few" else [
        (i * 5) % 67 for i in range(seqs)]
    lengths = [n + (i * 37) % 90 if i % 7 else n for i, n in enumerate(new)]
    lengths[700] = new[700] + 3000
    p = problem(new, lengths, 8, 2, 64, 16, torch.bfloat16, seed=2)
    c = f4.cache(*p["held"])
    got = call(c, p, single=kind == "single").cpu()
    assert c.status() == 0
    ends = p["starts"].tolist()
    for b in list(range(0, seqs, 43)) + [699, 700, 701, seqs - 1]:
        if new[b]:
            want, bound = ref.attend(p["q"][ends[b]:ends[b + 1]], p["k"][b], p["v"][b], 0.125, torch.int8)
            assert ((got[ends[b]:ends[b + 1]].double() - want).abs() <= bound).all(), b
    if kind != "single":
        for starts in (torch.roll(p["starts"], 5), p["starts"] + 3, -p["starts"]):
            p["starts"] = starts.contiguous()
            assert call(c, p).shape == got.shape and c.status() in (-9, -4)


@pytest.mark.parametrize("new", [[1, 1], [40, 300]])
def test_two_calls_at_once(new):
    """Two streams, one cache: each call has its own workspace."""
    p = problem(new, [9000, 5000], 8, 2, 128, 64, torch.bfloat16, seed=4)
    c = f4.cache(*p["held"])
    q, table, lengths, starts = (t.cuda() for t in (p["q"], p["table"], p["lengths"], p["starts"]))
    other = torch.randn_like(q.float()).to(q.dtype)
    want = [c.attend(x, table, lengths, starts) for x in (q, other)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, (x, s) in enumerate(zip((q, other), streams)):
            got[i].append(c.attend(x, table, lengths, starts, stream=s))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs) and c.status() == 0


def test_a_cache_follows_its_tensors():
    from flash_moe_hip.kv_cache import PagedCache

    c = PagedCache.empty(2, 1, 64, 16, f4.CODES)
    x = rows(1, 1, 64, torch.float16, 1)
    slots = torch.tensor([17]).cuda()
    c.write(x, x, slots)
    before = c.k.detach()
    kept = before.view(torch.uint8).clone()
    c.k.set_(torch.zeros(2, 1, 16, 32, dtype=torch.uint8, device="cuda").view(f4.CODES))
    c.write(2 * x, 2 * x, slots)
    assert torch.equal(before.view(torch.uint8), kept) and c.k.view(torch.uint8).any()
    k, v = c.read(slots)
    assert torch.equal(k, v) and c.status() == 0
    c.v_scale.data = torch.zeros(2, 1, 16, 2, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="no longer"):
        c.read(slots)


@pytest.mark.parametrize("new", [1, 5, 60])
def test_large_queries_and_scales(new):
    """A query's power of two times the softmax scale past FP32: scores of 0 stay 0, the largest key alone is left."""
    p = problem([new], [300], 4, 2, 64, 16, torch.bfloat16, seed=6)
    q = torch.zeros(new, 4, 64)
    q[..., 0] = 1e38
    k = torch.zeros(300, 2, 64)
    k[1, :, 0] = 6.0
    p["held"][0], p["held"][2], p["k"] = f4.paged([k], p["table"], 16, p["held"][0].shape[0])
    p["q"] = q.bfloat16()
    c = f4.cache(*p["held"])
    got = call(c, p, single=new == 1, scale=100.0)
    v = p["v"][0][1].repeat_interleave(2, 0)
    assert c.status() == 0 and (got.cpu().double() - v).abs().max() <= 2.0 ** -8 * v.abs().max()


FAR = {   # new, length: a prompt from nothing, one token, drafts, chunks; keys of one workgroup and of several
    "prompt": (9, 9), "single": (1, 300), "few": (5, 300), "many": (100, 300), "single split": (1, 9000),
    "few split": (5, 9000), "many split": (100, 9000)}


def means(v, chosen, new):
    """What rows see whose chosen keys all have the same, by far the largest score: the mean of their values."""
    some = chosen.double().view(-1, 1, 1)
    total, n = (v * some).cumsum(0), some.cumsum(0).clamp(min=1)
    return (total / n)[-new:], ((v.abs() * some).cumsum(0) / n)[-new:]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kind", FAR)
def test_scores_far_from_zero(kind, dim):
    """Scores whose logarithms pass FP32's whole numbers, of either sign: the largest key alone, or equal ones alike.

    Their probabilities are the same power of two or 0: a sum's rounding and the output's (near 2^20 one rounding of
    FP16 for all of them)."""
    new, length = FAR[kind]
    g = torch.Generator().manual_seed(dim + length)
    for qt, size in ((torch.bfloat16, 4e5), (torch.bfloat16, 3e8), (torch.bfloat16, 1e10), (torch.bfloat16, -1e12),
                     (torch.bfloat16, 1e20), (torch.float16, 3e4), (torch.float16, -3e4)):
        p = problem([new], [length], 4, 2, dim, 16, qt, seed=6)
        factor = 1.0 if qt == torch.bfloat16 else 4096.0   # FP16 queries meet keys of 24,576
        p["q"] = torch.zeros(new, 4, dim)
        p["q"][..., 0] = size * (1 + torch.rand(new, 4, generator=g))
        p["q"] = p["q"].to(qt)
        i = torch.arange(length)
        for name, high in (("one", i == 0), ("all", i >= 0), ("some", i % 3 == 0)):
            k = torch.zeros(length, 2, dim)
            k[..., 0] = torch.where(high, 6.0, 4.0 if name == "some" else 0.0).view(-1, 1) * factor * math.copysign(1, size)
            if size < 0 and name == "all":
                k = -k       # every score far below zero
            p["held"][0], p["held"][2], _ = f4.paged([k], p["table"], 16, p["held"][0].shape[0])
            c = f4.cache(*p["held"])
            print(kind, dim, qt, size, name, flush=True)
            got = call(c, p, single=new == 1, scale=0.3).cpu().double()
            want, mass = (t.repeat_interleave(2, 1) for t in means(p["v"][0], high, new))
            off = (2.0 ** -11 if abs(size) == 4e5 else 0.0) + (length + 64) * 2.0 ** -23
            bound = ref.half_step(qt) * want.abs() + off * mass * 1.01 + (2.0 ** -25 if qt == torch.float16 else 0.0)
            assert c.status() == 0 and ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("kind", FAR)
def test_scores_that_are_not_finite_are_reported(kind):
    """A query of infinities: no score is a number, none above the others."""
    new, length = FAR[kind]
    p = problem([new], [length], 4, 2, 64, 16, torch.bfloat16, seed=6)
    k = torch.zeros(length, 2, 64)
    k[..., 0] = 1.0
    p["held"][0], p["held"][2], _ = f4.paged([k], p["table"], 16, p["held"][0].shape[0])
    clean = call(f4.cache(*p["held"]), p, single=new == 1).cpu()
    for size in (-math.inf, math.inf):
        q = p["q"].clone()
        p["q"][-1, 1] = 0
        p["q"][-1, 1, 0] = size
        c = f4.cache(*p["held"])
        got = call(c, p, single=new == 1).cpu()
        assert got[-1, 1].isnan().all() and c.status() == -4, size
        got[-1, 1] = clean[-1, 1]
        assert torch.equal(got, clean)
        p["q"] = q


@pytest.mark.parametrize("new,lengths", [([2, 1], [300, 40]), ([2, 1], [3000, 4000]), ([150, 200], [300, 400]),
                                         ([150, 200], [5000, 4000])])
def test_bad_starts_are_reported_and_write_no_other_rows(new, lengths):
    total = sum(new)
    for starts in ([0, total + 5, 2], [-3, 1, total], [0, 1, total + 9], [total, 0, 1], [1, total, 0]):
        print(new, lengths, starts, flush=True)
        p = problem(new, lengths, 4, 2, 64, 16, torch.float16)
        p["starts"] = torch.tensor(starts, dtype=torch.int32)
        c = f4.cache(*p["held"])
        room = torch.full((total + 16, 4, 64), 7.0, dtype=torch.float16, device="cuda")
        call(c, p, out=room[8:8 + total])
        assert c.status() == -9
        free = torch.ones(total + 16, dtype=torch.bool)
        for a, b in zip(starts, starts[1:]):
            a = min(max(a, 0), total)
            free[8 + a:8 + max(min(b, total), a)] = False
        assert (room.cpu()[free] == 7).all(), starts


@pytest.mark.parametrize("kind", ["few", "many"])
def test_bad_starts_of_many_sequences_are_reported(kind):
    """Past 1,024 sequences, where every tile is one piece."""
    seqs = 1100
    new = [(i * 7) % 4 if kind == "few" else (i * 5) % 67 for i in range(seqs)]
    p = problem(new, [n + (i * 37) % 90 for i, n in enumerate(new)], 8, 2, 64, 16, torch.bfloat16, seed=2)
    c = f4.cache(*p["held"])
    total = sum(new)
    for starts in (torch.roll(p["starts"], 5), p["starts"] + 3, -p["starts"]):
        p["starts"] = starts.contiguous()
        room = torch.full((total + 16, 8, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        call(c, p, out=room[8:8 + total])
        assert c.status() == -9 and (room[:8] == 7).all() and (room[8 + total:] == 7).all()


@pytest.mark.parametrize("seqs,rows", [(1025, 3), (4096, 3), (4161, 40), (70001, 2)])
def test_sequences_are_found_among_thousands(seqs, rows):
    """Past 1,024 sequences a workgroup searches for its own: with none before it, none behind, runs without tokens."""
    g = torch.Generator().manual_seed(seqs)
    new = torch.randint(0, rows + 1, (seqs,), generator=g)
    new[:70], new[200:333], new[-1] = 0, 0, rows
    lengths = (new + torch.randint(0, 30, (seqs,), generator=g)).clamp(max=48)
    p = problem([48], [48], 8, 2, 64, 16, torch.bfloat16, seed=2)   # (all sequences share three pages)
    c = f4.cache(*p["held"])
    starts = torch.nn.functional.pad(new.cumsum(0), (1, 0))
    q = torch.randn(int(starts[-1]), 8, 64, generator=g).bfloat16()
    got = c.attend(q.cuda(), p["table"].expand(seqs, -1).contiguous().cuda(), lengths.int().cuda(), starts.int().cuda()).cpu()
    assert c.status() == 0
    k, v = (t[0].float().repeat_interleave(4, 1) for t in (p["k"], p["v"]))
    position = torch.repeat_interleave(lengths - new, new) + torch.arange(len(q)) - torch.repeat_interleave(starts[:-1], new)
    worst = 0.0
    for at in range(0, len(q), 8192):   # (FP32 here: the bounds of the checked rows are far above its errors)
        s = torch.einsum("thd,khd->htk", q[at:at + 8192].float(), k) * 0.125
        s = s.masked_fill(torch.arange(48).view(1, 1, -1) > position[at:at + 8192].view(1, -1, 1), -math.inf)
        want = torch.einsum("htk,khd->thd", s.softmax(-1), v)
        worst = max(worst, float((got[at:at + 8192].float() - want).abs().max()))
    # BF16's half step of the result, FP16's of the probabilities and FP32's of the scores, twice, of the largest value
    assert worst <= (2.0 ** -8 + 2.0 ** -11 + 2 * 2.0 ** -16) * float(v.abs().max())
