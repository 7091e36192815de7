"""What the calls of the 4-bit cache, page tables and rotary positions refuse (CPU only: every check precedes any HIP call)."""
from __future__ import annotations

import ctypes as C
import math
import struct

import pytest
import torch

P = C.c_void_p(4096)
F4 = 5


@pytest.fixture(scope="module")
def lib():
    from flash_moe_hip import _lib

    return _lib.load()


def test_f4_cache_constructor():
    from flash_moe_hip.kv_cache import PagedCache

    codes, scales = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu

    def make(dim=128, scale=(2, 2, 16, 4), scale_type=scales, v_dtype=codes, with_scales=True):
        k = torch.zeros(2, 2, 16, dim // 2, dtype=torch.uint8)
        s = torch.zeros(scale, dtype=torch.uint8).view(scale_type) if with_scales else None
        return PagedCache(k.view(codes), k.view(v_dtype), s, s)

    with pytest.raises(ValueError, match="CUDA device"):
        make()
    with pytest.raises(ValueError, match="head_dim"):
        make(dim=96)
    with pytest.raises(ValueError, match="needs k_scale"):
        make(with_scales=False)
    with pytest.raises(ValueError, match="head_dim / 32"):
        make(scale=(2, 2, 16, 8))
    with pytest.raises(ValueError, match="float8_e8m0fnu"):
        make(scale_type=torch.uint8)
    with pytest.raises(ValueError, match="one type"):
        make(v_dtype=torch.uint8)
    with pytest.raises(ValueError, match="head_dim"):
        PagedCache.empty(2, 2, 96, 16, codes, "cpu")


def test_f4_cache_codes(lib):
    cache = dict(kc=P, vc=P, ks=P, vs=P, ct=F4, pages=4, heads=2, page=16, dim=64)

    def write(**kw):
        a = dict(k=P, kt=256, kh=64, v=P, vt=256, vh=64, type=1, slots=P, tokens=4, **cache, flags=P, stream=None)
        a.update(kw)
        return lib.mqh_kv_write(*a.values())

    def read(**kw):
        a = dict(slots=P, tokens=4, **cache, k=P, v=P, type=1, flags=P, stream=None)
        a.update(kw)
        return lib.mqh_kv_read(*a.values())

    def attend(**kw):
        a = dict(q=P, qt=512, qh=64, q_type=1, tokens=4, starts=P, seqs=2, n=8, **cache, table=P, stride=4, cols=4,
                 lengths=P, scale=0.125, out=P, ws=P, bytes=1 << 30, flags=P, stream=None)
        a.update(kw)
        return lib.mqh_attend(*a.values())

    for call in (write, read, attend):
        for bad in (dict(ks=None), dict(vs=None), dict(ks=C.c_void_p(4100)), dict(vs=C.c_void_p(4097)), dict(kc=None),
                    dict(page=24), dict(vc=C.c_void_p(4104))):
            assert call(**bad) == -1, bad
        assert call(dim=96) == -2 and call(dim=32) == -2
    assert write(type=5) == -2 and read(type=5) == -2 and attend(q_type=0) == -2 and attend(q_type=5) == -2


def test_page_table_constructor():
    from flash_moe_hip.page_table import PageTable

    def make(table=(2, 4), lengths=2, free=8, count=1, dtype=torch.int32, page_size=16):
        return PageTable(torch.zeros(table, dtype=torch.int32), torch.zeros(lengths, dtype=dtype),
                         torch.zeros(free, dtype=torch.int32), torch.zeros(count, dtype=torch.int32), page_size)

    with pytest.raises(ValueError, match="CUDA device"):
        make()
    for bad, why in ((dict(page_size=24), "page_size"), (dict(lengths=3), "lengths"), (dict(count=2), "count"),
                     (dict(dtype=torch.int64), "lengths"), (dict(table=(8193, 1), lengths=8193), "sequences"),
                     (dict(table=(2, 2 ** 26 + 1)), "columns"), (dict(table=(2, 0)), "columns"), (dict(free=0), "page"),
                     (dict(table=(2, 4, 1)), "columns")):
        with pytest.raises(ValueError, match=why):
            make(**bad)


def test_page_codes(lib):
    def extend(**kw):
        a = dict(grow=P, table=P, cols=4, lengths=P, free=P, count=P, seqs=3, pages=8, page=16, rows=5, starts=P, slots=P,
                 positions=P, flags=P, stream=None)
        a.update(kw)
        words = [getattr(x, "value", x) or 0 for x in a.values()]
        assert lib.mqh_pages_extend_words(struct.pack("15q", *words)) == -1
        return lib.mqh_pages_extend(*a.values()) if all(abs(w) < 2 ** 31 for w in words) else -1

    def trim(**kw):
        a = dict(keep=P, table=P, cols=4, lengths=P, free=P, count=P, seqs=3, pages=8, page=16, flags=P, stream=None)
        a.update(kw)
        words = [getattr(x, "value", x) or 0 for x in a.values()]
        assert lib.mqh_pages_trim_words(struct.pack("11q", *words)) == -1
        return lib.mqh_pages_trim(*a.values()) if all(abs(w) < 2 ** 31 for w in words) else -1

    both = (dict(table=None), dict(lengths=None), dict(free=None), dict(count=None), dict(flags=None), dict(seqs=0),
            dict(seqs=8193), dict(cols=0), dict(cols=2 ** 26 + 1), dict(pages=0), dict(page=24), dict(page=8),
            dict(seqs=2 ** 32 + 1), dict(cols=2 ** 32 + 4), dict(pages=2 ** 32 + 1), dict(page=2 ** 32 + 16))
    for bad in both:
        assert extend(**bad) == -1 and trim(**bad) == -1, bad
    assert trim(keep=None) == -1
    for bad in (dict(grow=None), dict(starts=None), dict(slots=None), dict(positions=None), dict(rows=-1),
                dict(rows=2 ** 30 + 1), dict(slots=C.c_void_p(4104)), dict(positions=C.c_void_p(4100)),
                dict(rows=2 ** 32 + 5)):
        assert extend(**bad) == -1, bad
    assert lib.mqh_pages_extend_words(None) == -1 and lib.mqh_pages_trim_words(None) == -1


def test_rotary_constructor():
    from flash_moe_hip.rotary import Rotary

    with pytest.raises(ValueError, match="CUDA device"):
        Rotary(128, device="cpu")
    for args, kw, why in (((96,), {}, "head_dim"), ((128, 256), {}, "rotary_dim"), ((128, 24), {}, "rotary_dim"),
                          ((128, 0), {}, "rotary_dim"), ((128,), dict(layout="other"), "layout"),
                          ((128,), dict(base=1.0), "base"), ((128,), dict(base=math.inf), "base"),
                          ((128,), dict(scaling=dict(kind="other", factor=2)), "kind"),
                          ((128,), dict(scaling=dict(kind="linear")), "linear scaling"),
                          ((128,), dict(scaling=dict(kind="linear", factor=2, original=9)), "linear scaling"),
                          ((128,), dict(scaling=dict(kind="linear", factor=0.5)), "factor at least 1"),
                          ((128,), dict(scaling=dict(kind="yarn", factor=2)), "yarn scaling"),
                          ((128,), dict(scaling=dict(kind="yarn", factor=2, original=100, fast=1, slow=1)), "fast"),
                          ((128,), dict(scaling=dict(kind="bands", factor=2, original=100, low=4, high=4)), "high"),
                          ((128,), dict(scaling=dict(kind="bands", factor=math.nan, original=100)), "positive")):
        with pytest.raises(ValueError, match=why):
            Rotary(*args, device="cpu", **kw)


def test_rotary_frequencies():
    """The scalings at values worked out by hand."""
    from flash_moe_hip.rotary import frequencies

    f, a = frequencies(8, 10000.0)
    assert a == 1.0 and f == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15)
    assert frequencies(8, 10000.0, dict(kind="linear", factor=4))[0] == pytest.approx([x / 4 for x in f], rel=1e-15)
    # over 2 pi * 100 positions the pairs turn 100, 10, 1 and 0.1 times
    n = 200 * math.pi
    got, a = frequencies(8, 10000.0, dict(kind="bands", factor=10, original=n, low=1, high=19))
    assert a == 1.0 and got == pytest.approx([1.0, 0.1 * (0.5 + 0.05), 0.001, 0.0001], rel=1e-12)
    # 10 turns: just past pair 1, 0.1 turns: just past pair 3, so the ramp is from 1 to 4
    got, a = frequencies(8, 10000.0, dict(kind="yarn", factor=math.e, original=n * 1.0000001, fast=10, slow=0.1))
    assert a == pytest.approx(1.1) and got[:2] == [1.0, 0.1]
    assert got[2:] == pytest.approx([0.01 * (2 / 3 + 1 / 3 / math.e), 0.001 * (1 / 3 + 2 / 3 / math.e)], rel=1e-12)
    assert frequencies(8, 1e4, dict(kind="yarn", factor=2, original=100, amplitude=1.5))[1] == 1.5


def test_rotary_codes(lib):
    def call(**kw):
        a = dict(q=P, qt=512, qh=128, k=P, kt=256, kh=128, type=1, positions=P, tokens=3, heads=4, kv_heads=2, dim=128,
                 turns=P, rotary=128, interleaved=0, amplitude=1.0, qw=None, kw=None, eps=1e-6, qo=P, qot=512, qoh=128, ko=P,
                 kot=256, koh=128, flags=P, stream=None)
        a.update(kw)
        words = [getattr(x, "value", x) or 0 for x in a.values()]
        big = any(isinstance(w, int) and abs(w) >= 2 ** 31 for w in words)
        got = lib.mqh_rotary_words(struct.pack("15qd2qd8q", *words))
        assert big or got == lib.mqh_rotary(*a.values())
        return got

    for bad in (dict(q=None), dict(k=None), dict(positions=None), dict(turns=None), dict(qo=None), dict(ko=None),
                dict(flags=None), dict(tokens=0), dict(tokens=2 ** 24 + 1), dict(heads=0), dict(kv_heads=4097),
                dict(rotary=24), dict(rotary=144), dict(rotary=0), dict(interleaved=2), dict(amplitude=0.0),
                dict(amplitude=math.inf), dict(eps=0.0), dict(eps=math.nan), dict(q=C.c_void_p(4097)),
                dict(turns=C.c_void_p(4100)), dict(positions=C.c_void_p(4098)), dict(kw=C.c_void_p(4098)),
                dict(type=0, qo=C.c_void_p(4098)), dict(tokens=2 ** 32 + 3), dict(heads=2 ** 32 + 4),
                dict(dim=2 ** 32 + 128)):
        assert call(**bad) == -1, bad
    for bad in (dict(type=3), dict(type=5), dict(dim=96)):
        assert call(**bad) == -2, bad
    assert lib.mqh_rotary_words(None) == -1


def test_rotary_amplitudes_fp32_cannot_hold():
    """A factor that is 0 or infinite in FP32 is refused where it is stated, not at the first call."""
    from flash_moe_hip.rotary import Rotary, frequencies

    for a in (1e-46, 1e39, 1e300, 5e-324):
        with pytest.raises(ValueError, match="amplitude"):
            frequencies(64, 1e4, dict(kind="yarn", factor=2, original=100, amplitude=a))
        with pytest.raises(ValueError, match="amplitude"):
            Rotary(128, device="cpu", scaling=dict(kind="yarn", factor=2, original=100, amplitude=a))
    for a in (1e-30, 1e30):
        assert frequencies(64, 1e4, dict(kind="yarn", factor=2, original=100, amplitude=a))[1] == a
