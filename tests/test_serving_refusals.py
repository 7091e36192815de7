"""What the 4-bit cache's calls refuse (CPU only: every check precedes any HIP call)."""
from __future__ import annotations

import ctypes as C

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
