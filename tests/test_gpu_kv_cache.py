"""The paged cache on the GPU: rows written (and quantized) and read back."""
from __future__ import annotations

import math

import pytest
import torch

from mixer_reference import half_step, quantized

pytestmark = pytest.mark.gpu

ROWS = [torch.float32, torch.float16, torch.bfloat16]
CACHES = [torch.float16, torch.bfloat16, torch.int8]


def rows(tokens, heads, dim, dtype, seed, strided=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, dim, generator=g) * torch.exp(torch.randn(tokens, heads, 1, generator=g))
    x = x.to(dtype)
    if strided:   # part of a wider row, off the 16-byte grid
        wide = torch.zeros(tokens, heads * dim + 7, dtype=dtype)
        wide[:, 3:3 + heads * dim] = x.flatten(1)
        return wide.cuda()[:, 3:3 + heads * dim].unflatten(1, (heads, dim))
    return x.cuda()


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("cache", CACHES, ids=str)
@pytest.mark.parametrize("dtype", ROWS, ids=str)
@pytest.mark.parametrize("tokens,heads,dim,page", [(1, 1, 64, 16), (37, 3, 128, 16), (130, 2, 256, 64), (65, 8, 64, 1024)])
def test_write_and_read(tokens, heads, dim, page, dtype, cache, strided):
    from flash_moe_hip.kv_cache import PagedCache

    print(tokens, heads, dim, page, dtype, cache, strided, flush=True)
    pages = -(-tokens // page) + 2
    c = PagedCache.empty(pages, heads, dim, page, cache)
    k, v = rows(tokens, heads, dim, dtype, 1, strided), rows(tokens, heads, dim, dtype, 2, strided)
    g = torch.Generator().manual_seed(3)
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[::5] = -1
    c.write(k, v, slots.cuda())
    assert c.status() == 0
    kept = slots >= 0
    # every other slot is as it was
    for t in (c.k, c.v):
        flat = t.cpu().transpose(1, 2).flatten(0, 1)
        untouched = torch.ones(pages * page, dtype=torch.bool)
        untouched[slots[kept]] = False
        assert not flat[untouched].any()
    for out in ROWS:
        rk, rv = c.read(slots.cuda(), dtype=out)
        assert c.status() == 0 and rk.dtype == out
        for got, x in ((rk.cpu(), k.cpu()), (rv.cpu(), v.cpu())):
            assert not got[~kept].any()
            if cache == torch.int8:
                codes, scale = quantized(x)
                want = (codes.float() * scale.unsqueeze(-1)).to(out)
            else:
                want = x.to(cache).to(out)
            torch.testing.assert_close(got[kept], want[kept], rtol=0, atol=0)
    # an int8 row is off by half a step of its scale (and the scale's and the product's FP32 roundings)
    if cache == torch.int8:
        rk, _ = c.read(slots.cuda())
        x = k.cpu().double()[kept]
        step = x.abs().amax(-1, keepdim=True) / 127
        assert ((rk.cpu().double()[kept] - x).abs() <= step * (0.5 + 3 * 127 * half_step(torch.float32))).all()


@pytest.mark.parametrize("cache", CACHES, ids=str)
@pytest.mark.parametrize("tokens,heads,dim", [(8195, 8, 128), (32773, 4, 64), (4101, 8, 256)])
def test_many_rows(tokens, heads, dim, cache):
    """Enough rows that a lane takes four, and a ragged end."""
    from flash_moe_hip.kv_cache import PagedCache

    g = torch.Generator(device="cuda").manual_seed(tokens)
    c = PagedCache.empty(-(-tokens // 32) + 1, heads, dim, 32, cache)
    k, v = (torch.randn(tokens, heads, dim, generator=g, device="cuda").bfloat16() for _ in range(2))
    slots = torch.randperm(c.pages * 32, generator=g, device="cuda")[:tokens]
    slots[-5:-1] = -1
    kept = slots >= 0
    c.write(k, v, slots)
    for got, x in zip(c.read(slots, torch.float32), (k, v)):
        if cache == torch.int8:   # (on the CPU: torch divides by a number on the GPU with its reciprocal)
            codes, scale = quantized(x.cpu())
            want = (codes.float() * scale.unsqueeze(-1)).cuda()
        else:
            want = x.to(cache).float()
        assert torch.equal(got[kept], want[kept]) and not got[~kept].any()
    assert c.status() == 0
    free = torch.ones(c.pages * 32, dtype=torch.bool, device="cuda")
    free[slots[kept]] = False
    assert not c.k.transpose(1, 2).flatten(0, 1)[free].any()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_edge_rows_of_an_int8_cache(dim):
    from flash_moe_hip.kv_cache import PagedCache

    c = PagedCache.empty(2, 1, dim, 16, torch.int8)
    x = torch.zeros(8, 1, dim)
    x[1, 0, 5] = 2.0 ** -140           # below the smallest scale: zeros
    x[2, 0, 7] = math.inf
    x[3, 0, 9] = math.nan
    x[4, 0] = torch.linspace(-3e38, 3e38, dim)
    x[5, 0] = -127.0
    x[6, 0] = torch.arange(dim) % 254 * 0.5 - 63.0   # ties: halves of the step 63.5 / 127
    x[7, 0, -1] = 2.0 ** -90
    slots = torch.arange(8).cuda()
    c.write(x.cuda(), x.cuda(), slots)
    assert c.status() == -4 and c.status() == 0
    k, _ = c.read(slots)
    k = k.cpu()
    assert not k[0].any() and not k[1].any()
    assert k[2].isnan().all() and k[3].isnan().all()
    codes, scale = quantized(x)
    want = codes.float() * scale.unsqueeze(-1)
    torch.testing.assert_close(k[4:], want[4:], rtol=0, atol=0, equal_nan=True)   # (row 4: linspace overflows)
    # the largest finite values
    x = torch.where(torch.arange(dim) % 3 == 0, 3e38, -1.5e38).view(1, 1, dim)
    c.write(x.cuda(), x.cuda(), slots[:1])
    k, _ = c.read(slots[:1])
    codes, scale = quantized(x)
    torch.testing.assert_close(k.cpu(), codes.float() * scale.unsqueeze(-1), rtol=0, atol=0)
    assert c.status() == 0


def test_values_an_fp16_cache_cannot_hold_are_reported():
    from flash_moe_hip.kv_cache import PagedCache

    c = PagedCache.empty(1, 1, 64, 16, torch.float16)
    x = torch.full((1, 1, 64), 65504.0)
    c.write(x.cuda(), x.cuda(), torch.zeros(1, dtype=torch.int64).cuda())
    assert c.status() == 0
    x[0, 0, 3] = 65520.0
    c.write(x.cuda(), x.cuda(), torch.zeros(1, dtype=torch.int64).cuda())
    assert c.status() == -4


def test_slots_past_the_cache_are_skipped_and_reported():
    from flash_moe_hip.kv_cache import PagedCache

    c = PagedCache.empty(2, 2, 64, 16, torch.int8)
    x = rows(3, 2, 64, torch.bfloat16, 1)
    slots = torch.tensor([32, 5, 2 ** 40]).cuda()
    c.write(x, x, slots)
    assert c.status() == -9 and c.status() == 0
    k, v = c.read(slots, torch.bfloat16)
    assert c.status() == -9
    assert not k[0].any() and not v[2].any() and k[1].any()


def test_more_than_32_bits_of_offset():
    """Pages whose byte offsets and element offsets pass 2^32."""
    from flash_moe_hip.kv_cache import PagedCache

    pages = (2 ** 32 // (64 * 128)) + 5   # elements past 2^32
    k = torch.empty(pages, 1, 64, 128, dtype=torch.int8, device="cuda")
    scale = torch.empty(pages, 1, 64, device="cuda")
    c = PagedCache(k, torch.empty_like(k), scale, torch.empty_like(scale))
    x = rows(6, 1, 128, torch.float32, 4)
    slots = torch.tensor([0, 63, 64, pages * 64 - 1, pages * 64 - 64, pages * 32]).cuda()
    c.write(x, x, slots)
    got, _ = c.read(slots)
    codes, s = quantized(x.cpu())
    torch.testing.assert_close(got.cpu(), codes.float() * s.unsqueeze(-1), rtol=0, atol=0)
    assert c.status() == 0


def test_another_stream_and_no_tokens():
    from flash_moe_hip.kv_cache import PagedCache

    c = PagedCache.empty(4, 2, 64, 16, torch.float16)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    e = torch.zeros(0, 2, 64, device="cuda")
    c.write(e, e, none)
    assert c.read(none)[0].shape == (0, 2, 64)
    side = torch.cuda.Stream()
    x = rows(20, 2, 64, torch.float16, 9)
    slots = torch.arange(20).cuda()
    side.wait_stream(torch.cuda.current_stream())
    c.write(x, x, slots, stream=side)
    k, v = c.read(slots, stream=side)
    side.synchronize()
    torch.testing.assert_close(k, x, rtol=0, atol=0)
    torch.testing.assert_close(v, x, rtol=0, atol=0)


@pytest.mark.parametrize("cache", [torch.bfloat16, torch.int8], ids=str)
def test_values_a_read_type_cannot_hold_are_reported(cache):
    """Finite rows read as a narrower type become infinite and say so; rows stored as they are not finite do not."""
    from flash_moe_hip.kv_cache import PagedCache

    c = PagedCache.empty(2, 1, 128, 16, cache)
    x = torch.ones(2, 1, 128)
    x[1, 0, 77] = 1e5
    slots = torch.tensor([3, 20]).cuda()
    c.write(x.cuda(), x.cuda(), slots)
    assert c.status() == 0
    k, _ = c.read(slots[:1], torch.float16)
    assert k.isfinite().all() and c.status() == 0
    for dtype in (torch.float32, torch.bfloat16):
        assert c.read(slots, dtype)[1].isfinite().all() and c.status() == 0
    k, v = c.read(slots, torch.float16)
    assert k[1, 0, 77].isinf() and v[1, 0, 77].isinf() and k[0].isfinite().all() and c.status() == -4
    x[1, 0, 77] = math.inf
    c.write(x.cuda(), x.cuda(), slots)
    assert c.status() == -4
    c.read(slots, torch.float16)
    assert c.status() == 0


@pytest.mark.parametrize("cache", [torch.float16, torch.int8], ids=str)
def test_a_cache_follows_its_tensors(cache):
    """The tensors cannot be exchanged for others; one whose storage moves is written and read where it lies."""
    from flash_moe_hip.kv_cache import PagedCache

    c = PagedCache.empty(2, 1, 64, 16, cache)
    for name in ("k", "v", "k_scale", "v_scale"):
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name))
    x = rows(1, 1, 64, torch.float16, 1)
    slots = torch.tensor([17]).cuda()
    c.write(x, x, slots)
    before = c.k.detach()          # keeps the old memory
    kept = before.clone()
    c.k.set_(torch.zeros_like(c.k))
    c.write(2 * x, 2 * x, slots)
    assert torch.equal(before, kept) and c.k.any()
    k, v = c.read(slots)
    assert torch.equal(k, v) and c.status() == 0
    for moved in (torch.zeros(1, 1, 16, 64, dtype=cache), torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16),
                  torch.zeros(2, 1, 64, 16, dtype=cache).transpose(2, 3), torch.zeros(0, dtype=cache)):
        moved = moved.cuda() if moved.is_contiguous() else moved.transpose(2, 3).cuda().transpose(2, 3)
        c = PagedCache.empty(2, 1, 64, 16, cache)
        c.v.data = moved
        for call in (lambda: c.write(x, x, slots), lambda: c.read(slots)):
            with pytest.raises(ValueError, match="no longer"):
                call()
    c = PagedCache.empty(2, 1, 64, 16, cache)
    c.k.untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="no longer"):
        c.attend(torch.zeros(1, 1, 64, dtype=torch.float16, device="cuda"), torch.zeros(1, 1, dtype=torch.int32,
                 device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda"))
