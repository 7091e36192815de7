"""Plain forms of the 4-bit cache: E2M1 codes, one power of two a 32 channels."""
from __future__ import annotations

import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
CODES, SCALES = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def quantized(x):
    """(codes [..., dim / 2], scale bytes [..., dim / 32], values [..., dim] float64) of rows [..., dim]."""
    y = x.double().unflatten(-1, (-1, 32))
    top = y.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(y).all(-1, keepdim=True) | (top >= 7 * 2.0 ** 13)
    top = torch.where(bad, 1.0, top)
    e = torch.full_like(top, -23.0)
    for i in range(-22, 14):   # the least e with top < 7 * 2^e
        e = torch.where(top >= 7 * 2.0 ** (i - 1), float(i), e)
    z = torch.where(bad, 0.0, y.abs()) / 2.0 ** e
    code = torch.zeros(z.shape, dtype=torch.int64)
    for i in range(7):   # past the middle of two numbers, or on it and the lower one's code is odd
        middle = (GRID[i] + GRID[i + 1]) / 2
        code += (z >= middle) if i % 2 else (z > middle)
    value = torch.where(bad, math.nan, torch.sign(y) * GRID[code] * 2.0 ** e).flatten(-2)
    code = torch.where(bad, 0, code + 8 * torch.signbit(y)).flatten(-2)
    scale = torch.where(bad, 255, e + 127).squeeze(-1).to(torch.uint8)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), scale, value


def paged(k, table, page_size, pages):
    """Rows [sequences][tokens, kv_heads, dim] laid out as a cache; unused places hold codes and the scale of a block
    that is not finite, as stale pages may."""
    heads, dim = k[0].shape[1:]
    c = torch.full((pages, heads, page_size, dim // 2), 0x73, dtype=torch.uint8)
    s = torch.full((pages, heads, page_size, dim // 32), 255, dtype=torch.uint8)
    values = []
    for b, rows in enumerate(k):
        at = torch.arange(rows.shape[0])
        page, off = table[b, at // page_size].long(), at % page_size
        c[page, :, off], s[page, :, off], value = quantized(rows)
        values.append(value)
    return c, s, values


def cache(k, v, k_scale, v_scale):
    from flash_moe_hip.kv_cache import PagedCache

    return PagedCache(k.cuda().view(CODES), v.cuda().view(CODES), k_scale.cuda().view(SCALES), v_scale.cuda().view(SCALES))
