"""Plain 64-bit forms of the token mixers and the error bounds their tests use.

Bounds are from the operands' types alone.  A rounding to a type is off by at
most half a step, eps / 2 of the value (finfo.eps / 2: BF16 2^-8, FP16 2^-11,
FP32 2^-24)."""
from __future__ import annotations

import math

import torch


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def quantized(x):
    """(codes, scale) of rows as the cache stores them, FP32 divisions."""
    x = x.float()
    top = x.abs().amax(-1)
    scale = top / 127.0
    scale = torch.where(scale < 2.0 ** -100, torch.zeros_like(scale), scale)
    scale = torch.where(torch.isfinite(x).all(-1), scale, torch.full_like(scale, math.nan))
    codes = torch.round(x / scale.unsqueeze(-1)).clamp(-127, 127)
    codes = torch.where((scale > 0).unsqueeze(-1), codes, torch.zeros_like(codes))
    return codes.to(torch.int8), scale


def paged(k, table, page_size, pages, dtype, scales=False):
    """Rows [sequences][tokens, kv_heads, dim] laid out as a cache; unused places
    hold NaN (16-bit) or 77 codes with scale NaN, as stale pages may."""
    heads, dim = k[0].shape[1:]
    if dtype == torch.int8:
        c = torch.full((pages, heads, page_size, dim), 77, dtype=torch.int8)
        s = torch.full((pages, heads, page_size), math.nan)
    else:
        c, s = torch.full((pages, heads, page_size, dim), math.nan, dtype=dtype), None
    values = []
    for b, rows in enumerate(k):
        at = torch.arange(rows.shape[0])
        page, off = table[b, at // page_size].long(), at % page_size
        if dtype == torch.int8:
            codes, scale = quantized(rows)
            c[page, :, off], s[page, :, off] = codes, scale
            values.append(codes.double() * scale.double().unsqueeze(-1))
        else:
            c[page, :, off] = rows.to(dtype)
            values.append(rows.to(dtype).double())
    return c, s, values


def attend(q, k, v, scale, cache_dtype):
    """One sequence: q [n, heads, dim] the last n of the tokens of k, v [L, kv_heads,
    dim] (values, float64).  Returns (out, bound) float64.

    The kernel rounds each probability (times the value's scale) once to the 16-bit
    type p of its matrix instruction and the result once to q's type; sums are FP32.
      |error| <= e_out |o| + (e_p + 2 d + (L + 64) 2^-23) A + L 2^-31 max|v|
    with A = sum p |v|, d the score's error, (dim + 4) 2^-24 scale sum |q k| for
    FP32 products and sums (twice that probability error: p and the sum of p), and
    the last term FP16's subnormal probabilities (held with 2^7: off by 2^-32 each,
    the sum of probabilities is at least 1)."""
    n, heads, dim = q.shape
    length, group = k.shape[0], heads // k.shape[1]
    e_p = half_step(torch.bfloat16 if cache_dtype == torch.bfloat16 else torch.float16)
    out = torch.zeros(n, heads, dim, dtype=torch.float64)
    bound = torch.zeros_like(out)
    qd = q.double()
    pos = torch.arange(length - n, length)
    hidden = torch.arange(length).view(1, -1) > pos.view(-1, 1)
    for h in range(heads):
        if not length:
            break
        kh, vh = k[:, h // group], v[:, h // group]
        s = (qd[:, h] @ kh.T) * scale
        mass = (qd[:, h].abs() @ kh.abs().T) * scale
        s = s.masked_fill(hidden, -math.inf)
        top = s.amax(1, keepdim=True)
        p = torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
        p = torch.where(hidden, torch.zeros_like(p), p)
        total = p.sum(1, keepdim=True)
        p = p / torch.where(total > 0, total, torch.ones_like(total))
        out[:, h] = p @ vh
        a = p @ vh.abs()
        d = (dim + 4) * 2.0 ** -24 * mass.masked_fill(hidden, 0).amax(1, keepdim=True)
        tiny = length * 2.0 ** -31 * vh.abs().amax() if length else 0.0
        bound[:, h] = half_step(q.dtype) * out[:, h].abs() + (e_p + 2 * d + (length + 64) * 2.0 ** -23) * a + tiny
    if q.dtype == torch.float16:
        bound += 2.0 ** -25   # subnormal outputs
    return out, bound * 1.01 + 1e-30   # (products of the terms above)


def linear(state, q, k, v, beta, gate):
    """Token by token in float64: state [heads, dv, dk], q, k [n, key_heads, dk], v
    [n, heads, dv], beta (or None) and gate [n, heads].  Returns (out, state, size)
    with size [heads, dv]: the largest of |S row| + |v| |k| met on the way."""
    heads = v.shape[1]
    s = state.double().clone()
    q, k = (t.double().repeat_interleave(heads // t.shape[1], 1) for t in (q, k))
    v, decay = v.double(), torch.exp(gate.double())
    out = torch.zeros(v.shape, dtype=torch.float64)
    size = s.norm(dim=2)
    for t in range(v.shape[0]):
        s = s * decay[t].view(-1, 1, 1)
        u = v[t]
        if beta is not None:
            u = beta[t].double().unsqueeze(1) * (u - torch.einsum("hvk,hk->hv", s, k[t]))
        s = s + u.unsqueeze(2) * k[t].unsqueeze(1)
        out[t] = torch.einsum("hvk,hk->hv", s, q[t])
        size = torch.maximum(size, s.norm(dim=2) + v[t].abs() * k[t].norm(dim=1, keepdim=True))
    return out, s, size


def linear_bound(size, tokens, key_dim, chunk=64):
    """How far a row of the state may be off, in 2-norm (and an output, for |q| <= 1),
    for keys of norm <= 1, gates <= 0 and beta in [0, 1]: a step of the recurrence
    then never lengthens an error, so those of the chunks add up.  A chunk's error is
    that of four FP32 products of at most key_dim + 64 terms (W S, the writes, the
    state, the output), each term off by 2^-24 of |S| + |v| |k|, and its solution
    of 1 + L doubles them at most (its inverse is a product of such steps)."""
    chunks = -(-tokens // chunk) + 1
    return chunks * 8 * (key_dim + chunk) * 2.0 ** -24 * size
