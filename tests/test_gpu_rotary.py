"""Rotary positions on the GPU against 64 bits."""
from __future__ import annotations

import math
from decimal import Decimal, getcontext

import pytest
import torch

from mixer_reference import half_step

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
SCALINGS = [None, dict(kind="linear", factor=4), dict(kind="yarn", factor=32, original=8192),
            dict(kind="bands", factor=8.0, original=8192)]


def reference(x, positions, rot, weight=None, eps=1e-6):
    """(out, bound) float64 of rows x [n, heads, dim].

    Cosine and sine: the angle is an FP32 number below pi / 4 with three roundings (3 * 0.79 * 2^-24), the series two of
    its own, the factor one: 6 * 2^-24 of the factor; a product's rounding and the sum's: 8 * 2^-24 A (|a| + |b|) in
    all.  Frequencies are doubles: position * frequency * 2^-51.  The norm: a sum of eight squares, then of the lanes,
    the mean, eps, root, quotient, two products: 16 * 2^-24.  The output rounds once."""
    dtype, x = x.dtype, x.double()
    step = 8 * 2.0 ** -24
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(2, keepdim=True) + eps) * weight.double()
        step += 16 * 2.0 ** -24
    f = torch.tensor(rot.frequencies, dtype=torch.float64)
    angle = positions.double().view(-1, 1, 1) * f
    cos, sin = torch.cos(angle) * rot.amplitude, torch.sin(angle) * rot.amplitude
    half = rot.rotary_dim // 2
    i = torch.arange(half)
    at = (i, i + half) if rot.layout == "half" else (2 * i, 2 * i + 1)
    a, b = x[..., at[0]], x[..., at[1]]
    out, bound = x.clone(), step * x.abs() if weight is not None else torch.zeros_like(x)
    out[..., at[0]], out[..., at[1]] = a * cos - b * sin, a * sin + b * cos
    off = (step + angle.abs() * 2.0 ** -51) * rot.amplitude * (a.abs() + b.abs())
    bound[..., at[0]], bound[..., at[1]] = off, off
    bound += half_step(dtype) * (out.abs() + bound)
    if dtype == torch.float16:
        bound += 2.0 ** -25
    return out, bound


def check(got, x, positions, rot, weight=None, eps=1e-6):
    want, bound = reference(x.cpu(), positions.cpu(), rot, weight, eps)
    err = (got.cpu().double() - want).abs()
    assert got.dtype == x.dtype and (err <= bound).all(), float((err / bound).nan_to_num(0).max())


def rows(n, heads, dim, dtype, seed, strided=False):
    x = torch.randn(n, heads, dim, generator=torch.Generator().manual_seed(seed)).to(dtype)
    if strided:   # part of a wider row, off the 16-byte grid
        wide = torch.zeros(n, heads * dim + 7, dtype=dtype)
        wide[:, 3:3 + heads * dim] = x.flatten(1)
        return wide.cuda()[:, 3:3 + heads * dim].unflatten(1, (heads, dim))
    return x.cuda()


def places(n, seed, far=100000):
    return torch.randint(0, far, (n,), generator=torch.Generator().manual_seed(seed)).to(torch.int32)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("n,heads,kv_heads,dim,rotary", [(1, 1, 1, 64, 64), (3, 5, 1, 128, 128), (37, 16, 2, 256, 64),
                                                         (130, 8, 8, 64, 16), (17, 7, 3, 128, 48), (9, 4, 2, 256, 256)])
def test_turned(n, heads, kv_heads, dim, rotary, layout, dtype):
    from flash_moe_hip.rotary import Rotary

    g = torch.Generator().manual_seed(n)
    weights = [1 + 0.3 * torch.randn(dim, generator=g) for _ in range(2)]
    for strided in (False, True):
        for scaling in SCALINGS:
            print(n, heads, kv_heads, dim, rotary, layout, dtype, strided, scaling, flush=True)
            rot = Rotary(dim, rotary, base=1e6, layout=layout, scaling=scaling)
            q, k = rows(n, heads, dim, dtype, 1, strided), rows(n, kv_heads, dim, dtype, 2, strided)
            at = places(n, 3)
            for qw, kw in ((None, None), weights, (None, weights[1]), (weights[0], None)):
                got = rot.apply(q, k, at.cuda(), q_weight=None if qw is None else qw.cuda(),
                                k_weight=None if kw is None else kw.cuda(), eps=1e-5)
                check(got[0], q, at, rot, qw, 1e-5)
                check(got[1], k, at, rot, kw, 1e-5)
                if qw is None and rotary < dim:
                    assert torch.equal(got[0][..., rotary:], q[..., rotary:])
            assert rot.status() == 0


@pytest.mark.parametrize("n,heads,kv_heads,dim", [(5000, 32, 8, 128), (2049, 3, 1, 256), (40001, 1, 1, 64)])
def test_many_rows(n, heads, kv_heads, dim):
    from flash_moe_hip.rotary import Rotary

    rot = Rotary(dim, base=500000.0)
    q, k, at = rows(n, heads, dim, torch.bfloat16, 1), rows(n, kv_heads, dim, torch.bfloat16, 2), places(n, 4, 2 ** 20)
    got = rot.apply(q, k, at.cuda())
    check(got[0], q, at, rot)
    check(got[1], k, at, rot)
    assert rot.status() == 0


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_in_place_and_strided_outputs(layout):
    from flash_moe_hip.rotary import Rotary

    rot = Rotary(128, 64, layout=layout)
    at = places(100, 3).cuda()
    for dtype in TYPES:
        wide = torch.randn(100, 10 * 128 + 5, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
        q, k = (wide[:, a:a + h * 128].unflatten(1, (h, 128)) for a, h in ((1, 6), (5 + 768, 4)))
        want = rot.apply(q, k, at)
        to = torch.full((110, 8, 300), 7.0, dtype=dtype, device="cuda")
        outs = to[3:103, 1:7, 9:137], to[3:103, 2:6, 150:278]
        got = rot.apply(q, k, at, out=outs)
        assert got[0] is outs[0] and torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        kept = torch.ones_like(to, dtype=torch.bool)
        kept[3:103, 1:7, 9:137] = kept[3:103, 2:6, 150:278] = False
        assert (to[kept] == 7).all()
        before = wide.clone()
        rot.apply(q, k, at, out=(q, k))
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])
        assert torch.equal(wide[:, 0], before[:, 0]) and torch.equal(wide[:, 769:773], before[:, 769:773])
    assert rot.status() == 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_results_lie_row_by_row(dtype):
    """Inputs of other orders (heads outermost, one row for all) give results in order."""
    from flash_moe_hip.rotary import Rotary

    rot, at = Rotary(64), places(37, 5).cuda()
    q = torch.randn(6, 37, 64, generator=torch.Generator().manual_seed(2)).to(dtype).cuda().transpose(0, 1)
    k = q[:1, :1].expand(37, 2, 64)
    got = rot.apply(q, k, at)
    want = rot.apply(q.contiguous(), k.contiguous(), at)
    for g, w in zip(got, want):
        assert g.is_contiguous() and torch.equal(g, w)


def test_far_and_negative_positions():
    """Every 32-bit position, against angles of 60 digits; a turn back undoes a turn."""
    from flash_moe_hip.rotary import Rotary

    getcontext().prec = 60
    pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494")
    rot = Rotary(64, base=1e6)
    at = [0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 30 + 12345, 999999937, -77777777, 2 ** 24 + 1]
    x = torch.zeros(len(at), 1, 64)
    x[..., :32] = 1.0
    got = rot.apply(x.cuda(), x.cuda(), torch.tensor(at, dtype=torch.int32).cuda())[0].cpu().double()
    for j, p in enumerate(at):
        for i, f in enumerate(rot.frequencies):
            turn = Decimal(p) * Decimal(f) / (2 * pi)
            angle = float((turn - int(turn)) * 2 * pi)
            # (a frequency's turns are a double: two roundings of the quotient by 2 pi)
            bound = 9 * 2.0 ** -24 + abs(p * f) * 2.0 ** -52 + 2.0 ** -31
            assert abs(got[j, 0, i] - math.cos(angle)) <= bound and abs(got[j, 0, 32 + i] - math.sin(angle)) <= bound, (p, i)
    q = rows(50, 4, 64, torch.float32, 5)
    pos = places(50, 6, 2 ** 30).cuda()
    back = rot.apply(*rot.apply(q, q, pos), -pos)[0]
    # two turns' errors, each of at most 8 * 2^-24 (|a| + |b|) (the angles' own cancel)
    assert ((back - q).abs() <= 2 * 9 * 2.0 ** -24 * 2 ** 0.5 * (q.abs() + q.roll(32, 2).abs()) + 1e-9).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_zero_rows_and_values_that_are_not_finite(dtype):
    from flash_moe_hip.rotary import Rotary

    rot = Rotary(128, 64)
    q, k = rows(20, 3, 128, dtype, 1), rows(20, 2, 128, dtype, 2)
    at = places(20, 3).cuda()
    w = torch.ones(128).cuda()
    q[4] = 0
    got = rot.apply(q, k, at, q_weight=w, eps=1e-6)
    assert not got[0][4].any() and rot.status() == 0
    clean = rot.apply(q, k, at)
    q[7, 1, 100], q[9, 2, 3] = math.inf, math.nan     # a channel that stays, one that is turned
    got = rot.apply(q, k, at)
    assert rot.status() == -4 and rot.status() == 0
    assert got[0][7, 1, 100] == math.inf and got[0][9, 2, 3].isnan() and got[0][9, 2, 35].isnan()
    same = torch.ones_like(q, dtype=torch.bool)
    same[7, 1, 100] = same[9, 2, 3] = same[9, 2, 35] = False
    assert torch.equal(got[0][same], clean[0][same]) and torch.equal(got[1], clean[1])
    if dtype == torch.float16:   # two large values that meet
        q = torch.full((1, 1, 128), 60000.0, dtype=dtype, device="cuda")
        rot.apply(q, q, torch.ones(1, dtype=torch.int32, device="cuda"))
        assert rot.status() == -4


def test_large_and_small_rows_are_normed():
    """Sums of squares from FP32's least normal numbers to near its largest."""
    from flash_moe_hip.rotary import Rotary

    rot = Rotary(256, 64)
    at = places(6, 3)
    w = 1 + 0.1 * torch.randn(256, generator=torch.Generator().manual_seed(2))
    for size, eps in ((1e17, 1e-6), (1e-3, 1e-12), (1e-18, 1e-30), (1.0, 10.0)):
        q = rows(6, 2, 256, torch.float32, 8) * size
        check(rot.apply(q, q, at.cuda(), q_weight=w.cuda(), eps=eps)[0], q, at, rot, w, eps)
    assert rot.status() == 0


def test_captured_replayed_other_streams_and_no_tokens():
    from flash_moe_hip.rotary import Rotary

    rot = Rotary(128)
    q, k, at = rows(33, 8, 128, torch.bfloat16, 1), rows(33, 2, 128, torch.bfloat16, 2), places(33, 3).cuda()
    want = [t.clone() for t in rot.apply(q, k, at)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = rot.apply(q, k, at, stream=side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rot.apply(q, k, at)
    for i in range(4):
        at.copy_(places(33, 10 + i))
        graph.replay()
        eager = rot.apply(q, k, at)
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])
    none = rot.apply(q[:0], k[:0], at[:0])
    assert none[0].shape == (0, 8, 128) and none[1].shape == (0, 2, 128) and rot.status() == 0


def test_refusals():
    from flash_moe_hip.rotary import Rotary

    rot = Rotary(128)
    q, k, at = torch.zeros(3, 4, 128, device="cuda"), torch.zeros(3, 2, 128, device="cuda"), torch.zeros(
        3, dtype=torch.int32, device="cuda")
    w = torch.ones(128, device="cuda")
    bad = [
        ((q[0], k, at), {}, "tokens, heads"), ((q, k[:2], at), {}, "shape"), ((q, k.half(), at), {}, "expected one of"),
        ((q.double(), k.double(), at), {}, "expected one of"), ((q[..., :64], k, at), {}, "shape"),
        ((q.cpu(), k, at), {}, "is on cpu"), ((q, k, at.long()), {}, "positions"), ((q, k, at[:2]), {}, "positions"),
        ((q, k, at.cpu()), {}, "is on cpu"), ((q.clone().requires_grad_(), k, at), {}, "no backward"),
        ((q, k, at), dict(q_weight=w.half()), "q_weight"), ((q, k, at), dict(k_weight=w[:64]), "k_weight"),
        ((q, k, at), dict(eps=0.0), "eps"), ((q, k, at), dict(eps=math.nan), "eps"),
        ((q, k, at), dict(out=(q, q)), "out"), ((q, k, at), dict(out=(q.half(), k)), "out"),
        ((q.transpose(1, 2).contiguous().transpose(1, 2), k, at), {}, "contiguous in its last"),
        ((q[:, :0], k, at), {}, "heads must be"),
    ]
    for args, kw, why in bad:
        with pytest.raises(ValueError, match=why):
            rot.apply(*args, **kw)
    assert rot.status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("dim,rotary,layout", [(64, 64, "half"), (128, 48, "interleaved"), (256, 64, "half")])
def test_rows_whose_squares_are_past_fp32_are_normed(dim, rotary, layout, dtype):
    """The norm of rows up to the type's largest numbers, beside rows of ones; weights that the norm's factor alone would
    carry out of range."""
    from flash_moe_hip.rotary import Rotary

    rot = Rotary(dim, rotary, layout=layout)
    at = places(7, 3)
    g = torch.Generator().manual_seed(2)
    for size, weight, eps in ((1e18, 1.0, 1e-6), (1e19, 1.0, 1e-6), (1e25, 1e-20, 1e-6), (5e37, 1.0, 1e30), (5e37, 1e-30, 1e-30),
                              (1e-18, 1e30, 1e-30)):
        w = weight * (1 + 0.1 * torch.randn(dim, generator=g))
        q, k = rows(7, 5, dim, torch.float32, 8), rows(7, 3, dim, torch.float32, 9)
        q[:, ::2], k[2:] = q[:, ::2] * size, k[2:] * size
        q, k = q.to(dtype), k.to(dtype)
        assert q.isfinite().all() and k.isfinite().all()
        print(dim, rotary, layout, dtype, size, weight, eps, flush=True)
        got = rot.apply(q, k, at.cuda(), q_weight=w.cuda(), k_weight=w.cuda(), eps=eps)
        check(got[0], q, at, rot, w, eps)
        check(got[1], k, at, rot, w, eps)
        assert rot.status() == 0
    q[3, 1, 5] = math.inf                # a row that is not finite is reported, the others stay
    clean = got
    got = rot.apply(q, k, at.cuda(), q_weight=w.cuda(), k_weight=w.cuda(), eps=eps)
    assert rot.status() == -4 and got[0][3, 1].isnan().any() and torch.equal(got[1], clean[1])
    got[0][3, 1] = clean[0][3, 1]
    assert torch.equal(got[0], clean[0])
