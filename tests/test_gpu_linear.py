"""Linear attention with a decay per head on the GPU (steps and prompts, with the
delta rule and without) against the recurrence in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import mixer_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def inputs(tokens, heads, key_heads, dk, dv, dtype, delta, seed=0, strided=False):
    g = torch.Generator().manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g)

    def unit(x):   # norm at most 1 after its rounding
        return (torch.nn.functional.normalize(x, dim=-1) * (1 - 2.0 ** -7)).to(dtype)

    q, k = unit(randn(tokens, key_heads, dk)), unit(randn(tokens, key_heads, dk))
    v = randn(tokens, heads, dv).to(dtype)
    if strided:
        rows = torch.cat([torch.zeros(tokens, 3, dtype=dtype)] + [t.flatten(1) for t in (q, k, v)], 1)
        a, b = key_heads * dk, heads * dv
        q, k, v = (rows[:, i:j].unflatten(1, s) for i, j, s in (
            (3, 3 + a, (key_heads, dk)), (3 + a, 3 + 2 * a, (key_heads, dk)), (3 + 2 * a, 3 + 2 * a + b, (heads, dv))))
    rate = torch.exp(-torch.arange(heads) * (8.0 / heads))
    gate = -torch.nn.functional.softplus(randn(tokens, heads)) * rate
    beta = torch.sigmoid(randn(tokens, heads)) if delta else None
    if strided:
        gate = torch.cat([gate, gate], 1)[:, :heads]
    return q, k, v, beta, gate


def cuda(args):
    """To the GPU with their strides."""
    def move(t):
        if t is None or t.is_contiguous():
            return None if t is None else t.cuda()
        base = torch.empty(0, dtype=t.dtype).set_(t.untyped_storage()).cuda()
        return base.as_strided(t.shape, t.stride(), t.storage_offset())

    return [move(t) for t in args]


def close(got, want, size, tokens, dk, dtype=None):
    err = (got.cpu().double() - want).abs()
    tol = ref.linear_bound(size, tokens, dk)
    if dtype is not None:   # an output of that type
        tol = tol + ref.half_step(dtype) * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
        assert (err <= tol).all(), f"{float((err / tol).max()):.3g} of the bound"
    else:
        assert (err.norm(dim=-1) <= tol).all(), f"{float((err.norm(dim=-1) / tol).max()):.3g} of the bound"


DIMS = [   # heads, key_heads, key_dim, value_dim
    (1, 1, 4, 4), (4, 2, 16, 32), (6, 2, 80, 100), (2, 2, 64, 16), (4, 1, 128, 128), (2, 1, 256, 48), (3, 3, 36, 1024),
    (1, 1, 200, 256),
]


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dims", DIMS, ids=str)
def test_steps(dims, dtype, delta):
    from flash_moe_hip.linear_attention import LinearState

    heads, key_heads, dk, dv = dims
    for seqs in (1, 5):
        print(seqs, dims, dtype, delta, flush=True)
        g = torch.Generator().manual_seed(7)
        start = torch.randn(seqs, heads, dv, dk, generator=g) * 0.1
        st = LinearState(seqs, heads, dv, dk, state=start.cuda())
        steps = [inputs(seqs, heads, key_heads, dk, dv, dtype, delta, seed=i, strided=i == 1) for i in range(3)]
        got = [st.step(*cuda(a)) for a in steps]
        assert st.status() == 0
        for b in range(seqs):
            rows = [None if t[0] is None else torch.stack([x[b] for x in t]) for t in zip(*steps)]
            want, state, size = ref.linear(start[b], *rows)
            close(torch.stack([x[b] for x in got]), want, size, 3, dk, dtype)
            close(st.state[b], state, size, 3, dk)


PROMPTS = [   # tokens of the sequences
    [1], [2], [64], [65], [63, 1, 130], [0, 200, 0, 7], [300],
]


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("parts", PROMPTS, ids=str)
@pytest.mark.parametrize("dims", DIMS, ids=str)
def test_prompts(dims, parts, dtype, delta):
    from flash_moe_hip.linear_attention import LinearState

    print(dims, parts, dtype, delta, flush=True)
    heads, key_heads, dk, dv = dims
    n = sum(parts)
    args = inputs(n, heads, key_heads, dk, dv, dtype, delta, seed=n, strided=len(parts) > 1)
    g = torch.Generator().manual_seed(7)
    start = torch.randn(len(parts), heads, dv, dk, generator=g) * 0.1
    st = LinearState(len(parts), heads, dv, dk, state=start.cuda())
    starts = torch.tensor([0] + parts).cumsum(0).to(torch.int32).cuda() if len(parts) > 1 else None
    got = st.prefill(*cuda(args), starts=starts)
    assert st.status() == 0 and got.dtype == dtype
    at = 0
    for b, m in enumerate(parts):
        rows = [None if t is None else t[at:at + m] for t in args]
        want, state, size = ref.linear(start[b], *rows)
        close(got[at:at + m], want, size, m, dk, dtype)
        close(st.state[b], state, size, m, dk)
        at += m


@pytest.mark.parametrize("delta", [True, False])
def test_a_prompt_in_pieces_and_steps_goes_on_where_it_stopped(delta):
    from flash_moe_hip.linear_attention import LinearState

    args = inputs(150, 4, 2, 64, 32, torch.float32, delta, seed=4)
    want, state, size = ref.linear(torch.zeros(4, 32, 64), *args)
    st = LinearState(1, 4, 32, 64)
    rows = cuda(args)
    cut = [None if t is None else t[:70] for t in rows]
    got = [st.prefill(*cut)]
    for t in range(70, 75):
        got.append(st.step(*[None if x is None else x[t:t + 1] for x in rows]))
    got.append(st.prefill(*[None if x is None else x[75:] for x in rows]))
    close(torch.cat(got), want, size, 64 * 9, 64, torch.float32)   # (a piece is a chunk more at most)
    close(st.state[0], state, size, 64 * 9, 64)
    st.reset()
    assert not st.state.any()


def test_delta_state_prefill_and_step():
    """DeltaState: prompt, then the bit-exact step from where it ended."""
    from flash_moe_hip.native_expert import DeltaState

    q, k, v, beta, gate = args = inputs(131, 8, 8, 128, 128, torch.float32, True, seed=11)
    want, state, size = ref.linear(torch.zeros(8, 128, 128), *args)
    ds = DeltaState(8, 128, 128)
    out = ds.prefill(*cuda([t[:130] for t in args]))
    last = ds.step(*cuda([t[130] for t in args]))
    assert ds.status() == 0
    close(torch.cat([out, last.unsqueeze(0)]), want, size, 131, 128, torch.float32)
    close(ds.state, state, size, 131, 128)
    with pytest.raises(ValueError, match="multiple of 4"):
        DeltaState(2, 6, 7).prefill(*cuda(inputs(3, 2, 2, 7, 6, torch.float32, True)))


@pytest.mark.parametrize("delta", [True, False])
def test_gates_at_their_ends(delta):
    """A gate of -inf forgets everything before its token; gates of 0 nothing; far gates keep their digits."""
    from flash_moe_hip.linear_attention import LinearState

    heads, n = 4, 140
    q, k, v, beta, gate = inputs(n, heads, 1, 64, 32, torch.float32, delta, seed=2)
    gate[:, 0] = 0.0
    gate[:, 1] = -0.01
    gate[3, 1] = gate[70, 1] = -math.inf
    gate[:, 2] = -1e-3
    gate[5, 2] = -9000.0
    gate[100, 2] = -3e38
    gate[:, 3] = -60.0
    args = q, k, v, beta, gate
    start = torch.randn(heads, 32, 64, generator=torch.Generator().manual_seed(3))
    want, state, size = ref.linear(start, *args)
    st = LinearState(1, heads, 32, 64, state=start.unsqueeze(0).cuda())
    got = st.prefill(*cuda(args))
    close(got, want, size, n, 64, torch.float32)
    close(st.state[0], state, size, n, 64)
    st = LinearState(1, heads, 32, 64, state=start.unsqueeze(0).cuda())
    rows = cuda(args)
    got = torch.cat([st.step(*[None if x is None else x[t:t + 1] for x in rows]) for t in range(n)])
    close(got, want, size, 64 * n, 64, torch.float32)   # (each step rounds as a chunk)
    assert st.status() == 0


@pytest.mark.parametrize("beta_of", [1.0, 0.9, 0.0])
def test_repeated_keys(beta_of):
    """The same key at every token, no decay: the triangular system at its worst."""
    from flash_moe_hip.linear_attention import LinearState

    q, k, v, beta, gate = inputs(200, 2, 2, 64, 32, torch.float32, True, seed=5)
    k[:] = k[:1]
    beta[:] = beta_of
    gate[:] = 0.0
    args = q, k, v, beta, gate
    want, state, size = ref.linear(torch.zeros(2, 32, 64), *args)
    st = LinearState(1, 2, 32, 64)
    close(st.prefill(*cuda(args)), want, size, 200, 64, torch.float32)
    close(st.state[0], state, size, 200, 64)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("delta", [True, False])
def test_a_value_that_is_not_finite_stays_in_its_sequence_and_row(delta, dtype):
    from flash_moe_hip.linear_attention import LinearState

    args = inputs(200, 2, 2, 64, 32, dtype, delta, seed=6)
    starts = torch.tensor([0, 90, 200], dtype=torch.int32).cuda()
    st = LinearState(2, 2, 32, 64)
    clean = st.prefill(*cuda(args), starts=starts)
    kept = st.state.clone()
    assert st.status() == 0
    args[2][70, 1, 3] = math.nan   # sequence 0, second chunk, head 1, value row 3
    st.reset()
    got = st.prefill(*cuda(args), starts=starts)
    assert st.status() == -4 and st.status() == 0
    assert torch.equal(got[:64], clean[:64]) and torch.equal(got[90:], clean[90:])
    others = [r for r in range(32) if r != 3]
    assert torch.equal(got[:, 0], clean[:, 0]) and torch.equal(got[:, 1][:, others], clean[:, 1][:, others])
    assert got[70:90, 1, 3].isnan().all() and st.state[0, 1, 3].isnan().all()
    assert torch.equal(st.state[1], kept[1])
    # a step from a state that is not finite
    one = [None if t is None else t[:2] for t in cuda(args)]
    assert st.step(*one)[0, 1, 3].isnan() and st.status() == -4


@pytest.mark.parametrize("delta", [True, False])
def test_rows_of_no_sequence_and_bad_starts(delta):
    from flash_moe_hip.linear_attention import LinearState

    args = inputs(100, 2, 1, 64, 32, torch.bfloat16, delta, seed=8)
    st = LinearState(2, 2, 32, 64)
    out = torch.full((100, 2, 32), 7.0, dtype=torch.bfloat16, device="cuda")
    starts = torch.tensor([5, 70, 90], dtype=torch.int32)
    assert st.prefill(*cuda(args), starts=starts.cuda(), out=out) is out
    assert st.status() == 0 and (out[:5] == 7).all() and (out[90:] == 7).all()
    for b in range(2):
        i, j = int(starts[b]), int(starts[b + 1])
        want, state, size = ref.linear(torch.zeros(2, 32, 64), *[None if t is None else t[i:j] for t in args])
        close(out[i:j], want, size, j - i, 64, torch.bfloat16)
        close(st.state[b], state, size, j - i, 64)
    for bad in ([0, 70, 30], [-1, 50, 100], [0, 50, 101]):
        st.prefill(*cuda(args), starts=torch.tensor(bad, dtype=torch.int32).cuda())
        assert st.status() == -9, bad


def test_no_tokens():
    from flash_moe_hip.linear_attention import LinearState

    st = LinearState(1, 2, 32, 64)
    assert st.prefill(*cuda(inputs(0, 2, 2, 64, 32, torch.float32, True))).shape == (0, 2, 32)


def test_many_sequences():
    from flash_moe_hip.linear_attention import LinearState

    parts = [(i * 29) % 71 for i in range(100)]
    n = sum(parts)
    args = inputs(n, 2, 1, 16, 8, torch.float32, True, seed=9)
    st = LinearState(100, 2, 8, 16)
    got = st.prefill(*cuda(args), starts=torch.tensor([0] + parts).cumsum(0).to(torch.int32).cuda())
    at = 0
    for b, m in enumerate(parts):
        want, state, size = ref.linear(torch.zeros(2, 8, 16), *[t[at:at + m] for t in args])
        close(got[at:at + m], want, size, m, 16, torch.float32)
        close(st.state[b], state, size, m, 16)
        at += m


def test_a_prompt_of_several_passes():
    """More chunks than the workspace holds: the same bits as in two calls at a chunk's end."""
    from flash_moe_hip import _lib
    from flash_moe_hip.linear_attention import LinearState

    heads, dk, dv, n = 64, 256, 512, 4200
    lib = _lib.load()
    size = [lib.mqh_linear_prefill_workspace_bytes(t, 1, heads, dk, dv, 0) for t in (n, 2 * n)]
    assert size[0] == size[1]   # as large as it gets
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k = (torch.nn.functional.normalize(torch.randn(n, 1, dk, generator=g, device="cuda"), dim=2) for _ in range(2))
    v = torch.randn(n, heads, dv, generator=g, device="cuda")
    gate = -torch.rand(n, heads, generator=g, device="cuda")
    one, two = (LinearState(1, heads, dv, dk) for _ in range(2))
    got = one.prefill(q, k, v, None, gate)
    cut = 64 * 32
    parts = [two.prefill(*[t[a:b] if t is not None else None for t in (q, k, v, None, gate)])
             for a, b in ((0, cut), (cut, n))]
    assert torch.equal(got, torch.cat(parts)) and torch.equal(one.state, two.state) and one.status() == 0


@pytest.mark.parametrize("delta", [True, False])
def test_captured_replayed_and_other_streams(delta):
    from flash_moe_hip.linear_attention import LinearState

    args = cuda(inputs(150, 4, 2, 64, 32, torch.bfloat16, delta, seed=3))
    other = cuda(inputs(150, 4, 2, 64, 32, torch.bfloat16, delta, seed=4))
    starts = torch.tensor([0, 40, 150], dtype=torch.int32).cuda()

    def eager(rows, calls=1, stream=None):
        st = LinearState(2, 4, 32, 64)
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
        for _ in range(calls):
            a = st.prefill(*rows, starts=starts, stream=stream)
            b = st.step(*[None if t is None else t[:2] for t in rows], stream=stream)
        if stream is not None:
            stream.synchronize()
        return a, b, st.state

    want = [eager(r, 1) for r in (args, other)]
    side = eager(args, 1, torch.cuda.Stream())
    assert all(torch.equal(x, y) for x, y in zip(side, want[0]))
    graphs = []
    for rows in (args, other):
        st = LinearState(2, 4, 32, 64)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a = st.prefill(*rows, starts=starts)
            b = st.step(*[None if t is None else t[:2] for t in rows])
        graphs.append((graph, a, b, st))
    for turn in range(3):
        for (graph, a, b, st), w, rows in zip(graphs, want, (args, other)):
            st.reset()
            graph.replay()
            again = eager(rows)
            assert all(torch.equal(x, y) for x, y in zip((a, b, st.state), w))
            assert all(torch.equal(x, y) for x, y in zip(again, w))
            assert st.status() == 0


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("dtype,value", [(torch.float16, 6e4), (torch.bfloat16, 3.3895e38)], ids=str)
def test_outputs_their_type_cannot_hold_are_reported(dtype, value, delta):
    """An FP32 output that is finite and rounds to infinity: writes of two tokens under one query."""
    from flash_moe_hip.linear_attention import LinearState

    v = torch.zeros(2, 1, 16, dtype=dtype)
    v[0], v[1, 0, 5] = 1.0, value
    q, k = torch.zeros(2, 1, 16, dtype=dtype), torch.zeros(2, 1, 16, dtype=dtype)
    k[0, 0, 0] = k[1, 0, 1] = 1.0   # orthogonal keys: beta 1 writes each value as it is
    q[:, 0, :2] = 1.0
    v[0, 0, 5] = value * 0.003 if dtype == torch.bfloat16 else value
    gate, beta = torch.zeros(2, 1), torch.ones(2, 1) if delta else None
    rows = cuda([q, k, v, beta, gate])
    for prompt in (False, True):
        st = LinearState(1, 1, 16, 16)
        if prompt:
            got = st.prefill(*rows)[1]
        else:
            got = [st.step(*[None if t is None else t[i:i + 1] for t in rows]) for i in range(2)][1][0]
        assert st.state.isfinite().all()
        assert got[0, 5].isinf() and got[0, :5].isfinite().all() and st.status() == -4, prompt
        st.reset()
        st.step(*[None if t is None else t[:1] for t in rows])
        assert st.status() == 0


@pytest.mark.parametrize("delta", [True, False])
def test_strides_past_32_bits_of_a_chunk(delta):
    """Steps over one token of a long buffer, prompts with the heads outside the tokens, one token of any stride."""
    from flash_moe_hip.linear_attention import LinearState

    heads, key_heads, dk, dv, far = 4, 2, 64, 32, 2 ** 22 + 8

    def spread(t, strides):   # the same rows a stride apart
        at = sum((n - 1) * s for n, s in zip(t.shape, strides)) + t.shape[-1]
        base = torch.zeros(at, dtype=t.dtype, device="cuda")
        return base.as_strided(t.shape, strides).copy_(t)

    args = inputs(3, heads, key_heads, dk, dv, torch.bfloat16, delta, seed=5)
    one, two = LinearState(3, heads, dv, dk), LinearState(3, heads, dv, dk)
    apart = [None if t is None else spread(t, (far,) + ((far * 4, 1) if t.dim() == 3 else (1,))) for t in args]
    assert torch.equal(one.step(*cuda(args)), two.step(*apart)) and torch.equal(one.state, two.state)

    args = inputs(100, heads, key_heads, dk, dv, torch.float32, delta, seed=6)
    q, k, v, beta, gate = args
    apart = [spread(t, (dim, far, 1)) for t, dim in ((q, dk), (k, dk), (v, dv))]
    apart += [None if t is None else spread(t, (2 ** 22 + 4, 1)) for t in (beta, gate)]
    one, two = LinearState(1, heads, dv, dk), LinearState(1, heads, dv, dk)
    assert torch.equal(one.prefill(*cuda(args)), two.prefill(*apart)) and torch.equal(one.state, two.state)

    rows = cuda([None if t is None else t[:1] for t in args])
    single = [None if t is None else t.as_strided(t.shape, (2 ** 30,) + t.stride()[1:]) for t in rows]
    assert torch.equal(one.prefill(*rows), two.prefill(*single))
    assert torch.equal(one.step(*rows), two.step(*single)) and torch.equal(one.state, two.state)
    assert one.status() == 0 and two.status() == 0
    with pytest.raises(ValueError, match="token stride"):
        one.prefill(*[None if t is None else spread(t[:2], (far,) + t.stride()[1:]) for t in args])


def test_products_of_a_prompts_outputs_to_fp32():
    """Outputs that are one product each, of the state and q or of a write and q k: what the kernel leaves out of a
    product and its roundings are counted.  The two factors are sums of three BF16 numbers to nearest (off by at most
    2^-8 of what they stand for, each the rest of the one before), and the products of the second with the third or
    less are left out: two of at most 2^-24 of the term, and 2^-32.  The six others are added in FP32 (five roundings,
    the partial sums at most 1.02 of the term)."""
    from flash_moe_hip.linear_attention import LinearState

    g = torch.Generator().manual_seed(0)
    i = torch.arange(64)
    # all bits of the second and third part set, for every first part; and any numbers
    x = torch.stack([1 + (i % 64) / 64 - 2.0 ** -23 * (1 + i % 5), 1 + (2 * i + 1) / 128 - 2.0 ** -23,
                     torch.randn(64, generator=g), torch.rand(64, generator=g) + 1])
    y = torch.stack([x[0].flip(0), 1 + (2 * i + 1) / 128 - 2.0 ** -22, torch.randn(64, generator=g), x[3].roll(9)])
    x, y = torch.cat([x, x]), torch.cat([y, x])
    heads = x.shape[0]
    tol = (2.0 ** -23 + 2.0 ** -32 + 5 * 1.02 * 2.0 ** -24) * (x.double() * y.double()).abs() * 1.001
    none, gate = torch.zeros(1, heads, 64), torch.zeros(1, heads)
    # the state: row r has one entry, in column r
    st = LinearState(1, heads, 64, 64, state=torch.diag_embed(y).unsqueeze(0).cuda())
    got = st.prefill(x.unsqueeze(0).cuda(), none.cuda(), none.cuda(), None, gate.cuda())[0].cpu().double()
    err = (got - x.double() * y.double()).abs()
    assert (err <= tol).all(), f"{float((err / tol).max()):.3g} of the bound"
    # a write: (q k) v of one token, a head for every x
    n = heads * 64
    one = torch.zeros(1, n, 64)
    one[:, :, 3] = 1.0
    k = torch.zeros(1, n, 64)
    k[0, :, 3] = x.flatten()
    st = LinearState(1, n, 4, 64)
    got = st.prefill(one.cuda(), k.cuda(), y.flatten().view(1, n, 1).expand(1, n, 4).contiguous().cuda(), None,
                     torch.zeros(1, n).cuda())[0, :, 1].cpu().double().view(heads, 64)
    err = (got - x.double() * y.double()).abs()
    assert (err <= tol).all(), f"{float((err / tol).max()):.3g} of the bound"


@pytest.mark.parametrize("delta", [True, False])
def test_several_passes_over_ragged_sequences(delta):
    """Sequences that end before a pass, begin in it, lie inside it, go over its ends, and hold nothing: the same bits
    as each alone in calls of one pass (cut at its chunks' ends), and as the recurrence in 64 bits."""
    from flash_moe_hip import _lib
    from flash_moe_hip.linear_attention import LinearState

    heads, dk, dv, parts = 64, 256, 512, [0, 700, 1500, 0, 30, 64, 900, 1, 0]
    n, seqs = sum(parts), len(parts)
    need = _lib.load().mqh_linear_prefill_workspace_bytes
    assert need(n, seqs, heads, dk, dv, int(delta)) == need(8 * n, seqs, heads, dk, dv, int(delta))   # as large as it gets
    assert need(1216, 1, heads, dk, dv, int(delta)) < need(n, seqs, heads, dk, dv, int(delta))        # one pass
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k = (torch.nn.functional.normalize(torch.randn(n, 1, dk, generator=g, device="cuda"), dim=2) * (1 - 2.0 ** -7)
            for _ in range(2))
    v = torch.randn(n, heads, dv, generator=g, device="cuda")
    gate = -torch.rand(n, heads, generator=g, device="cuda") * 0.1
    beta = torch.rand(n, heads, generator=g, device="cuda") if delta else None
    first = torch.randn(seqs, heads, dv, dk, generator=g, device="cuda") * 0.1
    st = LinearState(seqs, heads, dv, dk, state=first.clone())
    starts = torch.tensor([0] + parts).cumsum(0)
    got = st.prefill(q, k, v, beta, gate, starts=starts.to(torch.int32).cuda())
    assert st.status() == 0
    for b, m in enumerate(parts):
        alone = LinearState(1, heads, dv, dk, state=first[b:b + 1].clone())
        for at in range(int(starts[b]), int(starts[b + 1]), 1216):
            to = min(at + 1216, int(starts[b + 1]))
            out = alone.prefill(*[None if t is None else t[at:to] for t in (q, k, v, beta, gate)])
            assert torch.equal(out, got[at:to]), b
        assert torch.equal(alone.state[0], st.state[b]), b
    b, h = 2, 5
    rows = [None if t is None else t[starts[b]:starts[b + 1]].cpu() for t in (q, k, v, beta, gate)]
    rows = rows[:2] + [None if t is None else t[:, h:h + 1] for t in rows[2:]]
    want, state, size = ref.linear(first[b, h:h + 1].cpu(), *rows)
    close(got[starts[b]:starts[b + 1], h:h + 1], want, size, parts[b], dk, torch.float32)
    close(st.state[b, h:h + 1], state, size, parts[b], dk)
