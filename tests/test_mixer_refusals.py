"""What the token mixers' calls refuse (CPU only: every check precedes any HIP call)."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from flash_moe_hip import _lib

    return _lib.load()


P = C.c_void_p(4096)


def test_cache_constructor():
    from flash_moe_hip.kv_cache import PagedCache

    def make(shape=(2, 2, 16, 64), dtype=torch.float16, **kw):
        return PagedCache(torch.zeros(shape, dtype=dtype), torch.zeros(shape, dtype=dtype), **kw)

    with pytest.raises(ValueError, match="CUDA device"):
        make()
    with pytest.raises(ValueError, match="head_dim"):
        make((2, 2, 16, 96))
    with pytest.raises(ValueError, match="page_size"):
        make((2, 2, 24, 64))
    with pytest.raises(ValueError, match="page_size"):
        make((2, 2, 8, 64))
    with pytest.raises(ValueError, match="int8"):
        make(dtype=torch.float32)
    with pytest.raises(ValueError, match="k_scale"):
        make(dtype=torch.int8)
    with pytest.raises(ValueError, match="scales must be"):
        make(dtype=torch.int8, k_scale=torch.zeros(2, 2, 8), v_scale=torch.zeros(2, 2, 16))
    with pytest.raises(ValueError, match="only int8"):
        make(k_scale=torch.zeros(2, 2, 16), v_scale=torch.zeros(2, 2, 16))
    with pytest.raises(ValueError, match="one type"):
        PagedCache(torch.zeros(2, 2, 16, 64, dtype=torch.float16), torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16))


def kv_write(lib, **kw):
    a = dict(k=P, kt=256, kh=64, v=P, vt=256, vh=64, type=1, slots=P, tokens=4, kc=P, vc=P, ks=None, vs=None, ct=1,
             pages=4, heads=2, page=16, dim=64, flags=P, stream=None)
    a.update(kw)
    return lib.mqh_kv_write(*a.values())


def test_write_codes(lib):
    for bad in (dict(k=None), dict(v=None), dict(slots=None), dict(kc=None), dict(vc=None), dict(flags=None),
                dict(tokens=0), dict(pages=0), dict(heads=0), dict(heads=1025), dict(page=24), dict(page=8),
                dict(page=2048), dict(kc=C.c_void_p(4098)), dict(ct=3), dict(ct=3, ks=P, vs=C.c_void_p(4100)),
                dict(k=C.c_void_p(4097)), dict(type=0, v=C.c_void_p(4098)), dict(pages=2 ** 31)):
        assert kv_write(lib, **bad) == -1, bad
    for bad in (dict(type=3), dict(type=7), dict(ct=0), dict(dim=96), dict(dim=32)):
        assert kv_write(lib, **bad) == -2, bad
    assert lib.mqh_kv_write_words(None) == -1 and lib.mqh_kv_read_words(None) == -1
    assert lib.mqh_attend_words(None) == -1


def test_read_codes(lib):
    def read(**kw):
        a = dict(slots=P, tokens=4, kc=P, vc=P, ks=None, vs=None, ct=1, pages=4, heads=2, page=16, dim=64, k=P, v=P,
                 type=1, flags=P, stream=None)
        a.update(kw)
        return lib.mqh_kv_read(*a.values())

    for bad in (dict(slots=None), dict(k=None), dict(v=C.c_void_p(4104)), dict(tokens=-1), dict(flags=None)):
        assert read(**bad) == -1, bad
    assert read(type=3) == -2 and read(ct=4) == -2 and read(dim=100) == -2


def attend(lib, **kw):
    a = dict(q=P, qt=512, qh=64, q_type=1, tokens=4, starts=P, seqs=2, heads=8, kc=P, vc=P, ks=None, vs=None, ct=1,
             pages=4, kv=2, page=16, dim=64, table=P, stride=4, cols=4, lengths=P, scale=0.125, out=P, ws=P,
             bytes=1 << 30, flags=P, stream=None)
    a.update(kw)
    return lib.mqh_attend(*a.values())


def test_attend_codes(lib):
    for bad in (dict(q=None), dict(table=None), dict(lengths=None), dict(out=None), dict(flags=None), dict(tokens=0),
                dict(seqs=0), dict(heads=7), dict(heads=0), dict(heads=258), dict(starts=None), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(out=C.c_void_p(4098)),
                dict(q=C.c_void_p(4097)), dict(cols=0), dict(stride=3), dict(kc=None), dict(page=17)):
        assert attend(lib, **bad) == -1, bad
    for bad in (dict(q_type=2), dict(q_type=0), dict(ct=2), dict(dim=80), dict(ct=0)):
        assert attend(lib, **bad) == -2, bad
    # a split call needs its workspace
    long = dict(cols=4096, stride=4096)
    need = lib.mqh_attend_workspace_bytes(4, 2, 0, 8, 2, 64, 4096 * 16)
    assert need > 0 and need % 256 == 0
    assert attend(lib, bytes=need - 1, **long) == -6
    assert attend(lib, ws=None, **long) == -1
    assert attend(lib, ws=C.c_void_p(4096 + 16), **long) == -1
    assert lib.mqh_attend_workspace_bytes(4, 2, 1, 8, 2, 64, 64) == -1
    assert lib.mqh_attend_workspace_bytes(4, 2, 0, 8, 3, 64, 64) == -1
    assert lib.mqh_attend_workspace_bytes(4096, 1, 0, 32, 8, 128, 4096) >= 0


def linear(lib, prompt=False, **kw):
    a = dict(q=P, qt=64, qh=16, k=P, kt=64, kh=16, v=P, vt=64, vh=16, type=0, beta=P, bt=4, gate=P, gt=4, state=P, out=P)
    if prompt:
        a.update(starts=P, tokens=8, seqs=2, heads=4, key_heads=4, key_dim=16, value_dim=16, ws=P, bytes=1 << 30)
    else:
        a.update(seqs=2, heads=4, key_heads=4, key_dim=16, value_dim=16)
    a.update(flags=P, stream=None)
    a.update(kw)
    return (lib.mqh_linear_prefill if prompt else lib.mqh_linear_step)(*a.values())


@pytest.mark.parametrize("prompt", [False, True])
def test_linear_codes(lib, prompt):
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(gate=None), dict(state=None), dict(out=None),
                dict(flags=None), dict(seqs=0), dict(heads=0), dict(heads=6), dict(key_heads=0), dict(heads=4100),
                dict(state=C.c_void_p(4100)), dict(q=C.c_void_p(4098)), dict(out=C.c_void_p(4098))):
        assert linear(lib, prompt, **bad) == -1, bad
    for bad in (dict(type=3), dict(key_dim=15), dict(key_dim=260), dict(value_dim=18), dict(value_dim=1028),
                dict(key_dim=0)):
        assert linear(lib, prompt, **bad) == -2, bad
    assert lib.mqh_linear_step_words(None) == -1 and lib.mqh_linear_prefill_words(None) == -1


def test_counts_past_32_bits_are_refused(lib):
    """The word forms: 2^32 + 4 tokens are not 4."""
    import struct

    p, n = 4096, 2 ** 32 + 4
    cache = [p, p, 0, 0, 1, 4, 2, 16, 64]
    assert lib.mqh_kv_write_words(struct.pack("20q", p, 128, 64, p, 128, 64, 1, p, n, *cache, p, 0)) == -1
    assert lib.mqh_kv_read_words(struct.pack("16q", p, n, *cache, p, p, 1, p, 0)) == -1
    for tokens, seqs, cols in ((n, 2, 4), (4, n, 4), (4, 2, n)):
        assert lib.mqh_attend_words(struct.pack("21qd5q", p, 512, 64, 1, tokens, p, seqs, 8, *cache, p, cols, cols, p,
                                                0.125, p, p, 1 << 30, p, 0)) == -1
    rows = [p, 64, 16, p, 64, 16, p, 64, 16, 0, p, 4, p, 4, p, p]
    assert lib.mqh_linear_step_words(struct.pack("23q", *rows, n, 4, 4, 16, 16, p, 0)) == -1
    for tokens, seqs in ((n, 2), (8, n)):
        assert lib.mqh_linear_prefill_words(struct.pack("27q", *rows, p, tokens, seqs, 4, 4, 16, 16, p, 1 << 30, p, 0)) == -1


def test_strides_past_a_chunk_are_refused(lib):
    for name in ("qt", "qh", "kt", "kh", "vt", "vh", "bt", "gt"):
        for prompt in (False, True):
            assert linear(lib, prompt, **{name: 2 ** 22 + 1}) == -1
            assert linear(lib, prompt, **{name: -1}) == -1


def test_linear_prompt_codes(lib):
    need = lib.mqh_linear_prefill_workspace_bytes(8, 2, 4, 16, 16, 1)
    assert need > lib.mqh_linear_prefill_workspace_bytes(8, 2, 4, 16, 16, 0) > 0
    assert linear(lib, True, bytes=need - 1) == -6
    assert linear(lib, True, tokens=0) == -1
    assert linear(lib, True, starts=None) == -1
    assert linear(lib, True, ws=None) == -1
    assert linear(lib, True, ws=C.c_void_p(4096 + 64)) == -1
    assert lib.mqh_linear_prefill_workspace_bytes(8, 2, 4, 18, 16, 1) == -1
    assert lib.mqh_linear_prefill_workspace_bytes(0, 2, 4, 16, 16, 1) == -1


def test_linear_state_constructor():
    from flash_moe_hip.linear_attention import LinearState

    with pytest.raises(ValueError, match="multiple of 4"):
        LinearState(1, 2, 16, 18, device="cpu")
    with pytest.raises(ValueError, match="multiple of 4"):
        LinearState(1, 2, 16, 260, device="cpu")
    with pytest.raises(ValueError, match="at least 1"):
        LinearState(0, 2, 16, 16, device="cpu")
    with pytest.raises(ValueError, match="CUDA device"):
        LinearState(1, 2, 16, 16, device="cpu")
    with pytest.raises(ValueError, match="shape"):
        LinearState(1, 2, 16, 16, state=torch.zeros(1, 2, 16, 8))
    with pytest.raises(ValueError, match="no backward"):
        LinearState(1, 2, 16, 16, state=torch.zeros(1, 2, 16, 16, requires_grad=True))


def test_row_checks():
    from flash_moe_hip.kv_cache import check_index, check_rows

    cpu, types = -1, (torch.float32, torch.float16)
    x = torch.zeros(4, 2, 64)
    check_rows(x, (4, 2, 64), types, cpu, "x")
    check_rows(torch.zeros(4, 200)[:, 3:131].unflatten(1, (2, 64)), (4, 2, 64), types, cpu, "x")
    for bad, why in ((x[:3], "shape"), (x.double(), "expected one of"), (x.transpose(0, 2), "shape"),
                     (torch.zeros(4, 64, 2).transpose(1, 2), "contiguous"), (x.clone().requires_grad_(), "backward")):
        with pytest.raises(ValueError, match=why):
            check_rows(bad, (4, 2, 64), types, cpu, "x")
    with pytest.raises(ValueError, match="on cpu"):
        check_rows(x, (4, 2, 64), types, 0, "x")
    i = torch.zeros(6, dtype=torch.int32)
    check_index(i, (6,), torch.int32, cpu, "i")
    for bad in (i[:5], i.long(), torch.zeros(12, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="contiguous"):
            check_index(bad, (6,), torch.int32, cpu, "i")
    with pytest.raises(ValueError, match="on cpu"):
        check_index(i, (6,), torch.int32, 0, "i")


def rows_of_stride(tokens, heads, dim, token, head):
    """[tokens, heads, dim] of any strides, without memory."""
    return torch.empty(0, device="meta").as_strided((tokens, heads, dim), (token, head, 1))


def test_strides_of_prompts_that_are_refused_by_name(monkeypatch):
    """Only a chunk's own token offsets are 32-bit: q, k and v of more than one token."""
    from flash_moe_hip import linear_attention as la

    far, near = 2 ** 22 + 4, 64
    state = torch.empty(2, 4, 16, 16, device="meta")
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: 4096)

    def inputs(prompt, n=8, q=near, k=near, v=near, head=16, gate=4):
        return la._inputs(state, n, rows_of_stride(n, 4, 16, q, head), rows_of_stride(n, 4, 16, k, head),
                          rows_of_stride(n, 4, 16, v, head), None,
                          torch.empty(0, device="meta").as_strided((n, 4), (gate, 1)), None, prompt)

    for name in "qkv":
        with pytest.raises(ValueError, match=f"{name} .*4194304"):
            inputs(True, **{name: far})
        inputs(False, n=2, **{name: far})   # a step
        inputs(True, n=1, **{name: far})    # one token: its stride means nothing
    inputs(True, head=far, gate=far)


def test_strides_that_the_word_forms_refuse(lib):
    import struct

    p = 4096

    def words(q=64, qh=16, bt=4, **_):
        return [p, q, qh, p, 64, 16, p, 64, 16, 0, p, bt, p, 4, p, p]

    def step(**kw):
        return lib.mqh_linear_step_words(struct.pack("23q", *words(**kw), 2, 4, 4, 16, 16, p, 0))

    def prompt(tokens=8, **kw):
        return lib.mqh_linear_prefill_words(struct.pack("27q", *words(**kw), p, tokens, 2, 4, 4, 16, 16, p, 1 << 30, p, 0))

    for call in (step, prompt):
        for bad in (dict(q=-1), dict(qh=-1), dict(bt=-1), dict(q=2 ** 41), dict(qh=2 ** 41), dict(bt=2 ** 41)):
            assert call(**bad) == -1, bad
    assert prompt(q=2 ** 22 + 1) == -1


def test_states_put_in_place_of_the_checked_one():
    """A state of another shape, type, device or layout than the object was made for is refused at the call."""
    from flash_moe_hip.linear_attention import LinearState
    from flash_moe_hip.native_expert import DeltaState

    good = torch.zeros(2, 4, 16, 16)
    rows = [torch.zeros(2, 4, 16) for _ in range(3)] + [None, torch.zeros(2, 4)]
    for bad in (good[:1], torch.zeros(2, 4, 16, 8), good.half(), good.transpose(2, 3).contiguous().transpose(2, 3),
                good.clone().requires_grad_()):
        st = LinearState.__new__(LinearState)   # (a CPU has none to make)
        st.shape, st._index, st.state = (2, 4, 16, 16), 0, bad
        for call in (st.step, st.prefill):
            with pytest.raises(ValueError, match="the state must be"):
                call(*rows)
    st.state = good
    with pytest.raises(ValueError, match="expected cuda:0"):
        st.step(*rows)
    one = [t if t is None else t[:1] for t in rows]
    for bad in (torch.zeros(4, 16, 8), good[:, 0], good[0].half(), good[0].transpose(1, 2), torch.zeros(4, 256)):
        ds = DeltaState.__new__(DeltaState)
        ds.shape, ds._flags, ds.state = (4, 16, 16), torch.zeros(64, dtype=torch.int32), bad
        with pytest.raises(ValueError, match="the state must be"):
            ds.prefill(*one)
    ds.state = good[0]
    with pytest.raises(ValueError, match="CUDA device"):
        ds.prefill(*one)


def test_streams_of_another_device(monkeypatch):
    """A launch goes to its stream's device: that has to be the tensors'."""
    from types import SimpleNamespace

    from flash_moe_hip.kv_cache import OnStream

    run = OnStream(torch.device("cuda", 0))
    monkeypatch.setattr(torch.cuda, "stream", lambda s: pytest.fail("the call went on"))
    with pytest.raises(ValueError, match="stream is on cuda:1, expected cuda:0"):
        run(SimpleNamespace(device=torch.device("cuda", 1), cuda_stream=0), lambda handle: None)
    from flash_moe_hip.linear_attention import LinearState
    from flash_moe_hip.native_expert import DeltaState
    from flash_moe_hip.kv_cache import PagedCache

    for cls in (PagedCache, LinearState):
        x = cls.__new__(cls)
        x._run = run
        x._flags, x.lib = torch.zeros(64, dtype=torch.int32), None
        with pytest.raises(ValueError, match="expected cuda:0"):
            x.status(SimpleNamespace(device=torch.device("cuda", 1), cuda_stream=0))


def test_status_on_the_objects_device(monkeypatch):
    """A default stream's handle is 0 on every device: the object's is made current for the wait and the copy."""
    from contextlib import contextmanager
    from types import SimpleNamespace

    from flash_moe_hip.kv_cache import OnStream, PagedCache
    from flash_moe_hip.linear_attention import LinearState

    seen, now = [], [1]

    @contextmanager
    def device(index):
        was, now[0] = now[0], index
        yield
        now[0] = was

    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(cuda_stream=0))
    run = OnStream(torch.device("cuda", 0))
    run._stream_of = lambda index: 0
    for cls in (PagedCache, LinearState):
        x = cls.__new__(cls)
        x._run, x._flags, x.device = run, torch.zeros(64, dtype=torch.int32), torch.device("cuda", 0)
        x.state = SimpleNamespace(device=x.device)
        x.lib = SimpleNamespace(mqh_status=lambda flags, handle: seen.append(now[0]) or 0)
        assert x.status() == 0
    assert seen == [0, 0] and now == [1]


def test_caches_that_require_grad():
    from flash_moe_hip.kv_cache import PagedCache

    def make(*grads, dtype=torch.float16):
        k, v = (torch.zeros(2, 2, 16, 64, dtype=dtype) for _ in range(2))
        scales = [torch.zeros(2, 2, 16) for _ in range(2)] if dtype == torch.int8 else [None, None]
        held = [k, v, *scales]
        for i in grads:
            held[i].requires_grad_()
        return PagedCache(*held)

    for grads, dtype in (((0,), torch.float16), ((1,), torch.bfloat16), ((2,), torch.int8), ((3,), torch.int8)):
        with pytest.raises(ValueError, match="no backward"):
            make(*grads, dtype=dtype)
    with pytest.raises(ValueError, match="CUDA device"):
        make()


def test_token_counts_whose_workgroups_pass_31_bits(lib):
    """The last workgroup's tokens are counted past the end: room for it."""
    for tokens in (2 ** 31 - 1, 2 ** 30 + 1):
        assert kv_write(lib, tokens=tokens, heads=1) == -1
        assert lib.mqh_kv_read(P, tokens, P, P, None, None, 1, 4, 1, 16, 64, P, P, 1, P, None) == -1


def test_words_of_every_int_argument_past_32_bits(lib):
    import struct

    p = 4096
    cache = [p, p, 0, 0, 1, 4, 2, 16, 64]
    rows = [p, 64, 16, p, 64, 16, p, 64, 16, 0, p, 4, p, 4, p, p]
    calls = (
        (lib.mqh_kv_write_words, "20q", [p, 128, 64, p, 128, 64, 1, p, 4, *cache, p, 0], (6, 8, 13, 15, 16, 17)),
        (lib.mqh_kv_read_words, "16q", [p, 4, *cache, p, p, 1, p, 0], (1, 6, 8, 9, 10, 13)),
        (lib.mqh_attend_words, "21qd5q", [p, 512, 64, 1, 4, p, 2, 8, *cache, p, 4, 4, p, 0.125, p, p, 1 << 30, p, 0],
         (3, 4, 6, 7, 12, 14, 15, 16, 19)),
        (lib.mqh_linear_step_words, "23q", [*rows, 2, 4, 4, 16, 16, p, 0], (9, 16, 17, 18, 19, 20)),
        (lib.mqh_linear_prefill_words, "27q", [*rows, p, 8, 2, 4, 4, 16, 16, p, 1 << 30, p, 0], (9, 17, 18, 19, 20, 21, 22)),
    )
    for call, layout, words, ints in calls:
        for i in ints:
            for far in (2 ** 32, -2 ** 32):
                bad = list(words)
                bad[i] += far
                assert call(struct.pack(layout, *bad)) == -1, (call.__name__, i)


def test_slots_of_positions_that_are_none():
    """A padded batch: a negative position has no slot, one past the table's columns a slot past the cache (which
    write and read report), and neither reads the table out of its bounds."""
    from flash_moe_hip.kv_cache import PagedCache

    c = PagedCache.__new__(PagedCache)
    c.page_size, c.pages = 16, 9
    table = torch.tensor([[3, 5, 8], [7, 1, -1]], dtype=torch.int32)
    seq = torch.tensor([0, 0, 0, 1, 1, 0, 0, 1, 1])
    position = torch.tensor([0, 17, 47, 15, 16, -1, 48, -1000, 2 ** 40])
    want = [48, 81, 143, 127, 16, -1, 144, -1, 144]
    assert c.slots(table, seq, position).tolist() == want
    assert c.slots(table, seq[:7], position[:7].int()).tolist() == want[:7]
    assert (c.slots(table, torch.tensor([1]), torch.tensor([40])) < 0).all()   # a page that is none
    assert c.slots(table[:, :0], seq[:0], position[:0]).tolist() == []
