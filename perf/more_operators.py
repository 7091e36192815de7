"""The operators around a 4-bit paged cache: what is timed of them, their plain forms and their 64-bit results.

Page tables and slots of a batch built on the GPU, rotary positions of queries and keys (with the norm of each head's
row before them or without), a paged key/value cache of 4-bit codes (E2M1 numbers with one power of two a 32 channels)
written and read back, and attention of new tokens over it.  Sizes are generic serving sizes: 64 sequences, 64-token
pages, prompts of thousands of tokens; lengths, head counts and types vary over what a serving program meets.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 32            # channels of one scale
LOWEST = -23          # the least exponent of a scale: half of 2^-23 is FP16's least number


def listed():
    return [
        # the next token of each of 64 sequences: rows to write, a new page for some
        dict(name="pages token 64", op="pages", seqs=64, new=64, prior=2051, page=64, padded=0, ragged=True),
        # prompts of 24 requests, padded to a batch of fixed size
        dict(name="pages prompts 65000", op="pages", seqs=24, new=65000, prior=300, page=16, padded=536, ragged=True),
        # the next token of 64 sequences, q and k as parts of one projection's rows
        dict(name="rotary token 64", op="rotary", tokens=64, heads=32, kv_heads=8, dim=128, rotary=128, layout="half",
             scaling="none", norm=False, dtype="bf16", far=8192, strided=True),
        # a long prompt, its context stretched to 32 times the trained one
        dict(name="rotary prompt 16384", op="rotary", tokens=16384, heads=32, kv_heads=8, dim=128, rotary=128,
             layout="half", scaling="yarn", norm=False, dtype="bf16", far=262144, strided=True),
        # heads normed before a quarter of each is rotated, FP32 activations
        dict(name="rotary normed 4099", op="rotary", tokens=4099, heads=16, kv_heads=2, dim=256, rotary=64,
             layout="interleaved", scaling="none", norm=True, dtype="f32", far=65536, strided=False),
        # one new token of each of 64 sequences quantized into the cache and read back
        dict(name="cache 64 tokens", op="cache", tokens=64, kv_heads=8, dim=128, page=64, src="bf16", out="bf16",
             skipped=0, strided=True),
        # a long prompt quantized into the cache, read back for a program's own use
        dict(name="cache 16384 tokens", op="cache", tokens=16384, kv_heads=8, dim=128, page=64, src="bf16", out="bf16",
             skipped=37, strided=True),
        # a whole prompt at once
        dict(name="attend prompt 8192", op="attend", seqs=1, new=8192, prior=0, heads=32, kv_heads=8, dim=128, page=64,
             q="bf16", ragged=False),
        # chunks of four long prompts
        dict(name="attend chunks 2048", op="attend", seqs=4, new=2048, prior=16384, heads=16, kv_heads=2, dim=256,
             page=64, q="bf16", ragged=True),
        # five drafted tokens of each of eight sequences
        dict(name="attend drafts 40", op="attend", seqs=8, new=40, prior=2051, heads=16, kv_heads=16, dim=64, page=32,
             q="f16", ragged=False),
        # the next token of one long sequence
        dict(name="attend token 1", op="attend", seqs=1, new=1, prior=32770, heads=16, kv_heads=2, dim=256, page=64,
             q="bf16", ragged=False),
        # the next token of each of 64 sequences
        dict(name="attend token 64", op="attend", seqs=64, new=64, prior=8191, heads=32, kv_heads=8, dim=128, page=64,
             q="bf16", ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pages", "rotary", "rotary", "cache", "attend", "attend", "token", "token"])
    if op == "pages":
        seqs = _log(rng, 1, 1024)
        return dict(op=op, seqs=seqs, new=rng.choice([seqs, _log(rng, seqs, 65536)]), prior=_log(rng, 1, 8192),
                    page=rng.choice([16, 32, 64, 128]), padded=rng.choice([0, 0, rng.randint(1, 500)]),
                    ragged=rng.random() < 0.7)
    if op == "rotary":
        kv_heads, dim = rng.choice([1, 2, 5, 8]), rng.choice([64, 128, 256])
        heads = kv_heads * rng.choice([1, 2, 4, 7, 8])
        return dict(op=op, tokens=_log(rng, 1, min(32768, 2 ** 26 // (heads * dim))), heads=heads, kv_heads=kv_heads,
                    dim=dim, rotary=rng.choice([dim, dim, dim // 2, dim // 4, 48]),
                    layout=rng.choice(["half", "half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "yarn", "bands"]), norm=rng.random() < 0.4,
                    dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), far=_log(rng, 1024, 2 ** 20),
                    strided=rng.random() < 0.5)
    if op == "cache":
        kv_heads, dim = rng.choice([1, 2, 5, 8]), rng.choice([64, 128, 256])
        return dict(op=op, tokens=_log(rng, 1, 2 ** 24 // (kv_heads * dim)), kv_heads=kv_heads, dim=dim,
                    page=rng.choice([16, 32, 64, 128]), src=rng.choice(["f32", "bf16", "f16"]),
                    out=rng.choice(["f16", "bf16", "f32"]), skipped=rng.choice([0, 0, 1]), strided=rng.random() < 0.5)
    kv_heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
    group = rng.choice([1, 2, 4, 5, 8, 16])
    case = dict(op="attend", seqs=_log(rng, 1, 8 if op == "attend" else 96), heads=kv_heads * group, kv_heads=kv_heads,
                dim=dim, page=rng.choice([16, 32, 64, 128]), q=rng.choice(["bf16", "f16"]), ragged=rng.random() < 0.6)
    if op == "token":
        room = 2 ** 29 // (case["seqs"] * kv_heads * dim)
        case.update(new=case["seqs"], prior=_log(rng, 1, min(65536, room)))
        return case
    room = 2 ** 35 // (case["heads"] * dim)   # products of a query and a key
    case["new"] = _log(rng, 2 * case["seqs"], min(4096, math.isqrt(room)))
    case["prior"] = rng.choice([0, _log(rng, 1, min(32768, room // case["new"]))])
    return case


# ------------------------------------------------------------------ lengths


def _share(i, ragged):
    """A number in (0, 1], the same for every i unless ragged."""
    return 1.0 - (i * 0.6180339887) % 1.0 if ragged else 1.0


def _spread(total, parts, ragged):
    """total as `parts` whole numbers (some may be 0), in proportion to their shares."""
    w = [_share(i, ragged) for i in range(parts)]
    ends = [int(round(total * sum(w[:i + 1]) / sum(w))) for i in range(parts)]
    return [b - a for a, b in zip([0] + ends, ends)]


def _lengths(case):
    """New tokens of each sequence (one each where there are as many) and the tokens it held before."""
    n = case["seqs"]
    new = [1] * n if case["new"] == n else _spread(case["new"], n, case["ragged"])
    return new, [int(case["prior"] * _share(i, case["ragged"])) for i in range(n)]


# ------------------------------------------------------------------ rotary frequencies


def _scaling(case):
    """How a program states the stretching of its positions."""
    return {"none": None,
            "linear": dict(kind="linear", factor=4.0),
            "yarn": dict(kind="yarn", factor=32.0, original=8192),
            "bands": dict(kind="bands", factor=8.0, original=8192, low=1.0, high=4.0)}[case["scaling"]]


BASE = 1e6


def _frequencies(case):
    """Radians a position of each pair of channels, in 64 bits, and what cosine and sine are multiplied by."""
    rotary, sc = case["rotary"], _scaling(case)
    i = torch.arange(rotary // 2, dtype=torch.float64, device=DEV)
    f = BASE ** (-2.0 * i / rotary)
    if sc is None:
        return f, 1.0
    low = f / sc["factor"]
    if sc["kind"] == "linear":
        return low, 1.0
    if sc["kind"] == "yarn":
        # pairs that turn more than 32 times over the trained context stay, those under once are stretched
        first, last = (rotary * math.log(sc["original"] / (turns * 2 * math.pi)) / (2 * math.log(BASE)) for turns in (32, 1))
        first, last = max(math.floor(first), 0), min(math.ceil(last), rotary - 1)
        ramp = ((i - first) / max(last - first, 0.001)).clamp(0, 1)
        return low * ramp + f * (1 - ramp), 0.1 * math.log(sc["factor"]) + 1.0
    turns = sc["original"] * f / (2 * math.pi)   # over the trained context
    keep = ((turns - sc["low"]) / (sc["high"] - sc["low"])).clamp(0, 1)
    return low * (1 - keep) + f * keep, 1.0


# ------------------------------------------------------------------ inputs


def _packed(parts, strided):
    """Tensors [tokens, heads, dim] as they are, or as parts of one projection's rows."""
    if not strided:
        return parts
    rows = torch.cat([p.flatten(1) for p in parts], 1)
    at, views = 0, []
    for p in parts:
        n = p.shape[1] * p.shape[2]
        views.append(rows[:, at:at + n].unflatten(1, p.shape[1:]))
        at += n
    return views


def _empty_cache(case, pages):
    shape = (pages, case["kv_heads"], case["page"])
    return (torch.zeros(*shape, case["dim"] // 2, dtype=torch.uint8, device=DEV),
            torch.zeros(*shape, case["dim"] // BLOCK, dtype=torch.uint8, device=DEV))


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    state = dict(case)
    if case["op"] == "pages":
        new, before = _lengths(case)
        size, seqs = case["page"], case["seqs"]
        held = [-(-n // size) for n in before]
        cols = max(-(-(n + a) // size) for n, a in zip(before, new)) + 2
        pages = sum(-(-(n + a) // size) for n, a in zip(before, new)) + 5
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        held_t = torch.tensor(held, device=DEV)
        at = held_t.cumsum(0) - held_t
        col = torch.arange(cols, device=DEV)
        mine = col < held_t.unsqueeze(1)
        table = torch.where(mine, order[torch.where(mine, at.unsqueeze(1) + col, 0)], 0)
        free, left = torch.zeros_like(order), pages - sum(held)
        free[:left] = order[sum(held):]
        as_int = dict(dtype=torch.int32, device=DEV)
        state.update(table=table, length=torch.tensor(before, **as_int), free=free, count=torch.tensor([left], **as_int),
                     grown=torch.tensor(new, **as_int), before=torch.tensor(before, **as_int),
                     rows=sum(new) + case["padded"])
        return state
    if case["op"] == "rotary":
        n, dim = case["tokens"], case["dim"]
        q, k = randn(n, case["heads"], dim), randn(n, case["kv_heads"], dim)
        state["queries"], state["keys"] = _packed([t.to(DTYPES[case["dtype"]]) for t in (q, k)], case["strided"])
        # prompts in a row that begin anywhere (single tokens of many sequences: anywhere each)
        run_of = 1 if n <= 256 else 1024
        first = torch.randint(0, max(case["far"] - run_of, 1), (-(-n // run_of),), generator=g, device=DEV)
        state["positions"] = (first.repeat_interleave(run_of)[:n] + torch.arange(n, device=DEV) % run_of).to(torch.int32)
        state["weights"] = [1.0 + 0.2 * randn(dim) if case["norm"] else None for _ in range(2)]
        return state
    if case["op"] == "cache":
        n, heads, dim, size = case["tokens"], case["kv_heads"], case["dim"], case["page"]
        pages = -(-n // size) + 3
        # heads and channels of unlike sizes, as keys have them
        spread = torch.exp(randn(1, heads, dim) * 0.7)
        k, v = ((randn(n, heads, dim) * s).to(DTYPES[case["src"]]) for s in (spread, 1.0))
        state["k"], state["v"] = _packed([k, v], case["strided"])
        # whole pages in any order
        order = torch.randperm(pages, generator=g, device=DEV)
        at = torch.arange(n, device=DEV)
        slots = order[at // size] * size + at % size
        if case["skipped"]:
            slots[n - min(n, case["skipped"]):] = -1   # padding
        (kc, ks), (vc, vs) = (_empty_cache(case, pages) for _ in range(2))
        state.update(slots=slots, kc=kc, vc=vc, ks=ks, vs=vs)
        return state
    new, before = _lengths(case)
    length = [a + n for a, n in zip(new, before)]
    heads, kv_heads, dim, size = case["heads"], case["kv_heads"], case["dim"], case["page"]
    counts = [-(-n // size) for n in length]
    pages, wide = sum(counts) + 2, max(max(counts), 1)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    rows, page_of, offset, used = [], [], [], 0
    for n, c in zip(length, counts):
        rows.append(torch.nn.functional.pad(order[used:used + c], (0, wide - c)))
        at = torch.arange(n, device=DEV)
        page_of.append(order[used + at // size].long())
        offset.append(at % size)
        used += c
    page_of, offset = torch.cat(page_of), torch.cat(offset)
    for c, s in (("kc", "ks"), ("vc", "vs")):
        state[c], state[s] = _empty_cache(case, pages)
        state[c][page_of, :, offset], state[s][page_of, :, offset] = _quantized(randn(sum(length), kv_heads, dim))
    single = all(n == 1 for n in new)
    ends = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
    state.update(q=randn(sum(new), heads, dim).to(DTYPES[case["q"]]), table=torch.stack(rows),
                 length=torch.tensor(length, dtype=torch.int32, device=DEV), starts=None if single else ends,
                 most=max(new))
    return state


# ------------------------------------------------------------------ plain forms


def _plain_pages(s):
    """What extending and taking the new tokens back again leaves, in whole numbers."""
    size, table, before, new = s["page"], s["table"], s["length"].long(), s["grown"].long()
    seqs, cols = table.shape
    starts = torch.nn.functional.pad(new.cumsum(0), (1, 0))
    held, need = (before + size - 1) // size, (before + new + size - 1) // size
    taken = (need - held).cumsum(0)
    first = taken - (need - held)
    # the pages that columns held .. need - 1 get, from the end of the free ones on
    col = torch.arange(cols, device=DEV)
    fresh = (col >= held.unsqueeze(1)) & (col < need.unsqueeze(1))
    left = s["count"].long()
    source = left - 1 - (first - held).unsqueeze(1) - col
    table.copy_(torch.where(fresh, s["free"][torch.where(fresh, source, 0)], table))
    # the rows
    row = torch.arange(s["rows"], device=DEV)
    seq = torch.searchsorted(starts[1:], row, right=True)
    real = seq < seqs
    seq = torch.where(real, seq, 0)
    position = before[seq] + row - starts[seq]
    page = table[seq, torch.where(real, position // size, 0)].long()
    slots = torch.where(real, page * size + position % size, -1)
    position = torch.where(real, position, -1).to(torch.int32)
    # and back: pages past the ones kept return to where they came from
    keep = s["before"].long()
    back = (col >= ((keep + size - 1) // size).unsqueeze(1)) & (col < need.unsqueeze(1))
    to = torch.where(back, source, s["free"].shape[0])
    free = torch.nn.functional.pad(s["free"], (0, 1))
    free[to] = table
    s["free"].copy_(free[:-1])
    s["length"].copy_(torch.minimum(before + new, keep))
    s["count"].copy_(left - taken[-1] + back.sum())
    return _pages_out(s, starts.to(torch.int32), slots, position)


def _pages_out(s, starts, slots, position):
    return {"starts": starts, "slots": slots, "positions": position, "table": s["table"], "lengths": s["length"],
            "free": s["free"], "count": s["count"]}


def _plain_rotary(s):
    f, amplitude = _frequencies(s)
    angle = s["positions"].double().unsqueeze(1) * f
    cos, sin = ((t * amplitude).float().unsqueeze(1) for t in (torch.cos(angle), torch.sin(angle)))
    out = []
    for x, w in ((s["queries"], s["weights"][0]), (s["keys"], s["weights"][1])):
        dtype, x = x.dtype, x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(2, keepdim=True) + 1e-6) * w
        part, rest = x[..., :s["rotary"]], x[..., s["rotary"]:]
        a, b = part.chunk(2, 2) if s["layout"] == "half" else (part[..., 0::2], part[..., 1::2])
        turned = (a * cos - b * sin, a * sin + b * cos)
        turned = torch.cat(turned, 2) if s["layout"] == "half" else torch.stack(turned, 3).flatten(2)
        out.append(torch.cat([turned, rest], 2).to(dtype))
    return out


def _quantized(x):
    """Codes (two a byte, the even channel low) and the scale of each 32 channels of rows [..., dim]: the least power of
    two 2^e with max|x| < 7 2^e, held as e + 127; 0, 0.5, 1, 1.5, 2, 3, 4, 6 to nearest, ties to even."""
    x = x.float().unflatten(-1, (-1, BLOCK))
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))   # m in [0.5, 1)
    e = torch.where(m > 0, e - 3 + (m >= 0.875), LOWEST).clamp(min=LOWEST)
    y = torch.ldexp(x.abs(), -e)
    code = torch.where(y < 2, torch.round(y * 2), torch.where(y < 4, torch.round(y) + 2, torch.round(y / 2) + 4))
    code = (code.clamp(max=7).to(torch.uint8) + 8 * torch.signbit(x).to(torch.uint8)).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, (e + 127).to(torch.uint8).squeeze(-1)


def _values(codes, scale):
    """The numbers that codes [..., dim / 2] stand for, FP32."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()
    size = torch.where(code % 8 < 4, (code % 8) * 0.5, (2 + code % 2) * torch.exp2((code % 8 // 2 - 2).float()))
    size = torch.where(code >= 8, -size, size).unflatten(-1, (-1, BLOCK))
    return torch.ldexp(size, scale.unsqueeze(-1).int() - 127).flatten(-2)


def _plain_cache(s):
    size = s["page"]
    kept = s["slots"] >= 0
    page_of, offset = s["slots"][kept] // size, s["slots"][kept] % size
    got = {}
    for x, c, sc in (("k", "kc", "ks"), ("v", "vc", "vs")):
        s[c][page_of, :, offset], s[sc][page_of, :, offset] = _quantized(s[x][kept])
        got[x] = torch.zeros(s[x].shape, dtype=DTYPES[s["out"]], device=DEV)
        got[x][kept] = _values(s[c][page_of, :, offset], s[sc][page_of, :, offset]).to(got[x].dtype)
    return got


def _plain_attend(s):
    size, kv_heads, group, dim = s["page"], s["kv_heads"], s["heads"] // s["kv_heads"], s["dim"]
    seqs, most = s["seqs"], s["most"]
    starts = s["starts"] if s["starts"] is not None else torch.arange(seqs + 1, device=DEV)
    new = starts[1:] - starts[:-1]
    at = torch.arange(s["table"].shape[1] * size, device=DEV)
    there = at < s["length"].unsqueeze(1)
    page_of, offset = s["table"].long()[:, at // size], (at % size).expand(seqs, -1)
    k, v = (torch.where(there[..., None, None], _values(s[c][page_of, :, offset], s[sc][page_of, :, offset]), 0.0)
            .transpose(1, 2) for c, sc in (("kc", "ks"), ("vc", "vs")))
    i = torch.arange(most, device=DEV)
    mine = i < new.unsqueeze(1)
    row = torch.where(mine, starts[:-1].unsqueeze(1) + i, 0).long()
    q = s["q"][row].float().unflatten(2, (kv_heads, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * dim ** -0.5
    last = (s["length"] - new).unsqueeze(1) + i
    seen = (at <= last.unsqueeze(2)).view(seqs, 1, 1, most, -1)
    scores = scores.unflatten(2, (group, most)).masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), v).unflatten(2, (group, most)) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)[mine]
    return out.to(s["q"].dtype)


# ------------------------------------------------------------------ one pass


def _own(state):
    """The program's handle on its tables, frequencies or cache, made once."""
    if "handle" not in state:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                          "intel-optimized-moe-streaming_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        if state["op"] == "pages":
            from flash_moe_hip.page_table import PageTable

            state["handle"] = PageTable(state["table"], state["length"], state["free"], state["count"], state["page"])
        elif state["op"] == "rotary":
            from flash_moe_hip.rotary import Rotary

            state["handle"] = Rotary(state["dim"], state["rotary"], base=BASE, layout=state["layout"],
                                     scaling=_scaling(state), device=DEV)
        else:
            from flash_moe_hip.kv_cache import PagedCache

            codes, scales = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
            state["handle"] = PagedCache(state["kc"].view(codes), state["vc"].view(codes), state["ks"].view(scales),
                                         state["vs"].view(scales))
    return state["handle"]


def run(state):
    s, op = state, state["op"]
    if not own:
        return {"pages": _plain_pages, "rotary": _plain_rotary, "cache": _plain_cache, "attend": _plain_attend}[op](s)
    handle = _own(s)
    if op == "pages":
        # new tokens are given places, and taken back as a program takes back drafts
        starts, slots, positions = handle.extend(s["grown"], s["rows"])
        handle.trim(s["before"])
        return _pages_out(s, starts, slots, positions)
    if op == "rotary":
        return list(handle.apply(s["queries"], s["keys"], s["positions"], q_weight=s["weights"][0],
                                 k_weight=s["weights"][1], eps=1e-6))
    if op == "cache":
        handle.write(s["k"], s["v"], s["slots"])
        k, v = handle.read(s["slots"], dtype=DTYPES[s["out"]])
        return {"k": k, "v": v}
    return handle.attend(s["q"], s["table"], s["length"], starts=s["starts"])


# ------------------------------------------------------------------ work


def work(case):
    if case["op"] == "pages":
        new, before = _lengths(case)
        size, rows = case["page"], sum(new) + case["padded"]
        fresh = sum(-(-(n + a) // size) - -(-n // size) for n, a in zip(before, new))
        # lengths and counts in twice, starts and lengths out, slots and positions out, pages moved there and back
        return {"bytes": 28 * case["seqs"] + 12 * rows + 16 * fresh, "flops": 4 * rows}
    if case["op"] == "rotary":
        rows = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * rows * case["dim"] * SIZE[case["dtype"]] + 4 * case["tokens"],
                "flops": rows * (3 * case["rotary"] + (4 * case["dim"] if case["norm"] else 0))}
    if case["op"] == "cache":
        rows, held = 2 * case["tokens"] * case["kv_heads"], case["dim"] // 2 + case["dim"] // BLOCK
        # the source in, the cache's rows out and in again, the values out
        return {"bytes": rows * (case["dim"] * (SIZE[case["src"]] + SIZE[case["out"]]) + 2 * held) + 8 * case["tokens"],
                "flops": 3 * rows * case["dim"]}
    new, before = _lengths(case)
    held = case["dim"] // 2 + case["dim"] // BLOCK
    pairs = sum(a * n + a * (a + 1) // 2 for a, n in zip(new, before))
    used = sum(a + n for a, n in zip(new, before) if a)
    return {"bytes": 2 * used * case["kv_heads"] * held + 4 * sum(new) * case["heads"] * case["dim"],
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ------------------------------------------------------------------ the same in 64 bits


def _exact_pages(s):
    """Sequence by sequence on the host."""
    size, rows = s["page"], s["rows"]
    table, free = s["table"].tolist(), s["free"].tolist()
    top = at = s["count"].item()
    starts, slots, positions = [0], [], []
    for b, (n, a) in enumerate(zip(s["before"].tolist(), s["grown"].tolist())):
        for p in range(n, n + a):
            if p % size == 0:
                at -= 1
                table[b][p // size] = free[at]
            slots.append(table[b][p // size] * size + p % size)
            positions.append(p)
        starts.append(starts[-1] + a)
    fill = [-1] * (rows - len(slots))

    def ints(x):
        return torch.tensor(x, dtype=torch.int64, device=DEV)

    return {"starts": ints(starts), "slots": ints(slots + fill), "positions": ints(positions + fill),
            "table": ints(table), "lengths": s["before"].long(), "free": ints(free), "count": ints([top])}


def _exact_rotary(s):
    f, amplitude = _frequencies(s)
    turn = amplitude * torch.exp(1j * s["positions"].double().unsqueeze(1) * f)   # [tokens, pairs]
    half, n = s["rotary"] // 2, s["rotary"]
    i = torch.arange(half, device=DEV)
    re, im = (i, i + half) if s["layout"] == "half" else (2 * i, 2 * i + 1)
    out = []
    for x, w in zip((s["queries"], s["keys"]), s["weights"]):
        y = x.double().clone()
        if w is not None:
            y = y / torch.sqrt(torch.linalg.vector_norm(y, dim=2, keepdim=True) ** 2 / y.shape[2] + 1e-6) * w.double()
        z = torch.complex(y[..., re], y[..., im]) * turn.unsqueeze(1)
        y[..., re], y[..., im] = z.real, z.imag
        out.append(y)
    return out


GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_cache(s):
    grid = torch.tensor(GRID, dtype=torch.float64, device=DEV)
    got = {}
    for name in ("k", "v"):
        x = s[name].double().unflatten(2, (-1, BLOCK))
        top = x.abs().amax(3, keepdim=True)
        step = torch.exp2(torch.arange(LOWEST, 120, dtype=torch.float64, device=DEV))
        step = step[(top >= 7 * step).sum(3, keepdim=True)]
        y, near = x.abs() / step, torch.zeros_like(x)
        for i, (a, b) in enumerate(zip(GRID, GRID[1:])):   # past the middle, or on it from an odd place
            near = torch.where((y >= (a + b) / 2) if i % 2 else (y > (a + b) / 2), grid[i + 1], near)
        got[name] = (near * step * torch.sign(x)).flatten(2) * (s["slots"] >= 0).view(-1, 1, 1)
    return got


def _numbers(codes, scale):
    grid = torch.tensor(GRID + tuple(-x for x in GRID), dtype=torch.float64, device=DEV)
    x = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=DEV)
    x[..., 0::2], x[..., 1::2] = grid[(codes % 16).long()], grid[(codes // 16).long()]
    return x * torch.exp2(scale.double() - 127).repeat_interleave(BLOCK, -1)


def _exact_attend(s):
    group, rows = s["heads"] // s["kv_heads"], []
    new, before = _lengths(s)
    q = s["q"].double().split(new)
    for b, (a, n) in enumerate(zip(new, before)):
        at = torch.arange(n + a, device=DEV)
        page, off = s["table"][b][at // s["page"]].long(), at % s["page"]
        out = torch.zeros(q[b].shape, dtype=torch.float64, device=DEV)
        hidden = at.view(1, -1) > torch.arange(n, n + a, device=DEV).view(-1, 1)
        for h in range(s["heads"]):
            if h % group == 0:
                k, v = (_numbers(s[c][page, h // group, off], s[sc][page, h // group, off])
                        for c, sc in (("kc", "ks"), ("vc", "vs")))
            z = (q[b][:, h] @ k.T.contiguous()) / math.sqrt(s["dim"])
            out[:, h] = torch.softmax(z.masked_fill_(hidden, -math.inf), 1) @ v
        rows.append(out)
    return torch.cat(rows)


def exact(case, seed):
    s = prepare(case, seed)
    return {"pages": _exact_pages, "rotary": _exact_rotary, "cache": _exact_cache, "attend": _exact_attend}[s["op"]](s)
