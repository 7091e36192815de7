"""The token mixers' operators: what is timed of them, their plain forms and their 64-bit results.

A paged key/value cache (16-bit, or 8-bit codes with one FP32 scale per token and head) that is written and read back,
attention of new tokens over it (chunks of prompts, drafts, single tokens), and linear attention with a decay per head
(with the delta rule or without) over prompts and single tokens.  32 heads of 128 x 128 state are the benchmark's
recurrent layers, 64 sequences and 64-token pages generic serving sizes; lengths, head counts and types vary over what a
serving program meets.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CHUNK = 64


def listed():
    return [
        # one new token of each of 64 sequences, quantized into the cache and read back
        dict(name="cache q8 64 tokens", op="cache", tokens=64, kv_heads=8, dim=128, page=64, cache="q8", src="bf16",
             out="bf16", skipped=0, strided=True),
        # a long prompt quantized into the cache, read back for a program's own use
        dict(name="cache q8 16384 tokens", op="cache", tokens=16384, kv_heads=8, dim=128, page=64, cache="q8",
             src="bf16", out="bf16", skipped=0, strided=True),
        # FP32 activations into a 16-bit cache, an odd number of them, some padding
        dict(name="cache f16 4099 tokens", op="cache", tokens=4099, kv_heads=2, dim=256, page=16, cache="f16",
             src="f32", out="f16", skipped=37, strided=False),
        # a whole prompt at once
        dict(name="attend prompt 8192", op="attend", seqs=1, new=8192, prior=0, heads=32, kv_heads=8, dim=128, page=64,
             cache="bf16", q="bf16", ragged=False),
        # chunks of four long prompts over an 8-bit cache
        dict(name="attend chunks q8", op="attend", seqs=4, new=2048, prior=16384, heads=16, kv_heads=2, dim=256,
             page=64, cache="q8", q="bf16", ragged=True),
        # five drafted tokens of each of eight sequences
        dict(name="attend drafts f16", op="attend", seqs=8, new=40, prior=2051, heads=16, kv_heads=16, dim=64, page=32,
             cache="f16", q="f16", ragged=False),
        # the next token of one sequence
        dict(name="attend token 1 q8", op="attend", seqs=1, new=1, prior=4098, heads=16, kv_heads=2, dim=256, page=64,
             cache="q8", q="bf16", ragged=False),
        # the next token of each of 64 sequences
        dict(name="attend token 64 bf16", op="attend", seqs=64, new=64, prior=8191, heads=32, kv_heads=8, dim=128,
             page=64, cache="bf16", q="bf16", ragged=True),
        # a recurrent layer's prompt
        dict(name="delta prompt 4096", op="prompt", rule="delta", seqs=1, tokens=4096, heads=32, key_heads=16,
             key_dim=128, value_dim=128, dtype="f32", ragged=False, strided=True),
        # ragged prompts of several sequences, without the delta rule
        dict(name="decay prompts 2501", op="prompt", rule="decay", seqs=5, tokens=2501, heads=16, key_heads=16,
             key_dim=64, value_dim=128, dtype="bf16", ragged=True, strided=False),
        # the next token of each of 64 sequences through a recurrent layer
        dict(name="delta step 64", op="step", rule="delta", seqs=64, heads=32, key_heads=16, key_dim=128,
             value_dim=128, dtype="f32", strided=False),
        # the next token of one sequence
        dict(name="decay step 1", op="step", rule="decay", seqs=1, heads=16, key_heads=16, key_dim=64, value_dim=128,
             dtype="bf16", strided=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["cache", "attend", "attend", "token", "token", "prompt", "prompt", "step"])
    if op == "cache":
        cache = rng.choice(["q8", "q8", "f16", "bf16"])
        out = rng.choice(["f16", "bf16", "f32"]) if cache == "q8" else cache
        kv_heads, dim = rng.choice([1, 2, 5, 8]), rng.choice([64, 128, 256])
        return dict(op=op, tokens=_log(rng, 1, 2 ** 23 // (kv_heads * dim)), kv_heads=kv_heads, dim=dim,
                    page=rng.choice([16, 32, 64, 128]), cache=cache, src=rng.choice(["f32", "bf16", "f16"]), out=out,
                    skipped=rng.choice([0, 0, 1]), strided=rng.random() < 0.5)
    if op in ("attend", "token"):
        kv_heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
        group = rng.choice([1, 2, 4, 5, 8, 16])
        cache = rng.choice(["q8", "bf16", "f16"])
        q = cache if cache != "q8" else rng.choice(["bf16", "f16"])
        case = dict(op="attend", seqs=_log(rng, 1, 8 if op == "attend" else 96), heads=kv_heads * group,
                    kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64, 128]), cache=cache, q=q,
                    ragged=rng.random() < 0.6)
        if op == "token":
            room = 2 ** 29 // (case["seqs"] * kv_heads * dim)
            case.update(new=case["seqs"], prior=_log(rng, 1, min(65536, room)))
            return case
        room = 2 ** 35 // (case["heads"] * dim)   # products of a query and a key
        case["new"] = _log(rng, 2 * case["seqs"], min(4096, math.isqrt(room)))
        case["prior"] = rng.choice([0, _log(rng, 1, min(32768, room // case["new"]))])
        return case
    rule, dtype = rng.choice(["delta", "delta", "decay"]), rng.choice(["f32", "bf16", "f16"])
    key_heads, group = rng.choice([1, 2, 3, 8, 16]), rng.choice([1, 1, 2, 4])
    case = dict(op=op, rule=rule, heads=key_heads * group, key_heads=key_heads,
                key_dim=rng.choice([16, 64, 80, 128, 128, 256]), value_dim=rng.choice([32, 64, 100, 128, 128, 256]),
                dtype=dtype, strided=rng.random() < 0.5)
    per_token = case["heads"] * max(case["key_dim"], case["value_dim"])
    if op == "step":
        room = 2 ** 25 // (case["heads"] * case["key_dim"] * case["value_dim"])
        case["seqs"] = _log(rng, 1, min(128, room))
        return case
    case.update(seqs=_log(rng, 1, 8), tokens=_log(rng, 2, min(4096, 2 ** 24 // per_token)), ragged=rng.random() < 0.6)
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
    """New tokens and all tokens of each sequence of an attention case (one new token each where there are as many)."""
    n = case["seqs"]
    new = [1] * n if case["new"] == n else _spread(case["new"], n, case["ragged"])
    return new, [a + int(case["prior"] * _share(i, case["ragged"])) for i, a in enumerate(new)]


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


def _paged(x, case, page_of, offset, pages):
    """x [tokens, kv_heads, dim] FP32 as a cache [pages, kv_heads, page, dim] and its scales."""
    heads, size, dim = case["kv_heads"], case["page"], case["dim"]
    if case["cache"] != "q8":
        c = torch.zeros(pages, heads, size, dim, dtype=DTYPES[case["cache"]], device=DEV)
        c[page_of, :, offset] = x.to(c.dtype)
        return c, None
    codes, scale = _quantized(x)
    c = torch.zeros(pages, heads, size, dim, dtype=torch.int8, device=DEV)
    s = torch.zeros(pages, heads, size, dtype=torch.float32, device=DEV)
    c[page_of, :, offset], s[page_of, :, offset] = codes, scale
    return c, s


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    state = dict(case)
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
        empty = torch.zeros(0, heads, dim, device=DEV)
        none = torch.zeros(0, dtype=torch.int64, device=DEV)
        (kc, ks), (vc, vs) = (_paged(empty, case, none, none, pages) for _ in range(2))
        state.update(slots=slots, kc=kc, vc=vc, ks=ks, vs=vs)
        return state
    if case["op"] == "attend":
        new, length = _lengths(case)
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
        kc, ks = _paged(randn(sum(length), kv_heads, dim), case, page_of, offset, pages)
        vc, vs = _paged(randn(sum(length), kv_heads, dim), case, page_of, offset, pages)
        single = all(n == 1 for n in new)
        ends = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
        state.update(q=randn(sum(new), heads, dim).to(DTYPES[case["q"]]), table=torch.stack(rows),
                     length=torch.tensor(length, dtype=torch.int32, device=DEV), starts=None if single else ends,
                     most=max(new), kc=kc, vc=vc, ks=ks, vs=vs)
        return state
    n = case["seqs"] if case["op"] == "step" else case["tokens"]
    heads, key_heads, dk, dv = case["heads"], case["key_heads"], case["key_dim"], case["value_dim"]
    unit = torch.nn.functional.normalize
    q, k = unit(randn(n, key_heads, dk), dim=2), unit(randn(n, key_heads, dk), dim=2)
    v = randn(n, heads, dv)
    q, k, v = _packed([t.to(DTYPES[case["dtype"]]) for t in (q, k, v)], case["strided"])
    # heads that forget at once and heads that remember thousands of tokens
    rate = torch.exp(-torch.arange(heads, device=DEV) * (8.0 / heads))
    gate = -torch.nn.functional.softplus(randn(n, heads) + 1.0) * rate
    beta = torch.sigmoid(randn(n, heads)) if case["rule"] == "delta" else None
    state.update(queries=q, keys=k, values=v, gate=gate, beta=beta, state=randn(case["seqs"], heads, dv, dk) * 0.1)
    if case["op"] == "prompt":
        parts = _spread(n, case["seqs"], case["ragged"])
        state["parts"] = parts
        state["starts"] = torch.tensor([0] + parts, device=DEV).cumsum(0).to(torch.int32)
    return state


# ------------------------------------------------------------------ plain forms


def _quantized(x):
    """8-bit codes and the scale of each token and head: the largest size / 127, the codes rounded to nearest, ties to even."""
    x = x.float()
    scale = x.abs().amax(-1) / 127.0
    codes = torch.where(scale.unsqueeze(-1) > 0, torch.round(x / scale.unsqueeze(-1)), torch.zeros_like(x))
    return codes.clamp(-127, 127).to(torch.int8), scale


def _plain_cache(s):
    size = s["page"]
    kept = s["slots"] >= 0
    page_of, offset = s["slots"][kept] // size, s["slots"][kept] % size
    got = {}
    for x, c, sc in (("k", "kc", "ks"), ("v", "vc", "vs")):
        values = s[x][kept]
        if s["cache"] == "q8":
            s[c][page_of, :, offset], s[sc][page_of, :, offset] = _quantized(values)
            read = s[c][page_of, :, offset].float() * s[sc][page_of, :, offset].unsqueeze(-1)
        else:
            s[c][page_of, :, offset] = values.to(s[c].dtype)
            read = s[c][page_of, :, offset]
        got[x] = torch.zeros(s[x].shape, dtype=DTYPES[s["out"]], device=DEV)
        got[x][kept] = read.to(DTYPES[s["out"]])
    return got


def _gathered(cache, scale, page_of, offset, there):
    """[sequences, kv_heads, positions, dim] FP32, zero where there is no token."""
    x = cache[page_of, :, offset].float()
    if scale is not None:
        x = x * scale[page_of, :, offset].unsqueeze(-1)
    return torch.where(there[..., None, None], x, 0.0).transpose(1, 2)


def _plain_attend(s):
    size, kv_heads, group, dim = s["page"], s["kv_heads"], s["heads"] // s["kv_heads"], s["dim"]
    seqs, most = s["seqs"], s["most"]
    starts = s["starts"] if s["starts"] is not None else torch.arange(seqs + 1, device=DEV)
    new = starts[1:] - starts[:-1]
    at = torch.arange(s["table"].shape[1] * size, device=DEV)
    there = at < s["length"].unsqueeze(1)
    page_of, offset = s["table"].long()[:, at // size], (at % size).expand(seqs, -1)
    k = _gathered(s["kc"], s["ks"], page_of, offset, there)
    v = _gathered(s["vc"], s["vs"], page_of, offset, there)
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


def _expanded(x, heads):
    return x.float().repeat_interleave(heads // x.shape[1], 1)


def _plain_step(s):
    q, k, v = (_expanded(s[n], s["heads"]) for n in ("queries", "keys", "values"))
    state = s["state"]
    state *= torch.exp(s["gate"])[..., None, None]
    if s["beta"] is not None:
        v = s["beta"].unsqueeze(2) * (v - (state * k.unsqueeze(2)).sum(3))
    state += v.unsqueeze(3) * k.unsqueeze(2)
    return {"out": (state * q.unsqueeze(2)).sum(3).to(s["values"].dtype), "state": state}


def _plain_prompt(s):
    """64 tokens at a time: what the tokens of a chunk write is solved within the chunk, and the state goes from one
    chunk to the next."""
    starts, seqs, heads = s["starts"].long(), s["seqs"], s["heads"]
    n = -(-max(s["parts"]) // CHUNK)
    i = torch.arange(n * CHUNK, device=DEV)
    mine = i < (starts[1:] - starts[:-1]).unsqueeze(1)
    row = torch.where(mine, starts[:-1].unsqueeze(1) + i, 0)

    def chunks(x):   # [sequences, heads, chunks, 64, ...], zero past a sequence's end
        x = torch.where(mine.view(seqs, -1, *[1] * (x.dim() - 1)), x[row], 0.0)
        return x.unflatten(1, (n, CHUNK)).movedim(3, 1)

    q, k, v = (chunks(_expanded(s[m], heads)) for m in ("queries", "keys", "values"))
    total = chunks(s["gate"].double()).cumsum(3)
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=DEV).tril()
    between = (total.unsqueeze(4) - total.unsqueeze(3)).masked_fill(~low, -math.inf)
    decay = torch.exp(between).float()
    from_start = torch.exp(total).float().unsqueeze(4)
    to_end = torch.exp(total[..., -1:] - total).float().unsqueeze(4)
    inside = decay * torch.matmul(q, k.transpose(3, 4).contiguous())
    writes, through = v, None
    if s["beta"] is not None:
        beta = chunks(s["beta"]).unsqueeze(4)
        lower = (beta * decay * torch.matmul(k, k.transpose(3, 4).contiguous())).tril(-1)
        solve = torch.eye(CHUNK, device=DEV).expand_as(lower).contiguous()
        for r in range(1, CHUNK):   # rows of (1 + lower)^-1
            solve[..., r, :r] = -torch.matmul(lower[..., r:r + 1, :r], solve[..., :r, :r]).squeeze(3)
        writes, through = torch.matmul(solve, beta * v), torch.matmul(solve, beta * from_start * k)
    state, out = s["state"], torch.empty_like(v)
    for c in range(n):
        across, u = state.transpose(2, 3).contiguous(), writes[:, :, c]
        if through is not None:
            u = u - torch.matmul(through[:, :, c], across)
        out[:, :, c] = from_start[:, :, c] * torch.matmul(q[:, :, c], across) + torch.matmul(inside[:, :, c], u)
        state *= from_start[:, :, c, -1:]
        state += torch.matmul((u * to_end[:, :, c]).transpose(2, 3).contiguous(), k[:, :, c])
    return {"out": out.movedim(1, 3).flatten(1, 2)[mine].to(s["values"].dtype), "state": state}


# ------------------------------------------------------------------ one pass


def _own(state):
    """The program's handle on its cache or states, made once."""
    if "handle" not in state:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                          "intel-optimized-moe-streaming_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        if "kc" in state:
            from flash_moe_hip.kv_cache import PagedCache

            state["handle"] = PagedCache(state["kc"], state["vc"], state["ks"], state["vs"])
        else:
            from flash_moe_hip.linear_attention import LinearState

            state["handle"] = LinearState(*state["state"].shape, state=state["state"])
    return state["handle"]


def run(state):
    s, op = state, state["op"]
    if not own:
        return {"cache": _plain_cache, "attend": _plain_attend, "prompt": _plain_prompt, "step": _plain_step}[op](s)
    handle = _own(s)
    if op == "cache":
        handle.write(s["k"], s["v"], s["slots"])
        k, v = handle.read(s["slots"], dtype=DTYPES[s["out"]])
        return {"k": k, "v": v}
    if op == "attend":
        return handle.attend(s["q"], s["table"], s["length"], starts=s["starts"])
    if op == "step":
        out = handle.step(s["queries"], s["keys"], s["values"], s["beta"], s["gate"])
    else:
        out = handle.prefill(s["queries"], s["keys"], s["values"], s["beta"], s["gate"], starts=s["starts"])
    return {"out": out, "state": handle.state}


# ------------------------------------------------------------------ work


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "cache":
        rows = 2 * case["tokens"] * case["kv_heads"]
        held = case["dim"] + 4 if case["cache"] == "q8" else case["dim"] * size[case["cache"]]
        # the source in, the cache's rows out and in again, the values out
        return {"bytes": rows * (case["dim"] * (size[case["src"]] + size[case["out"]]) + 2 * held) + 8 * case["tokens"],
                "flops": 3 * rows * case["dim"]}
    if case["op"] == "attend":
        new, length = _lengths(case)
        held = case["dim"] + 4 if case["cache"] == "q8" else case["dim"] * size[case["cache"]]
        pairs = sum(a * (n - a) + a * (a + 1) // 2 for a, n in zip(new, length))
        used = sum(n for a, n in zip(new, length) if a)
        return {"bytes": 2 * used * case["kv_heads"] * held + 4 * sum(new) * case["heads"] * case["dim"],
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    n = case["seqs"] if case["op"] == "step" else case["tokens"]
    dk, dv, h = case["key_dim"], case["value_dim"], case["heads"]
    rows = n * (2 * case["key_heads"] * dk + 2 * h * dv) * size[case["dtype"]] + 4 * n * h
    rows += 4 * n * h if case["rule"] == "delta" else 0
    # a token reads the state, writes its row into it and decays it, the delta rule reads it once more
    return {"bytes": rows + 8 * case["seqs"] * h * dk * dv,
            "flops": n * h * dk * dv * (7 if case["rule"] == "delta" else 5)}


# ------------------------------------------------------------------ the same in 64 bits


def _exact_cache(s):
    got = {}
    for name in ("k", "v"):
        x = s[name].double()
        if s["cache"] == "q8":
            step = x.abs().max(2, keepdim=True).values / 127
            x = torch.nan_to_num((x / step).round()) * step
        else:
            x = x.to(DTYPES[s["cache"]]).double()
        got[name] = x * (s["slots"] >= 0).view(-1, 1, 1)
    return got


def _exact_attend(s):
    group, rows = s["heads"] // s["kv_heads"], []
    new, length = _lengths(s)
    q = s["q"].double().split(new)
    for b, n in enumerate(length):
        at = torch.arange(n, device=DEV)
        page, off = s["table"][b][at // s["page"]].long(), at % s["page"]
        out = torch.zeros(q[b].shape, dtype=torch.float64, device=DEV)
        hidden = at.view(1, -1) > torch.arange(n - new[b], n, device=DEV).view(-1, 1)
        for h in range(s["heads"]):
            k, v = s["kc"][page, h // group, off].double(), s["vc"][page, h // group, off].double()
            if s["ks"] is not None:
                k, v = k * s["ks"][page, h // group, off].double()[:, None], v * s["vs"][page, h // group, off].double()[:, None]
            z = (q[b][:, h] @ k.T.contiguous()) / math.sqrt(s["dim"])
            z.masked_fill_(hidden, -math.inf)
            out[:, h] = torch.softmax(z, 1) @ v
        rows.append(out)
    return torch.cat(rows)


def _exact_linear(s):
    """Token by token."""
    heads, state = s["heads"], s["state"].double()
    q, k = (s[n].double().repeat_interleave(heads // s["key_heads"], 1) for n in ("queries", "keys"))
    v, decay = s["values"].double(), torch.exp(s["gate"].double())
    parts = s.get("parts", [1] * s["seqs"])
    first = torch.tensor([0] + parts).cumsum(0)[:-1].to(DEV)
    length = torch.tensor(parts, device=DEV)
    out = torch.zeros(v.shape, dtype=torch.float64, device=DEV)
    for t in range(max(parts)):
        live = (length > t).nonzero().flatten() if min(parts) <= t else slice(None)
        at = first[live] + t
        key = k[at].unsqueeze(2)
        m = state[live] * decay[at].view(-1, heads, 1, 1)
        u = v[at]
        if s["beta"] is not None:
            u = s["beta"][at].double().unsqueeze(2) * (u - (m @ key.transpose(2, 3)).squeeze(3))
        m = torch.addcmul(m, u.unsqueeze(3), key)
        state[live] = m
        out[at] = (m @ q[at].unsqueeze(3)).squeeze(3)
    return {"out": out, "state": state}


def exact(case, seed):
    s = prepare(case, seed)
    return {"cache": _exact_cache, "attend": _exact_attend, "prompt": _exact_linear, "step": _exact_linear}[s["op"]](s)
