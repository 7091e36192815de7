"""A small hybrid stack as a serving program runs it: a recurrent layer, an attention layer over a paged cache and a
mixture-of-experts layer, for two sequences: prompts in chunks of different lengths, then token by token.

The outputs at every position have to be those of the whole sequences run through the prompt kernels at once.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KEY_HEADS, DK, DV = 512, 4, 2, 64, 128
Q_HEADS, KV_HEADS, DIM, PAGE = 8, 2, 64, 16


def make_layer():
    from flash_moe_hip.layer_store import ExpertLayer

    return ExpertLayer.synthetic({"gate": 12, "up": 12, "down": 14}, 16, HIDDEN, 256, seed=3, shared_types=None,
                                 scale=0.001, device="cuda")


class Stack:
    def __init__(self, layer, cache_type, sequences, pages):
        from flash_moe_hip.kv_cache import PagedCache
        from flash_moe_hip.linear_attention import LinearState
        from flash_moe_hip.moe_gpu import MoeRunner

        g = torch.Generator(device="cuda").manual_seed(1)

        def w(*shape):
            return torch.randn(*shape, generator=g, device="cuda") * shape[0] ** -0.5

        self.w_in = w(HIDDEN, 2 * KEY_HEADS * DK + HEADS * DV + 2 * HEADS)
        self.w_mix = w(HEADS * DV, HIDDEN)
        self.w_qkv = w(HIDDEN, (Q_HEADS + 2 * KV_HEADS) * DIM)
        self.w_out = w(Q_HEADS * DIM, HIDDEN)
        self.w_route = w(HIDDEN, 16).T.contiguous()
        self.layer, self.runner = layer, MoeRunner()
        self.states = LinearState(sequences, HEADS, DV, DK)
        self.cache = PagedCache.empty(pages, KV_HEADS, DIM, PAGE, cache_type)
        self.table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).view(sequences, -1).contiguous()
        self.held = [0] * sequences

    def run(self, x, parts):
        """x [tokens, HIDDEN]: parts[b] new tokens of sequence b, packed."""
        single = all(n == 1 for n in parts)
        starts = None if single else torch.tensor([0] + parts).cumsum(0).to(torch.int32).cuda()
        y = torch.nn.functional.rms_norm(x, (HIDDEN,)) @ self.w_in
        q, k, v, beta, gate = y.split([KEY_HEADS * DK, KEY_HEADS * DK, HEADS * DV, HEADS, HEADS], 1)
        unit = torch.nn.functional.normalize
        q, k = (unit(t.unflatten(1, (KEY_HEADS, DK)), dim=2) for t in (q, k))
        args = q, k, v.unflatten(1, (HEADS, DV)), torch.sigmoid(beta), -torch.nn.functional.softplus(gate) * 0.1
        mixed = self.states.step(*args) if single else self.states.prefill(*args, starts=starts)
        x = x + mixed.flatten(1) @ self.w_mix

        # (one projection's rows: the calls take its parts as they lie)
        y = (torch.nn.functional.rms_norm(x, (HIDDEN,)) @ self.w_qkv).half().unflatten(1, (Q_HEADS + 2 * KV_HEADS, DIM))
        q, k, v = y.split([Q_HEADS, KV_HEADS, KV_HEADS], 1)
        seq = torch.cat([torch.full((n,), b) for b, n in enumerate(parts)]).cuda()
        pos = torch.cat([torch.arange(self.held[b], self.held[b] + n) for b, n in enumerate(parts)]).cuda()
        self.cache.write(k, v, self.cache.slots(self.table, seq, pos))
        self.held = [h + n for h, n in zip(self.held, parts)]
        lengths = torch.tensor(self.held, dtype=torch.int32).cuda()
        x = x + self.cache.attend(q, self.table, lengths, starts).float().flatten(1) @ self.w_out

        h = torch.nn.functional.rms_norm(x, (HIDDEN,)).contiguous()
        if x.shape[0] <= 4:
            out, _, _ = self.runner.decode_routed(self.layer, h, 4, router_w=self.w_route)
        else:
            ids, weights = self.runner.route(self.layer, h, 4, router_w=self.w_route)
            out = self.runner.prefill(self.layer, h, ids, weights)
        return x + out

    def check(self):
        assert self.states.status() == 0 and self.cache.status() == 0 and self.runner.status() == 0


@pytest.mark.parametrize("cache_type", [torch.float16, torch.int8], ids=str)
def test_chunks_and_steps_are_the_whole_sequence(cache_type):
    layer = make_layer()
    lengths = [93, 150]
    g = torch.Generator(device="cuda").manual_seed(2)
    x = [torch.randn(n, HIDDEN, generator=g, device="cuda") for n in lengths]
    whole = Stack(layer, cache_type, 2, 32)
    want = whole.run(torch.cat(x), lengths).split(lengths)
    whole.check()

    stack = Stack(layer, cache_type, 2, 32)
    got = [[], []]
    at = [0, 0]
    for parts in ([64, 30], [5, 0], [20, 116], [1, 1], [1, 1], [1, 1], [1, 1]):
        rows = torch.cat([t[a:a + n] for t, a, n in zip(x, at, parts)])
        out = stack.run(rows, parts).split(parts)
        for b in range(2):
            got[b].append(out[b])
            at[b] += parts[b]
    stack.check()
    for b in range(2):
        rows = torch.cat(got[b])
        assert rows.shape[0] == at[b]
        # the decode kernels' 16-bit activations and, in an int8 cache, codes that round the
        # other way after them (a step of 1 / 127) are the only differences but for FP32 sums
        err = (rows - want[b][:at[b]]).norm() / want[b][:at[b]].norm()
        assert err < (2e-3 if cache_type == torch.float16 else 1e-2), float(err)
    # the cache holds what was written, read back by position
    pos = torch.arange(at[0], device="cuda")
    slots = stack.cache.slots(stack.table, torch.zeros_like(pos), pos)
    k, v = stack.cache.read(slots)
    k2, v2 = whole.cache.read(whole.cache.slots(whole.table, torch.zeros_like(pos), pos))
    for a, b in ((k, k2), (v, v2)):
        assert np.isfinite(a.float().cpu().numpy()).all()
        assert ((a.float() - b.float()).norm() / b.float().norm()) < 1e-2


def test_a_captured_decode_step_replays():
    """One captured step (recurrent layer, cache write, attention) replayed over new inputs in place, against eager ones."""
    stacks = [Stack(make_layer(), torch.int8, 2, 32) for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(5)
    prompt = torch.randn(40, HIDDEN, generator=g, device="cuda")
    for s in stacks:
        s.run(prompt, [25, 15])
    eager, other = stacks

    def mix(s, q, k, v, beta, gate, qkv, slots, lengths):
        a = s.states.step(q, k, v, beta, gate)
        s.cache.write(qkv[:, Q_HEADS:Q_HEADS + KV_HEADS], qkv[:, Q_HEADS + KV_HEADS:], slots)
        return a, s.cache.attend(qkv[:, :Q_HEADS], s.table, lengths)

    def inputs():
        def randn(*shape):
            return torch.randn(*shape, generator=g, device="cuda")

        return [torch.nn.functional.normalize(randn(2, KEY_HEADS, DK), dim=2),
                torch.nn.functional.normalize(randn(2, KEY_HEADS, DK), dim=2), randn(2, HEADS, DV),
                torch.rand(2, HEADS, generator=g, device="cuda"), -torch.rand(2, HEADS, generator=g, device="cuda"),
                randn(2, Q_HEADS + 2 * KV_HEADS, DIM).half()]

    held = torch.tensor([25, 15], dtype=torch.int32, device="cuda")
    seq = torch.arange(2, device="cuda")
    static = inputs() + [other.cache.slots(other.table, seq, held.long()), held + 1]
    state0 = other.states.state.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = mix(other, *static)
    assert torch.equal(other.states.state, state0)   # (captured, not run)
    for step in range(4):
        new = inputs()
        length = held + step + 1
        slots = eager.cache.slots(eager.table, seq, (length - 1).long())
        for t, n in zip(static, new + [slots, length]):
            t.copy_(n)
        graph.replay()
        want = mix(eager, *new, slots, length)
        assert all(torch.equal(a, b) for a, b in zip(y, want)), step
        assert torch.equal(other.states.state, eager.states.state)
    eager.check()
    other.check()
