"""Attention of new tokens, its accumulated weights and eviction as a serving loop
runs them: a prompt in two chunks, the cache cut by its last queries' weights,
decode steps over it, eager and as one graph."""
import numpy as np
import pytest
import torch

import _sparse_refs as R
import _varlen_refs as V

pytestmark = pytest.mark.gpu

HQ, HKV, DIM, SECTIONS = 8, 2, 64, (8, 12, 12)
I32 = torch.int32


def _ints(x):
    return torch.tensor(np.asarray(x), dtype=I32, device="cuda")


class Loop:
    """Three sequences with room for 600 tokens each, one of them idle."""

    def __init__(self, seed=0):
        rng = self.rng = np.random.default_rng(seed)
        ids = rng.permutation(3 * 38 + 2).astype(np.int32)
        self.table = ids[:3 * 38].reshape(3, 38)
        self.want = list(R.random_cache(rng, 3 * 38 + 2, HKV, DIM))
        self.cache = [torch.from_numpy(x.copy()).cuda() for x in self.want]
        self.mass = torch.from_numpy(rng.random((3 * 38 + 2, HKV, 16)).astype(np.float32)).cuda()  # of earlier owners
        ang = np.arange(2000)[:, None] * 10000.0 ** (-np.arange(DIM // 2) / (DIM // 2))
        self.cos, self.sin = (R.to_type(f(ang), torch.bfloat16).cuda() for f in (np.cos, np.sin))

    def tokens(self, n):
        return [R.to_type(self.rng.standard_normal((n, h, DIM)), torch.bfloat16).cuda() for h in (HQ, HKV, HKV)]

    def slots(self, b, places):
        return self.table[b][places // 16] * 16 + places % 16

    def append(self, query, key, value, pos, slots):
        from iris_kernel.fused_kv import fused_mrope_int4_paged_append

        pos = np.stack([pos, pos // 2, pos // 3]).astype(np.int32)
        return fused_mrope_int4_paged_append(key, value, _ints(pos), _ints(slots), self.cos, self.sin, *self.cache, query,
                                             sections=SECTIONS, rotary_dim=DIM, page_size=16)

    def host(self):
        return [x.cpu().numpy() for x in self.cache]


def _close(got, want, far):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all() and (np.abs(got - want) <= far).all()


def _prompt(loop, how):
    """Two chunks of prompts of 500 and 333 tokens, then the cache cut to 100 by the last 32 queries."""
    from iris_kernel.fused_kv import fused_int4_paged_evict
    from iris_kernel.varlen_attention import fused_int4_paged_attention_mass, fused_int4_paged_varlen_attention

    lens, total = np.zeros(3, np.int32), (500, 0, 333)
    table = torch.from_numpy(loop.table).cuda()
    for chunk in ((300, 0, 333), (200, 0, 0)):
        pos = np.concatenate([np.arange(n, n + m) for n, m in zip(lens, chunk)])
        slots = np.concatenate([loop.slots(b, np.arange(n, n + m)) for b, (n, m) in enumerate(zip(lens, chunk))])
        query, key, value = loop.tokens(sum(chunk))
        rotated = loop.append(query, key, value, pos, slots)
        lens = lens + np.array(chunk, np.int32)
        cu = np.concatenate([[0], np.cumsum(chunk)]).astype(np.int32)
        out, lse = fused_int4_paged_varlen_attention(rotated, *loop.cache, table, _ints(lens), _ints(cu), return_lse=True,
                                                     **how)
        o, s, fo, fs = V.attend_ref(R.f32(rotated), loop.host(), loop.table, lens, cu, torch.bfloat16, **how)
        _close(out, o, fo)
        _close(lse, s, fs)
    assert tuple(lens) == total
    # the last 32 rows of the last call belong to sequence 0; sequence 2's weights come from its own chunk's
    last = _ints([0, 32, 32, 32])
    mass = loop.mass.cpu().numpy()
    fused_int4_paged_attention_mass(rotated[-32:], lse[-32:], loop.cache[0], loop.cache[2], table, _ints(lens), loop.mass,
                                    last, **how)
    want, far = V.mass_ref(R.f32(rotated[-32:]), lse[-32:].cpu().numpy(), loop.host(), loop.table, lens,
                           last.cpu().numpy(), mass, None, 1.0, **how)
    _close(loop.mass, want, far)
    want, weights = loop.host(), loop.mass.cpu().numpy()
    new = fused_int4_paged_evict(*loop.cache, loop.mass, table, _ints(lens), budget=100, sink_tokens=4, recent_tokens=20)
    V.evict_ref(want, weights, loop.table, lens, 100, 4, 20)
    for x, w in zip((*loop.cache, loop.mass), (*want, weights)):
        assert x.cpu().numpy().tobytes() == w.tobytes()
    assert new.tolist() == [100, 0, 100]
    return new


@pytest.mark.parametrize("how", [{}, dict(logit_cap=8.0), dict(window=60)])
def test_a_prompt_and_decode_steps_within_a_budget(how):
    from iris_kernel.fused_kv import fused_int4_paged_evict
    from iris_kernel.step import BudgetDecodeStep
    from iris_kernel.varlen_attention import fused_int4_paged_attention_mass, fused_int4_paged_varlen_attention

    eager, graph = Loop(), Loop()
    lens = _prompt(eager, how)
    glens = _prompt(graph, how)
    table = torch.from_numpy(eager.table).cuda()
    kw = dict(budget=100, sink_tokens=4, recent_tokens=20)
    before = [x.clone() for x in (*graph.cache, graph.mass)]
    step = BudgetDecodeStep(*graph.cache, graph.mass, table, glens, graph.cos, graph.sin, num_q_heads=HQ,
                            sections=SECTIONS, rotary_dim=DIM, decay=0.9, **kw, **how)
    assert glens.tolist() == [100, 0, 100] and all(torch.equal(x, y) for x, y in zip(before, (*graph.cache, graph.mass)))
    for i in range(4):
        query, key, value = eager.tokens(3)
        pos = np.array([500 + i, 0, 333 + i])
        slots = np.array([eager.slots(0, np.array([100]))[0], -1, eager.slots(2, np.array([100]))[0]])
        rotated = eager.append(query, key, value, pos, slots)
        lens = _ints([101, 0, 101])
        out, lse = fused_int4_paged_varlen_attention(rotated, *eager.cache, table, lens, return_lse=True, **how)
        host, at = eager.host(), np.array([101, 0, 101], np.int32)
        cu = np.arange(4)
        o, s, fo, fs = V.attend_ref(R.f32(rotated), host, eager.table, at, cu, torch.bfloat16, **how)
        _close(out, o, fo)
        weights = eager.mass.cpu().numpy()
        fused_int4_paged_attention_mass(rotated, lse, eager.cache[0], eager.cache[2], table, lens, eager.mass,
                                        first_token=lens - 1, decay=0.9, **how)
        w, far = V.mass_ref(R.f32(rotated), lse.cpu().numpy(), host, eager.table, at, cu, weights, at - 1, 0.9, **how)
        _close(eager.mass, w, far)
        weights = eager.mass.cpu().numpy()
        new = fused_int4_paged_evict(*eager.cache, eager.mass, table, lens, **kw)
        V.evict_ref(host, weights, eager.table, at, 100, 4, 20)
        for x, y in zip((*eager.cache, eager.mass), (*host, weights)):
            assert x.cpu().numpy().tobytes() == y.tobytes()
        # the same step as one replay
        glens.copy_(lens)
        p3 = np.stack([pos, pos // 2, pos // 3]).astype(np.int32)
        got = step(query, key, value, _ints(p3), _ints(slots), check=True)
        torch.cuda.synchronize()
        assert torch.equal(got, out) and torch.equal(glens, new)
        assert all(torch.equal(x, y) for x, y in zip((*eager.cache, eager.mass), (*graph.cache, graph.mass)))


def test_two_streams_at_once():
    """Calls in flight on two streams, with workspaces of their own."""
    from iris_kernel.varlen_attention import fused_int4_paged_varlen_attention
    from test_gpu_varlen_attention import Case

    cases = [Case([3], [30000], 8, 1, 64, seed=1), Case([1] * 4, [7000, 3, 900, 50], 8, 2, 128, seed=2, offsets=False)]
    want = [c.check()[0] for c in cases]
    args = [c.args() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(fused_int4_paged_varlen_attention(*args[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
