"""Prompt and masked attention over the INT4 paged cache, and the cache kept to a budget, as measured cases.

Three operators that a serving loop runs around the dense decode:

* ``attend``: attention of any number of new tokens a sequence (prompts, chunks of prompts, drafts, single tokens) over
  the INT4 cache, causal, with logits capped by a tanh, a bias that falls with distance, a sliding window, a prefix that
  every token sees and documents that do not see one another (`fused_int4_paged_varlen_attention`);
* ``mass``: the attention weight that each cached token received from those queries, summed over a KV head's queries and
  added up in the cache's own layout (`fused_int4_paged_attention_mass`);
* ``evict``: per sequence and KV head, the tokens with the least of it leave the cache, and the others move together
  (`fused_int4_paged_evict`); the cache is read back afterwards (`fused_int4_paged_gather`), so that what is stored in 4
  bits is compared as the values it stands for.

`run` computes them in elementary torch operations, or with ``own`` set through the package.
Cache layout: ``k_data / v_data [pages, 16, Hkv, D/2]`` uint8 (low nibble first), ``k_scale / v_scale [pages, 16, Hkv,
D/32]`` fp16, weights ``mass [pages, Hkv, 16]`` fp32.
"""
import functools
import math
import os
import sys

import torch

own = False

PAGE = 16
GROUP = 32
DEV = "cuda"
LOG2E = 1.0 / math.log(2.0)
NOWHERE = 1 << 30  # a first visible token that no sequence has: the row sees nothing


# ------------------------------------------------------------------ cases
def _attend(name, **kw):
    return dict(dict(name=name, op="attend", hq=32, hkv=8, dim=128, dtype="float16", cap=0.0, bias=False, window=0,
                     prefix=0, docs=0, blank=0), **kw)


def _mass(name, **kw):
    return dict(_attend(name), **dict(dict(op="mass", decay=1.0, first=False), **kw))


def _evict(name, **kw):
    return dict(dict(name=name, op="evict", hkv=8, dim=128, sink=4, recent=64), **kw)


def listed():
    return [
        # two whole prompts, attended to as they were cached
        _attend("prompt 2x4096", seqs=2, new=4096, history=0),
        # a chunk of a long prompt behind what is cached already, logits capped
        _attend("chunk 2048 at 30720 cap", seqs=1, new=2048, history=30720, dtype="bfloat16", cap=50.0),
        # a packed batch of ragged prompts: documents, a bias by distance, a padded end that sees nothing; every head with
        # keys of its own
        _attend("documents 5x1021 bias", seqs=5, new=1021, history=0, hq=16, hkv=16, dim=64, docs=3, blank=2, bias=True,
                dtype="bfloat16"),
        # a picture's tokens see one another, the text behind them a window and the picture
        _attend("prefix 8x1500 window", seqs=8, new=1500, history=100, prefix=256, window=512),
        # drafts of five tokens checked against conversations of a few thousand
        _attend("draft 16x5", seqs=16, new=5, history=4091),
        # one token each of 64 conversations, logits capped
        _attend("token 64x4096 cap", seqs=64, new=1, history=4095, cap=30.0),
        # one token of one short conversation: latency
        _attend("token 1x517", seqs=1, new=1, history=516, hq=16, hkv=16, dim=64),
        # the weights that a decode step's queries gave
        _mass("mass token 64x4096", seqs=64, new=1, history=4095),
        # the weights that a prompt's last 32 tokens gave, by which its cache is thinned out
        _mass("mass last 32 of 8x8191", seqs=8, new=32, history=8159, dtype="bfloat16", first=True),
        # after a decode step: one token too many in 16 conversations
        _evict("evict step 16x1025", seqs=16, length=1025, budget=1024),
        # after a prompt: ragged caches cut to an eighth
        _evict("evict 8x8192 to 1024", seqs=8, length=8192, budget=1024),
        # one very long conversation
        _evict("evict 1x131072 to 4096", seqs=1, length=131072, budget=4096, recent=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "mass", "evict"])
    dim = rng.choice([64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    if op == "evict":
        seqs = _log(rng, 1, 32)
        budget = _log(rng, 16, min(8192, 16384 // seqs))
        sink = rng.choice([0, 1, 4])
        c = _evict(None, seqs=seqs, length=budget + _log(rng, 1, max(2, min(131072, 262144 // seqs) - budget)),
                   budget=budget, hkv=hkv, dim=dim, sink=sink, recent=rng.randint(0, min(256, budget - sink)))
        del c["name"]
        return c
    hq = hkv * rng.choice([1, 2, 3, 4, 8])
    seqs = _log(rng, 1, 64)
    kind = rng.choice(["token", "draft", "chunk", "chunk"])
    if op == "mass":
        new = {"token": 1, "draft": rng.randint(2, 8), "chunk": _log(rng, 9, 64)}[kind]
    else:
        new = {"token": 1, "draft": rng.randint(2, 8), "chunk": _log(rng, 9, max(10, 8192 // seqs))}[kind]
    # all scores of the batch, with its padding, at most 2^28; all tokens at most those of the longest listed batch
    most = min((1 << 28) // (seqs * new * hq) - new, 262144 // seqs - new)
    history = _log(rng, 1, most) - 1 if most >= 1 else 0
    kw = dict(seqs=seqs, new=new, history=history, hq=hq, hkv=hkv, dim=dim, dtype=rng.choice(["float16", "bfloat16"]),
              cap=rng.choice([0.0, 0.0, 30.0, 50.0]), bias=rng.random() < 0.3,
              window=rng.choice([0, 0, _log(rng, 1, 4096)]), prefix=rng.choice([0, 0, rng.randint(1, 300)]),
              docs=rng.choice([0, 0, rng.randint(2, 5)]), blank=rng.choice([0, 0, 0, 1]) if new > 1 else 0)
    if op == "mass":
        c = _mass(None, decay=rng.choice([1.0, 0.95]), first=rng.random() < 0.5, **kw)
    else:
        c = _attend(None, **kw)
    del c["name"]
    return c


def _ragged(top, n):
    """The first has `top`, the others up to a fifth less (host numbers, the same for every seed)."""
    return [max(1, top - (i * 7919) % max(1, top // 5 + 1)) for i in range(n)]


def _pages(n):
    return -(-n // PAGE)


def _batch(case):
    """New tokens and cached tokens (the new ones among them) of each sequence."""
    new = _ragged(case["new"], case["seqs"])
    return new, [n + (h if case["history"] else 0) for n, h in zip(new, _ragged(max(1, case["history"]), case["seqs"]))]


def _first_visible(case, new, lens):
    """Each new token's first visible token: its document's first, or nowhere for the last `blank` ones."""
    out = []
    for n, length in zip(new, lens):
        for i in range(n):
            pos = length - n + i
            first = 0
            if case["docs"]:
                first = max(length * d // case["docs"] for d in range(case["docs"]) if length * d // case["docs"] <= pos)
            out.append(NOWHERE if i >= n - case["blank"] else first)
    return out


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _table(g, counts):
    """Scattered disjoint pages: [B, max pages] int32, unused columns pointing at page 0."""
    total = sum(counts)
    ids = torch.randperm(total, generator=g, device=DEV).int()
    bt = torch.zeros(len(counts), max(counts), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(counts):
        bt[b, :n] = ids[at:at + n]
        at += n
    return bt, total


def _stored(g, pages, hkv, dim):
    """A cache as quantisation of normal keys and values leaves it: nibbles in [-7, 7], scales near amax / 7."""
    def data():
        q = (_randn(g, pages, PAGE, hkv, dim) * 3.0).round_().clamp_(-7, 7).to(torch.int8)
        return ((q[..., 0::2] & 15) | (q[..., 1::2] << 4)).view(torch.uint8)

    def scale():
        return (0.28 + 0.06 * _randn(g, pages, PAGE, hkv, dim // GROUP)).clamp_(0.1, 0.6).half()
    return data(), data(), scale(), scale()


def prepare(case, seed):
    g = _gen(seed)
    hkv, dim = case["hkv"], case["dim"]
    if case["op"] == "evict":
        lens = _ragged(case["length"], case["seqs"])
        bt, pages = _table(g, [_pages(n) for n in lens])
        kept = [min(n, case["budget"]) for n in lens]
        cu = [sum(kept[:b]) for b in range(len(kept) + 1)]
        # weights as attention leaves them: a few tokens have most
        return dict(case=case, cache=_stored(g, pages, hkv, dim), block_table=bt, lens=_ints(lens), cu=_ints(cu),
                    tokens=cu[-1], counts=torch.tensor(kept, device=DEV), longest=max(lens),
                    mass=(2.0 * _randn(g, pages, hkv, PAGE)).exp())
    new, lens = _batch(case)
    bt, pages = _table(g, [_pages(n) for n in lens])
    cache = _stored(g, pages, hkv, dim)
    cu = [sum(new[:b]) for b in range(len(new) + 1)]
    s = dict(case=case, cache=cache, block_table=bt, lens=_ints(lens), cu=_ints(cu), longest=max(lens),
             counts=torch.tensor(new, device=DEV), query=_randn(g, cu[-1], case["hq"], dim).to(getattr(torch, case["dtype"])),
             slopes=None, prefix=None, first_visible=None)
    if case["bias"]:
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / case["hq"]) for h in range(case["hq"])], device=DEV)
    if case["prefix"]:
        s["prefix"] = _ints([min(case["prefix"], n) for n in lens])
    if case["docs"] or case["blank"]:
        s["first_visible"] = _ints(_first_visible(case, new, lens))
    if case["op"] == "mass":
        s["mass"] = _randn(g, pages, hkv, PAGE).exp()
        s["first"] = _ints([0] * len(lens) if case["first"] else [n - m for n, m in zip(lens, new)])
        # the log-sum-exp that the attention of the same queries left
        logit = _logits(s)
        top = logit.amax(-1, keepdim=True)
        top = torch.where(top == -math.inf, 0.0, top)
        s["lse"] = _rows(s, ((top + (logit - top).exp().sum(-1, keepdim=True).log()) * LOG2E).squeeze(-1))
    return s


# ------------------------------------------------------------------ the plain forms
def _unpack(data, scale):
    lo = (data & 15).to(torch.float32)
    hi = (data >> 4).to(torch.float32)
    q = torch.stack((lo, hi), dim=-1).flatten(-2)
    q = torch.where(q >= 8, q - 16, q)
    return (q.unflatten(-1, (-1, GROUP)) * scale.float()[..., None]).flatten(-2)


def _dense(s, data, scale):
    """[B, Hkv, longest, D]: each sequence's keys or values, side by side."""
    pages = s["block_table"][:, :_pages(s["longest"])].long()
    return _unpack(data[pages], scale[pages]).flatten(1, 2)[:, :s["longest"]].transpose(1, 2)


def _places(s):
    """Sequence and place in it of each query row."""
    t = s["query"].shape[0]
    seq = torch.repeat_interleave(torch.arange(s["counts"].shape[0], device=DEV), s["counts"], output_size=t)
    return seq, torch.arange(t, device=DEV) - s["cu"][seq]


def _padded(s, x, fill):
    """Rows [T, ..] as [B, most rows, ..]."""
    seq, at = _places(s)
    out = torch.full((s["counts"].shape[0], s["case"]["new"], *x.shape[1:]), fill, dtype=x.dtype, device=DEV)
    out[seq, at] = x
    return out


def _rows(s, x):
    """[B, Hkv, group, rows, ..] back as [T, Hq, ..]."""
    seq, at = _places(s)
    return x.flatten(1, 2).transpose(1, 2)[seq, at]


def _logits(s):
    """[B, Hkv, group, rows, tokens]: scaled, capped and biased logits, -inf where a token is not visible."""
    c = s["case"]
    q = _padded(s, s["query"].float(), 0.0).unflatten(2, (c["hkv"], -1)).permute(0, 2, 3, 1, 4)
    key = _dense(s, s["cache"][0], s["cache"][2])
    x = (q.flatten(2, 3) @ key.transpose(-1, -2)).unflatten(2, q.shape[2:4]) * c["dim"] ** -0.5
    if c["cap"]:
        x = c["cap"] * (x / c["cap"]).tanh()
    col = torch.arange(s["longest"], device=DEV)
    pos = ((s["lens"] - s["counts"])[:, None] + torch.arange(c["new"], device=DEV))[:, :, None]  # [B, rows, 1]
    if s["slopes"] is not None:
        x = x - s["slopes"].view(c["hkv"], -1, 1, 1) * (pos - col).abs()[:, None, None]
    seen = col <= pos
    if c["window"]:
        seen = seen & (col > pos - c["window"])
    if s["prefix"] is not None:
        seen = seen | (col < s["prefix"][:, None, None])
    if s["first_visible"] is not None:
        seen = seen & (col >= _padded(s, s["first_visible"], 0)[:, :, None])
    seen = seen & (col < s["lens"][:, None, None])
    return torch.where(seen[:, None, None], x, -math.inf)


def _attend_plain(s):
    logit = _logits(s)
    top = logit.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weight = (logit - top).exp()
    total = weight.sum(-1, keepdim=True)
    value = _dense(s, s["cache"][1], s["cache"][3])
    out = (weight.flatten(2, 3) @ value).unflatten(2, weight.shape[2:4]) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()) * LOG2E
    return {"out": _rows(s, out).to(s["query"].dtype), "lse": _rows(s, lse.squeeze(-1))}


def _mass_plain(s):
    c = s["case"]
    lse = _padded(s, s["lse"], 0.0).unflatten(2, (c["hkv"], -1)).permute(0, 2, 3, 1)[..., None] / LOG2E
    logit = _logits(s)
    there = torch.arange(c["new"], device=DEV) < s["counts"][:, None]
    logit = torch.where(there[:, None, None, :, None], logit, -math.inf)  # (a shorter sequence's missing rows)
    weight = torch.where(logit == -math.inf, 0.0, (logit - lse).exp()).sum((2, 3))  # [B, Hkv, tokens]
    col = torch.arange(s["longest"], device=DEV)
    live = (col < s["lens"][:, None]).nonzero(as_tuple=True)
    page, at = s["block_table"][live[0], live[1] // PAGE].long(), live[1] % PAGE
    before = s["mass"][page, :, at]  # [tokens, Hkv]
    before = torch.where((live[1] >= s["first"][live[0]])[:, None], 0.0, before * c["decay"])
    s["mass"][page, :, at] = before + weight.transpose(1, 2)[live]
    return {"mass": s["mass"]}


def _kept(s):
    """[B, Hkv, budget]: the token that each place of the thinned cache holds, -1 behind the last."""
    c = s["case"]
    budget, sink, recent = c["budget"], c["sink"], c["recent"]
    heavy = budget - recent
    lens = s["lens"].long()[:, None, None]
    col = torch.arange(s["longest"], device=DEV)
    mass = s["mass"][s["block_table"][:, :_pages(s["longest"])].long()].transpose(1, 2).flatten(2)[..., :s["longest"]]
    open_ = (col >= sink) & (col < lens - recent)
    score = torch.where(open_, mass, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :heavy - sink]  # ties: the lowest token
    chosen = torch.zeros(score.shape, dtype=torch.bool, device=DEV).scatter_(2, order, True) & (lens > budget)
    place = torch.arange(budget, device=DEV).expand(*score.shape[:2], budget).contiguous()
    moving = chosen & (col >= heavy)
    hole = ((col >= sink) & (col < heavy) & ~chosen & (lens > budget))[..., :budget]
    place[hole] = moving.nonzero()[:, 2]  # both in rising order, as many of one as of the other
    place[..., heavy:] = torch.where(lens > budget, lens - budget + place[..., heavy:], place[..., heavy:])
    return torch.where(torch.arange(budget, device=DEV) < lens, place, -1)


def _evict_plain(s):
    c = s["case"]
    kept = _kept(s)
    b, h, to = (kept >= 0).nonzero(as_tuple=True)
    src = kept[b, h, to]
    old = s["block_table"][b, src // PAGE].long(), src % PAGE
    new = s["block_table"][b, to // PAGE].long(), to % PAGE
    for x in s["cache"]:
        x[new[0], new[1], h] = x[old[0], old[1], h]
    s["mass"][new[0], h, new[1]] = s["mass"][old[0], h, old[1]]
    seq = torch.repeat_interleave(torch.arange(s["counts"].shape[0], device=DEV), s["counts"], output_size=s["tokens"])
    at = torch.arange(s["tokens"], device=DEV) - s["cu"][seq]
    page, at = s["block_table"][seq, at // PAGE].long(), at % PAGE
    kd, vd, ks, vs = (x[page, at] for x in s["cache"])
    return {"key": _unpack(kd, ks).half(), "value": _unpack(vd, vs).half(), "mass": s["mass"], "kept": kept.int(),
            "lens": s["lens"].clamp(max=c["budget"])}


# ------------------------------------------------------------------ the package's calls
@functools.lru_cache(maxsize=None)
def _package():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "iris-kernel_b200"))
    import iris_kernel
    from iris_kernel import fused_kv, varlen_attention

    iris_kernel.set_validation_mode("deferred")  # as in a serving loop: errors are read between steps
    return fused_kv, varlen_attention


def _how(s):
    c = s["case"]
    return dict(cu_seqlens=None if c["new"] == 1 else s["cu"], logit_cap=c["cap"], slopes=s["slopes"], window=c["window"],
                prefix_lens=s["prefix"], first_visible=s["first_visible"])


def _attend_own(s):
    out, lse = _package()[1].fused_int4_paged_varlen_attention(s["query"], *s["cache"], s["block_table"], s["lens"],
                                                               return_lse=True, **_how(s))
    return {"out": out, "lse": lse}


def _mass_own(s):
    _package()[1].fused_int4_paged_attention_mass(s["query"], s["lse"], s["cache"][0], s["cache"][2], s["block_table"],
                                                  s["lens"], s["mass"], first_token=s["first"], decay=s["case"]["decay"],
                                                  **_how(s))
    return {"mass": s["mass"]}


def _evict_own(s):
    kv, c = _package()[0], s["case"]
    lens, kept = kv.fused_int4_paged_evict(*s["cache"], s["mass"], s["block_table"], s["lens"], budget=c["budget"],
                                           sink_tokens=c["sink"], recent_tokens=c["recent"], return_kept=True)
    k, v = kv.fused_int4_paged_gather(*s["cache"], s["block_table"], s["cu"], num_tokens=s["tokens"])
    return {"key": k, "value": v, "mass": s["mass"], "kept": kept, "lens": lens}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attend": _attend_own, "mass": _mass_own, "evict": _evict_own}[op](state)
    return {"attend": _attend_plain, "mass": _mass_plain, "evict": _evict_plain}[op](state)


# ------------------------------------------------------------------ definitions in 64 bits
def _nibbles64(data, scale):
    b = data.to(torch.int64)
    q = torch.empty(*b.shape[:-1], 2 * b.shape[-1], dtype=torch.float64, device=b.device)
    q[..., 0::2] = ((b & 15) ^ 8) - 8
    q[..., 1::2] = ((b >> 4) ^ 8) - 8
    return q * scale.to(torch.float64).repeat_interleave(GROUP, dim=-1)


def _tokens(s, b, n):
    """Page and place in it of a sequence's first n tokens."""
    t = torch.arange(n, device=DEV)
    return s["block_table"][b].long()[t // PAGE], t % PAGE


def _scores64(s, b, h, r0, r1):
    """Logits of query head h's rows r0 .. r1 of the batch, all of sequence b, over its tokens."""
    c = s["case"]
    n = int(s["lens"][b])
    page, at = _tokens(s, b, n)
    kv = h // (c["hq"] // c["hkv"])
    key = _nibbles64(s["cache"][0][page, at, kv], s["cache"][2][page, at, kv])
    x = s["query"][r0:r1, h].to(torch.float64) @ key.t() / math.sqrt(c["dim"])
    if c["cap"]:
        x = torch.tanh(x / c["cap"]) * c["cap"]
    end = int(s["cu"][b + 1])
    pos = torch.arange(r0, r1, device=DEV)[:, None] + (n - end)
    col = torch.arange(n, device=DEV)[None]
    if s["slopes"] is not None:
        x = x - s["slopes"][h].to(torch.float64) * (pos - col).abs()
    hidden = col > pos
    if c["window"]:
        hidden |= pos - col >= c["window"]
    if s["prefix"] is not None:
        hidden &= col >= int(s["prefix"][b])
    if s["first_visible"] is not None:
        hidden |= col < s["first_visible"][r0:r1, None]
    return x.masked_fill(hidden, -math.inf)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "evict":
        return _exact_evict(s)
    t, hq, hkv = s["query"].shape[0], case["hq"], case["hkv"]
    cu = s["cu"].tolist()
    if case["op"] == "attend":
        out = torch.zeros(t, hq, case["dim"], dtype=torch.float64, device=DEV)
        lse = torch.full((t, hq), -math.inf, dtype=torch.float64, device=DEV)
        for b, n in enumerate(s["lens"].tolist()):
            page, at = _tokens(s, b, n)
            for h in range(hq):
                value = _nibbles64(s["cache"][1][page, at, h // (hq // hkv)], s["cache"][3][page, at, h // (hq // hkv)])
                x = _scores64(s, b, h, cu[b], cu[b + 1])
                lse[cu[b]:cu[b + 1], h] = torch.logsumexp(x, -1) / math.log(2.0)
                out[cu[b]:cu[b + 1], h] = torch.nan_to_num(torch.softmax(x, -1), nan=0.0) @ value
        return {"out": out, "lse": lse}
    mass = s["mass"].to(torch.float64)
    lse = s["lse"].to(torch.float64) * math.log(2.0)
    for b, n in enumerate(s["lens"].tolist()):
        page, at = _tokens(s, b, n)
        for h in range(hkv):
            before = mass[page, h, at] * case["decay"]
            before[int(s["first"][b]):] = 0.0
            for q in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                x = _scores64(s, b, q, cu[b], cu[b + 1])
                before += torch.where(x > -math.inf, (x - lse[cu[b]:cu[b + 1], q, None]).exp(), 0.0).sum(0)
            mass[page, h, at] = before
    return {"mass": mass}


def _exact_evict(s):
    c = s["case"]
    lens = s["lens"].tolist()
    kept = torch.full((len(lens), c["hkv"], c["budget"]), -1, dtype=torch.int32)
    mass = s["mass"].cpu()
    table = s["block_table"].cpu().long()
    kd, vd = _nibbles64(s["cache"][0], s["cache"][2]), _nibbles64(s["cache"][1], s["cache"][3])
    moved, keys, values = s["mass"].to(torch.float64), [], []
    for b, n in enumerate(lens):
        t = torch.arange(n)
        heavy = c["budget"] - c["recent"]
        rows = []
        for h in range(c["hkv"]):
            place = list(range(min(n, c["budget"])))
            if n > c["budget"]:
                weight = mass[table[b, t // PAGE], h, t % PAGE].tolist()
                best = sorted(range(c["sink"], n - c["recent"]), key=lambda i: (-weight[i], i))[:heavy - c["sink"]]
                best = set(best)
                late = iter(sorted(i for i in best if i >= heavy))
                for i in range(c["sink"], heavy):
                    if i not in best:
                        place[i] = next(late)
                place[heavy:] = range(n - c["recent"], n)
            kept[b, h, :len(place)] = torch.tensor(place, dtype=torch.int32)
            rows.append(torch.tensor(place))
        rows = torch.stack(rows).to(DEV)  # [Hkv, kept]
        to = torch.arange(rows.shape[1], device=DEV)
        row = s["block_table"][b].long()
        head = torch.arange(c["hkv"], device=DEV)[:, None]
        keys.append(kd[row[rows // PAGE], rows % PAGE, head].transpose(0, 1))
        values.append(vd[row[rows // PAGE], rows % PAGE, head].transpose(0, 1))
        moved[row[to // PAGE], head, to % PAGE] = s["mass"].to(torch.float64)[row[rows // PAGE], head, rows % PAGE]
    return {"key": torch.cat(keys), "value": torch.cat(values), "mass": moved, "kept": kept,
            "lens": torch.tensor([min(n, c["budget"]) for n in lens], dtype=torch.int32)}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    hkv, dim = case["hkv"], case["dim"]
    row = hkv * (dim // 2 + dim // GROUP * 2)  # one token's stored keys (or values), all heads
    if case["op"] == "evict":
        lens = _ragged(case["length"], case["seqs"])
        kept = sum(min(n, case["budget"]) for n in lens)
        # a head's kept token is read and written when it comes from behind the budget; of the others, evenly likely to
        # be kept, so many stay: that share of the open tokens lies before the heavy places' end
        heavy, moves = case["budget"] - case["recent"], 0.0
        for n in lens:
            if n > case["budget"]:
                open_ = n - case["recent"] - case["sink"]
                moves += (heavy - case["sink"]) * (1.0 - (heavy - case["sink"]) / open_) + case["recent"]
        weights = sum(n for n in lens if n > case["budget"]) * hkv * 4
        return {"bytes": moves * (4 * row + 4 * hkv) + weights + kept * (4 * hkv + 2 * row + 4 * hkv * dim),
                "flops": weights / 4 + kept * 2 * hkv * dim}
    new, lens = _batch(case)
    first = iter(_first_visible(case, new, lens)) if case["docs"] or case["blank"] else None
    pairs = read = 0
    for n, length in zip(new, lens):
        edge = [0] * (length + 1)  # tokens that any row sees
        for i in range(n):
            pos = length - n + i
            lo = max(0, pos - case["window"] + 1) if case["window"] else 0
            f = next(first) if first else 0
            pre = min(case["prefix"], length)
            spans = [(f, max(f, pre)), (max(f, lo, pre), pos + 1)] if pre else [(max(f, lo), pos + 1)]
            for a, e in spans:
                if e > a:
                    pairs += e - a
                    edge[a] += 1
                    edge[e] -= 1
        seen = 0
        for j in range(length):
            seen += edge[j]
            read += seen > 0
    tokens, pages = sum(new), sum(_pages(n) for n in lens)
    io = tokens * case["hq"] * dim * 2
    if case["op"] == "attend":
        return {"bytes": 2 * io + tokens * case["hq"] * 4 + read * 2 * row + 4 * pages, "flops": pairs * case["hq"] * 4 * dim}
    return {"bytes": io + tokens * case["hq"] * 4 + read * row + sum(lens) * hkv * 8 + 4 * pages,
            "flops": pairs * case["hq"] * 2 * dim}
