"""Operators of sparse long-context decode over the INT4 paged cache, as measured cases.

Five operators that a serving loop runs next to the dense decode:

* ``append``: rotary positions with several axes, INT4 quantisation and paged append of a batch of
  new tokens, then the batch read back from the cache (`fused_mrope_int4_paged_append`,
  `fused_int4_paged_gather`): what is stored in 4 bits comes back as the values it stands for;
* ``read``: a cached context read back as dense keys and values (`fused_int4_paged_gather`);
* ``bounds``: per page, KV head and channel, the lowest and highest stored key
  (`fused_int4_page_bounds`);
* ``select``: per sequence and KV head, the pages whose keys could give the largest logits
  (`fused_page_select`);
* ``attend``: decode attention over the selected pages only
  (`fused_int4_sparse_paged_decode_attention`).

`run` computes them in elementary torch operations, or with ``own`` set through the package.
Cache layout: ``k_data / v_data [pages, 16, Hkv, D/2]`` uint8 (low nibble first), ``k_scale /
v_scale [pages, 16, Hkv, D/32]`` fp16, bounds ``[pages, Hkv, 2, D]`` int8 with one fp32 step per
page and head.
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
TINY = 2.0 ** -14  # smallest normal fp16: the floor of a group scale
TOP = 65504.0  # largest finite fp16: the ceiling of a group scale


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 64 conversations: one new token each, its query rotated in the same call
        dict(name="append step 64", op="append", seqs=64, new=1, history=4096, pad=0, hq=32, hkv=8, dim=128,
             rotary=128, sections="16,24,24", interleaved=False, dtype="float16", key_out=False),
        # an image prompt's prefill: 8192 tokens at once, the rotated keys wanted for the prefill attention
        dict(name="append prefill 8192", op="append", seqs=2, new=4096, history=0, pad=0, hq=32, hkv=8, dim=128,
             rotary=128, sections="24,20,20", interleaved=True, dtype="bfloat16", key_out=True),
        # ragged chunks behind a history that ends inside a page, padded to a fixed batch; half the dims rotate
        dict(name="append ragged 1021", op="append", seqs=5, new=203, history=37, pad=6, hq=16, hkv=16, dim=64,
             rotary=32, sections="4,6,6", interleaved=False, dtype="float16", key_out=False),
        # one short context read back
        dict(name="read 1x517", op="read", seqs=1, length=517, hkv=8, dim=64, dtype="float16"),
        # eight long prefixes read back for another chunk of prefill
        dict(name="read 8x8192", op="read", seqs=8, length=8192, hkv=8, dim=128, dtype="bfloat16"),
        # after a decode step: the last page of 64 sequences
        dict(name="bounds step 64", op="bounds", seqs=64, length=4097, new=1, hkv=8, dim=128),
        # after a prefill: every page of ragged prompts
        dict(name="bounds all 16x8191", op="bounds", seqs=16, length=8191, new=0, hkv=8, dim=128),
        # one very long conversation
        dict(name="select 1x131072", op="select", seqs=1, length=131072, hq=64, hkv=8, dim=128, budget=128,
             dtype="float16"),
        # a batch of ragged long contexts
        dict(name="select 64x16384", op="select", seqs=64, length=16384, hq=32, hkv=8, dim=128, budget=128,
             dtype="float16"),
        # one conversation's token over 2048 selected tokens a head
        dict(name="attend 1x128p", op="attend", seqs=1, length=131072, hq=64, hkv=8, dim=128, budget=128,
             dtype="float16"),
        # a batch's tokens over 2048 selected tokens a head
        dict(name="attend 64x128p", op="attend", seqs=64, length=8192, hq=32, hkv=8, dim=128, budget=128,
             dtype="float16"),
        # every head with keys of its own, ragged lengths, short lists
        dict(name="attend mha 96x45p", op="attend", seqs=96, length=4099, hq=16, hkv=16, dim=64, budget=45,
             dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "read", "bounds", "select", "attend"])
    dim = rng.choice([64, 128])
    hkv = rng.choice([1, 2, 4, 8, 16])
    if op == "append":
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, min(4096, 8192 // seqs)))
        rotary = rng.choice([dim, dim, dim // 2])
        a = rng.choice([2, 3, 3, 4])
        half, cut = rotary // 2, []
        for k in range(a - 1):
            cut.append(rng.randint(1, half - sum(cut) - (a - 1 - k)) if k else rng.randint(1, half // 2))
        cut.append(half - sum(cut))
        hkv = min(hkv, 8)
        return dict(op=op, seqs=seqs, new=new, history=rng.randint(0, 2000), pad=rng.choice([0, 0, 3]),
                    hq=hkv * rng.choice([1, 2, 4]), hkv=hkv, dim=dim, rotary=rotary,
                    sections=",".join(map(str, cut)), interleaved=rng.random() < 0.5,
                    dtype=rng.choice(["float16", "bfloat16"]), key_out=rng.random() < 0.5)
    hkv = min(hkv, 8)
    if op == "read":
        seqs = _log(rng, 1, 16)
        return dict(op=op, seqs=seqs, length=_log(rng, 1, 57000 // seqs), hkv=hkv, dim=dim,
                    dtype=rng.choice(["float16", "bfloat16"]))
    if op == "bounds":
        seqs = _log(rng, 1, 64)
        length = _log(rng, 1, 120000 // seqs)
        return dict(op=op, seqs=seqs, length=length, new=rng.choice([0, 1, min(length, 100)]), hkv=hkv, dim=dim)
    g = rng.choice([1, 2, 4, 8, 16])
    if op == "select":
        seqs = _log(rng, 1, 64)
        return dict(op=op, seqs=seqs, length=_log(rng, 1, min(200000, 900000 // seqs)), hq=hkv * g, hkv=hkv, dim=dim,
                    budget=_log(rng, 4, 512), dtype=rng.choice(["float16", "bfloat16"]))
    seqs = _log(rng, 1, 64)
    budget = _log(rng, 2, min(1024, 8192 // seqs))
    return dict(op=op, seqs=seqs, length=_log(rng, 1, min(131072, 524288 // seqs)), hq=hkv * g, hkv=hkv, dim=dim,
                budget=budget, dtype=rng.choice(["float16", "bfloat16"]))


def _lengths(case):
    """Ragged lengths: the first sequence has the case's length, the others end up to a fifth earlier
    (host numbers, the same for every seed, so that tables and outputs have one shape)."""
    n, top = case["seqs"], case["length"]
    return [max(1, top - (i * 7919) % max(1, top // 5 + 1)) for i in range(n)]


def _pages(n):
    return -(-n // PAGE)


def _axes(case):
    """Which position axis turns each frequency: runs of the sections, or the axes dealt out in turn,
    an axis that has its section's count being passed over."""
    left = [int(s) for s in case["sections"].split(",")]
    if not case["interleaved"]:
        return [a for a, s in enumerate(left) for _ in range(s)]
    out = []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _table(g, counts, width=None):
    """Scattered disjoint pages: [B, max pages] int32, unused columns pointing at page 0."""
    total = sum(counts)
    ids = torch.randperm(total, generator=g, device=DEV).int()
    bt = torch.zeros(len(counts), max(max(counts), width or 0), dtype=torch.int32, device=DEV)
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


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    hkv, dim = case["hkv"], case["dim"]
    if case["op"] == "append":
        dtype = getattr(torch, case["dtype"])
        b, n, t = case["seqs"], case["new"], case["seqs"] * case["new"] + case["pad"]
        hist = [case["history"] + (i * 13) % 29 for i in range(b)]
        bt, pages = _table(g, [_pages(h + n) for h in hist])
        cache = _stored(g, pages, hkv, dim)
        first = _ints(hist)
        index = first.long()[:, None] + torch.arange(n, device=DEV)  # index in the sequence, [B, n]
        slots = bt.gather(1, index // PAGE).long() * PAGE + index % PAGE
        slots = torch.cat([slots.reshape(-1), torch.full((case["pad"],), -1, device=DEV)]).int()
        # positions: text moves every axis by one; a picture (every second run of 256 tokens) stands still on
        # the first axis and counts rows and columns of a 16-wide grid on the others
        axes = len(case["sections"].split(","))
        pic = (index // 256) % 2 == 1
        rows = [torch.where(pic, index // 256 * 256 if a == 0 else index // 256 * 256
                            + (index % 256 // 16 if a == 1 else index % 16), index) for a in range(axes)]
        pos = torch.stack([torch.cat([r.reshape(-1), torch.zeros(case["pad"], dtype=torch.int64, device=DEV)])
                           for r in rows]).int()
        top = max(hist) + n
        half = case["rotary"] // 2
        inv = 10000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
        angle = torch.arange(top, device=DEV, dtype=torch.float64)[:, None] * inv
        key = _randn(g, t, hkv, dim)
        key[..., :4] *= 8.0  # a few channels stand out, as in trained models
        s.update(key=key.to(dtype), value=_randn(g, t, hkv, dim).to(dtype), query=_randn(g, t, case["hq"], dim).to(dtype),
                 positions=pos, slots=slots, cos=angle.cos().to(dtype), sin=angle.sin().to(dtype), cache=cache,
                 block_table=bt, first=first, cu=torch.arange(b + 1, device=DEV, dtype=torch.int32) * n, tokens=b * n,
                 counts=torch.full((b,), n, device=DEV), axis=torch.tensor(_axes(case), device=DEV),
                 sections=tuple(int(x) for x in case["sections"].split(",")))
        return s
    lens = _lengths(case)
    counts = [_pages(n) for n in lens]
    bt, pages = _table(g, counts)
    s.update(block_table=bt, lens=_ints(lens))
    if case["op"] == "read":
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        s.update(cache=_stored(g, pages, hkv, dim), cu=_ints(cu), tokens=cu[-1], counts=s["lens"].long(),
                 dtype=getattr(torch, case["dtype"]))
        return s
    if case["op"] == "bounds":
        kd, _, ks, _ = _stored(g, pages, hkv, dim)
        first = [max(0, n - case["new"]) if case["new"] else 0 for n in lens]
        changed = [_pages(n) - f // PAGE for n, f in zip(lens, first)]
        s.update(k_data=kd, k_scale=ks, first=_ints(first), changed=torch.tensor(changed, device=DEV),
                 total=sum(changed), bounds=torch.zeros(pages, hkv, 2, dim, dtype=torch.int8, device=DEV),
                 step=torch.zeros(pages, hkv, dtype=torch.float32, device=DEV),
                 values=torch.zeros(pages, hkv, 2, dim, dtype=torch.float16, device=DEV))
        return s
    s["query"] = _randn(g, case["seqs"], case["hq"], dim).to(getattr(torch, case["dtype"]))
    if case["op"] == "select":
        # the lowest and highest of 16 normal keys lie near -1.77 and 1.77, around a mean of the channel's own
        mid = _randn(g, 1, hkv, dim)
        high = mid + 1.77 + 0.5 * _randn(g, pages, hkv, dim)
        low = torch.minimum(mid - 1.77 + 0.5 * _randn(g, pages, hkv, dim), high)
        both = torch.stack([low, high], dim=2)
        step = both.abs().amax((2, 3)) / 127
        s.update(bounds=(both / step[..., None, None]).round().clamp(-127, 127).to(torch.int8), step=step)
        return s
    # attend: what a selection gives: distinct pages in rising order, the first and the last among them
    budget, b = case["budget"], case["seqs"]
    npages = torch.tensor(counts, device=DEV)
    score = torch.rand(b, hkv, bt.shape[1], generator=g, device=DEV)
    col = torch.arange(bt.shape[1], device=DEV)
    score[:, :, 0] = 2.0
    score = torch.where(col == npages[:, None, None] - 1, 3.0, score)
    score = torch.where(col < npages[:, None, None], score, -1.0)
    take = min(budget, bt.shape[1])
    got, at = score.topk(take, dim=-1)
    at = torch.where(got > 0, at, 1 << 30).sort(-1).values
    lists = torch.full((b, hkv, budget), -1, dtype=torch.int32, device=DEV)
    lists[:, :, :take] = torch.where(at < (1 << 30), at, -1).int()
    s.update(cache=_stored(g, pages, hkv, dim), lists=lists, listed=(lists >= 0).sum(-1).int())
    return s


# ------------------------------------------------------------------ the plain forms
def _unpack(data, scale):
    lo = (data & 15).to(torch.float32)
    hi = (data >> 4).to(torch.float32)
    q = torch.stack((lo, hi), dim=-1).flatten(-2)
    q = torch.where(q >= 8, q - 16, q)
    return (q.unflatten(-1, (-1, GROUP)) * scale.float()[..., None]).flatten(-2)


def _over(x, n):
    """x / n, rounded once (by a tensor: a division by a Python number multiplies with its reciprocal)."""
    return x / torch.full((), float(n), device=DEV)


def _quantise(x):
    """[.., D] fp32 -> packed bytes and fp16 scales, one a group of 32."""
    x = x.unflatten(-1, (-1, GROUP))
    scale = _over(x.abs().amax(-1), 7).clamp(min=TINY, max=TOP).half()
    q = (x / scale.float()[..., None]).round().clamp(-7, 7).to(torch.int8).flatten(-2)
    return ((q[..., 0::2] & 15) | (q[..., 1::2] << 4)).view(torch.uint8), scale


def _rotate(x, cos, sin, rotary):
    x = x.float()
    a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rotary:]], dim=-1)


def _angles(s, table):
    """[T, 1, rotary / 2]: each frequency's entry at its own axis's position."""
    half = table.shape[1]
    rows = s["positions"][s["axis"]].long()  # [half, T]
    return table[rows, torch.arange(half, device=DEV)[:, None]].t()[:, None]


def _read(s, first):
    """The cache rows of each sequence's tokens, one after another."""
    n = s["tokens"]
    seq = torch.repeat_interleave(torch.arange(s["counts"].shape[0], device=DEV), s["counts"], output_size=n)
    at = torch.arange(n, device=DEV) - s["cu"][seq] + (first[seq] if first is not None else 0)
    rows = s["block_table"][seq, at // PAGE].long() * PAGE + at % PAGE
    kd, vd, ks, vs = (x.flatten(0, 1)[rows] for x in s["cache"])
    return _unpack(kd, ks), _unpack(vd, vs)


def _append_plain(s):
    c, n = s["case"], s["tokens"]
    dtype = s["key"].dtype
    cos, sin = _angles(s, s["cos"].float()), _angles(s, s["sin"].float())
    query = _rotate(s["query"], cos, sin, c["rotary"])
    key = _rotate(s["key"], cos, sin, c["rotary"])
    live = (s["slots"] >= 0)[:, None, None]  # a padding token's rows come back as zeros
    slots = s["slots"][:n].long()
    kd, ks = _quantise(key[:n])
    vd, vs = _quantise(s["value"][:n].float())
    for cache, rows in zip(s["cache"], (kd, vd, ks, vs)):
        cache.view(-1, *cache.shape[2:])[slots] = rows
    k, v = _read(s, s["first"])
    out = {"query": torch.where(live, query, 0).to(dtype), "key": k.to(dtype), "value": v.to(dtype)}
    if c["key_out"]:
        out["rotated"] = torch.where(live, key, 0).to(dtype)
    return out


def _read_plain(s):
    k, v = _read(s, None)
    return {"key": k.to(s["dtype"]), "value": v.to(s["dtype"])}


def _bounds_plain(s):
    n = s["total"]
    seq = torch.repeat_interleave(torch.arange(s["changed"].shape[0], device=DEV), s["changed"], output_size=n)
    start = s["changed"].cumsum(0) - s["changed"]
    col = torch.arange(n, device=DEV) - start[seq] + s["first"][seq] // PAGE
    page = s["block_table"][seq, col].long()
    key = _unpack(s["k_data"][page], s["k_scale"][page])  # [n, 16, Hkv, D]
    there = (col[:, None] * PAGE + torch.arange(PAGE, device=DEV) < s["lens"][seq][:, None])[:, :, None, None]
    low = torch.where(there, key, math.inf).amin(1)
    high = torch.where(there, key, -math.inf).amax(1)
    step = _over(torch.maximum(low.abs(), high.abs()).amax(-1), 127)
    unit = torch.where(step > 0, step, 1.0)[..., None]
    codes = torch.stack([(low / unit).floor(), (high / unit).ceil()], dim=2).clamp(-127, 127)
    s["bounds"][page] = codes.to(torch.int8)
    s["step"][page] = step
    s["values"][page] = (codes * step[..., None, None]).half()
    return {"values": s["values"], "step": s["step"]}


def _scores(query, bounds, step, table, hkv):
    """[B, Hkv, pages]: the largest logit that any query head of the group could find in the page."""
    b, hq, dim = query.shape
    q = query.float()
    unit = _over(q.abs().amax(-1), 127)
    code = (q / torch.where(unit > 0, unit, 1.0)[..., None]).round().clamp(-127, 127)
    both = torch.cat([code.clamp(max=0), code.clamp(min=0)], dim=-1).view(b, hkv, hq // hkv, 2 * dim)
    page = bounds[table.long()].flatten(3).permute(0, 2, 3, 1).float()  # [B, Hkv, 2D, P]
    dot = both @ page  # whole numbers below 2^24: exact in fp32
    dot = dot * step[table.long()].permute(0, 2, 1)[:, :, None]
    return (dot * unit.view(b, hkv, -1, 1)).amax(2)


def _select_plain(s):
    c = s["case"]
    bt, budget = s["block_table"], c["budget"]
    score = _scores(s["query"], s["bounds"], s["step"], bt, c["hkv"])
    col = torch.arange(bt.shape[1], device=DEV)
    n = ((s["lens"] + PAGE - 1) // PAGE)[:, None, None]
    score = torch.where((col == 0) | (col == n - 1), math.inf, score)  # one page at each end is always kept
    score = torch.where(col < n, score, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :budget]  # ties: the lowest page
    order = torch.where(order < n, order, 1 << 30).sort(-1).values
    lists = torch.full((*order.shape[:2], budget), -1, dtype=torch.int32, device=DEV)
    lists[..., :order.shape[-1]] = torch.where(order < (1 << 30), order, -1).int()
    return {"pages": lists, "count": (lists >= 0).sum(-1).int()}


def _attend_plain(s, dtype=torch.float32):
    c = s["case"]
    b, hkv, dim, budget = c["seqs"], c["hkv"], c["dim"], c["budget"]
    lists = s["lists"]
    page = torch.gather(s["block_table"].long()[:, None].expand(-1, hkv, -1), 2, lists.long().clamp(min=0))
    head = torch.arange(hkv, device=DEV)[None, :, None]
    kd, vd, ks, vs = (x.permute(0, 2, 1, 3)[page, head] for x in s["cache"])  # [B, Hkv, K, 16, ..]
    key = _unpack(kd, ks).flatten(2, 3).to(dtype)
    value = _unpack(vd, vs).flatten(2, 3).to(dtype)
    query = s["query"].to(dtype).view(b, hkv, c["hq"] // hkv, dim)
    logit = (query @ key.transpose(-1, -2)) * dim ** -0.5
    token = lists.long()[..., None] * PAGE + torch.arange(PAGE, device=DEV)
    there = ((lists[..., None] >= 0) & (token < s["lens"].long()[:, None, None, None])).flatten(2)[:, :, None]
    logit = torch.where(there, logit, -math.inf)
    top = logit.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weight = (logit - top).exp()
    total = weight.sum(-1, keepdim=True)
    out = (weight @ value) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()) / math.log(2.0)
    return out.view(b, c["hq"], dim), lse.view(b, c["hq"])


# ------------------------------------------------------------------ the package's calls
@functools.lru_cache(maxsize=None)
def _package():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "iris-kernel_b200"))
    import iris_kernel
    from iris_kernel import fused_kv, sparse_attention

    iris_kernel.set_validation_mode("deferred")  # as in a serving loop: errors are read between steps
    return fused_kv, sparse_attention


def _append_own(s):
    kv, _ = _package()
    c = s["case"]
    dtype = s["key"].dtype
    rotated = torch.empty_like(s["key"]) if c["key_out"] else None
    query = kv.fused_mrope_int4_paged_append(
        s["key"], s["value"], s["positions"], s["slots"], s["cos"], s["sin"], *s["cache"], s["query"],
        sections=s["sections"], interleaved=c["interleaved"], rotary_dim=c["rotary"], page_size=PAGE, key_out=rotated)
    k, v = kv.fused_int4_paged_gather(*s["cache"], s["block_table"], s["cu"], num_tokens=s["tokens"],
                                      first_token=s["first"], dtype=dtype)
    out = {"query": query, "key": k, "value": v}
    if rotated is not None:
        out["rotated"] = rotated
    return out


def _read_own(s):
    k, v = _package()[0].fused_int4_paged_gather(*s["cache"], s["block_table"], s["cu"], num_tokens=s["tokens"],
                                                 dtype=s["dtype"])
    return {"key": k, "value": v}


def _bounds_own(s):
    _package()[1].fused_int4_page_bounds(s["k_data"], s["k_scale"], s["block_table"], s["lens"], s["bounds"], s["step"],
                                         first_token=s["first"], values=s["values"])
    return {"values": s["values"], "step": s["step"]}


def _select_own(s):
    lists, count = _package()[1].fused_page_select(s["query"], s["bounds"], s["step"], s["block_table"], s["lens"],
                                                   max_pages=s["case"]["budget"], sink_pages=1, recent_pages=1)
    return {"pages": lists, "count": count}


def _attend_own(s):
    out, lse = _package()[1].fused_int4_sparse_paged_decode_attention(
        s["query"], *s["cache"], s["block_table"], s["lens"], s["lists"], s["listed"], return_lse=True)
    return {"out": out, "lse": lse}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _append_own, "read": _read_own, "bounds": _bounds_own, "select": _select_own,
                "attend": _attend_own}[op](state)
    if op == "attend":
        out, lse = _attend_plain(state)
        return {"out": out.to(state["query"].dtype), "lse": lse}
    return {"append": _append_plain, "read": _read_plain, "bounds": _bounds_plain, "select": _select_plain}[op](state)


# ------------------------------------------------------------------ definitions in 64 bits
def _nibbles64(data, scale):
    b = data.to(torch.int64)
    q = torch.empty(*b.shape[:-1], 2 * b.shape[-1], dtype=torch.float64, device=b.device)
    q[..., 0::2] = ((b & 15) ^ 8) - 8
    q[..., 1::2] = ((b >> 4) ^ 8) - 8
    return q * scale.to(torch.float64).repeat_interleave(GROUP, dim=-1)


def _turn64(x, s, rotary):
    x = x.to(torch.float64)
    half = rotary // 2
    out = x.clone()
    for i, a in enumerate(_axes(s["case"])):
        c = s["cos"].to(torch.float64)[s["positions"][a].long(), i][:, None]
        d = s["sin"].to(torch.float64)[s["positions"][a].long(), i][:, None]
        out[..., i] = x[..., i] * c - x[..., i + half] * d
        out[..., i + half] = x[..., i + half] * c + x[..., i] * d
    return out


def _stored64(x):
    """What 4 bits and an fp16 scale a group keep of x."""
    y = x.reshape(*x.shape[:-1], -1, GROUP)
    scale = (y.abs().amax(-1) / 7).clamp(TINY, TOP).half().to(torch.float64)[..., None]
    return ((y / scale).round().clamp(-7, 7) * scale).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "append":
        n = s["tokens"]
        live = (s["slots"] >= 0).to(torch.float64)[:, None, None]
        key = _turn64(s["key"], s, case["rotary"])
        out = {"query": _turn64(s["query"], s, case["rotary"]) * live, "key": _stored64(key[:n]),
               "value": _stored64(s["value"][:n].to(torch.float64))}
        if case["key_out"]:
            out["rotated"] = key * live
        return out
    lens = s["lens"].tolist()
    if op == "read":
        kd, vd, ks, vs = s["cache"]
        key, value = [], []
        for b, n in enumerate(lens):
            ids = s["block_table"][b, :_pages(n)].long()
            key.append(_nibbles64(kd[ids].flatten(0, 1)[:n], ks[ids].flatten(0, 1)[:n]))
            value.append(_nibbles64(vd[ids].flatten(0, 1)[:n], vs[ids].flatten(0, 1)[:n]))
        return {"key": torch.cat(key), "value": torch.cat(value)}
    if op == "bounds":
        values = torch.zeros(s["values"].shape, dtype=torch.float64, device=DEV)
        step = torch.zeros(s["step"].shape, dtype=torch.float64, device=DEV)
        first = s["first"].tolist()
        for b, n in enumerate(lens):
            f = first[b] // PAGE
            ids = s["block_table"][b, f:_pages(n)].long()
            key = _nibbles64(s["k_data"][ids], s["k_scale"][ids])
            gone = torch.arange(f * PAGE, _pages(n) * PAGE, device=DEV).view(-1, PAGE) >= n
            both = torch.stack([key.masked_fill(gone[:, :, None, None], math.inf).amin(1),
                                key.masked_fill(gone[:, :, None, None], -math.inf).amax(1)], dim=2)
            unit = both.abs().amax((2, 3)) / 127
            u = unit.masked_fill(unit == 0, 1.0)[..., None]
            values[ids] = torch.stack([(both[:, :, 0] / u).floor() * u, (both[:, :, 1] / u).ceil() * u],
                                      dim=2).clamp(-127 * u[:, :, None], 127 * u[:, :, None])
            step[ids] = unit
        return {"values": values, "step": step}
    if op == "select":
        return None  # page numbers and counts only
    kd, vd, ks, vs = s["cache"]
    group = case["hq"] // case["hkv"]
    out = torch.zeros(case["seqs"], case["hq"], case["dim"], dtype=torch.float64, device=DEV)
    lse = torch.full((case["seqs"], case["hq"]), -math.inf, dtype=torch.float64, device=DEV)
    lists = s["lists"].tolist()
    for b, n in enumerate(lens):
        for h in range(case["hkv"]):
            cols = [p for p in lists[b][h] if p >= 0]
            if not cols:
                continue
            ids = s["block_table"][b][torch.tensor(cols, device=DEV)].long()
            tok = (torch.tensor(cols, device=DEV)[:, None] * PAGE + torch.arange(PAGE, device=DEV)).flatten()
            keep = tok < n
            key = _nibbles64(kd[ids, :, h], ks[ids, :, h]).flatten(0, 1)[keep]
            value = _nibbles64(vd[ids, :, h], vs[ids, :, h]).flatten(0, 1)[keep]
            q = s["query"][b, h * group:(h + 1) * group].to(torch.float64)
            x = q @ key.t() / math.sqrt(case["dim"])
            out[b, h * group:(h + 1) * group] = torch.softmax(x, -1) @ value
            lse[b, h * group:(h + 1) * group] = torch.logsumexp(x, -1) / math.log(2.0)
    return {"out": out, "lse": lse}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    hkv, dim, op = case["hkv"], case["dim"], case["op"]
    row = hkv * (dim // 2 + dim // GROUP * 2)  # one token's stored keys (or values), all heads
    if op == "append":
        n = case["seqs"] * case["new"]
        axes = len(case["sections"].split(","))
        # keys, values and queries in, positions and slots; the rotary rows (each needed once); rotated queries
        # (and keys) out; the stored rows written, then read back, and the values they stand for written
        b = n * (2 * hkv * dim * 2 + case["hq"] * dim * 4 + 4 * axes + 4)
        b += (case["history"] + case["new"]) * case["rotary"] * 2
        b += n * (hkv * dim * 2 if case["key_out"] else 0) + n * 2 * row * 2 + n * 2 * hkv * dim * 2
        return {"bytes": b, "flops": n * (6 * (case["hq"] + hkv) * case["rotary"] // 2 + 8 * hkv * dim)}
    lens = _lengths(case)
    pages = sum(_pages(n) for n in lens)
    if op == "read":
        n = sum(lens)
        return {"bytes": n * (2 * row + 2 * hkv * dim * 2) + 4 * pages, "flops": n * 2 * hkv * dim}
    if op == "bounds":
        first = [max(0, n - case["new"]) if case["new"] else 0 for n in lens]
        tokens = sum(n - f // PAGE * PAGE for n, f in zip(lens, first))
        changed = sum(_pages(n) - f // PAGE for n, f in zip(lens, first))
        return {"bytes": tokens * row + changed * (hkv * (2 * dim + 4 + 4 * dim) + 4),
                "flops": tokens * 3 * hkv * dim + changed * hkv * 6 * dim}
    io = case["seqs"] * case["hq"] * dim * 2
    if op == "select":
        return {"bytes": io + pages * (hkv * (2 * dim + 4) + 4) + case["seqs"] * hkv * (case["budget"] + 1) * 4,
                "flops": pages * case["hq"] * 2 * 2 * dim}
    kept = sum(min(case["budget"], _pages(n)) for n in lens)
    tokens = sum(min(case["budget"], _pages(n)) * PAGE - (-n) % PAGE for n in lens)
    return {"bytes": 2 * io + case["seqs"] * case["hq"] * 4 + tokens * 2 * row + kept * (hkv * 4 + 4),
            "flops": tokens * case["hq"] * 4 * dim}
