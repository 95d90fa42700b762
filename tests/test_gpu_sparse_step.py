"""The operators of the sparse decode together: SparseDecodeStep (append,
bounds, selection and attention in one CUDA graph) equals the same calls made
one by one, bit for bit, and the plain implementations on the same cache, over
steps that cross a page and with an idle row; a rejected append inside the
graph is reported and writes nothing; and on keys with a few outstanding
pages, the selected attention is close to the dense one."""
import numpy as np
import pytest
import torch

import _sparse_refs as R

pytestmark = pytest.mark.gpu

SECTIONS, D, HQ, HKV, KEEP = (16, 24, 24), 128, 8, 2, 6


def _setup(dtype, seed=0):
    rng = np.random.default_rng(seed)
    lens = [250, 15, 0, 97]  # the third row is idle
    width = 20
    bt = rng.permutation(4 * width).astype(np.int32).reshape(4, width)
    cache = R.random_cache(rng, 4 * width, HKV, D)
    half = D // 2
    ang = np.arange(400)[:, None] * 10000.0 ** (-np.arange(half) / half)
    t = dict(cache=[torch.from_numpy(x).cuda() for x in cache], bt=torch.from_numpy(bt).cuda(),
             lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
             cos=R.to_type(np.cos(ang), dtype).cuda(), sin=R.to_type(np.sin(ang), dtype).cuda(),
             bounds=torch.zeros(4 * width, HKV, 2, D, dtype=torch.int8, device="cuda"),
             step=torch.zeros(4 * width, HKV, device="cuda"))
    return rng, t


def _prefill_bounds(t):
    from iris_kernel.sparse_attention import fused_int4_page_bounds

    fused_int4_page_bounds(t["cache"][0], t["cache"][2], t["bt"], t["lens"], t["bounds"], t["step"])


def _tokens(rng, dtype, lens, bt):
    def make(*shape):
        return R.to_type(rng.standard_normal(shape), dtype).cuda()

    pos = torch.stack([lens, lens // 2, lens // 3]).int()
    page = bt.gather(1, (lens // 16).long().unsqueeze(1)).squeeze(1)
    slots = torch.where(lens > 0, page * 16 + lens % 16, -1).int()  # an idle row stays idle
    return make(4, HQ, D), make(4, HKV, D), make(4, HKV, D), pos, slots


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_graph_step_equals_the_calls_and_the_plain_forms(dtype):
    from iris_kernel.fused_kv import fused_mrope_int4_paged_append
    from iris_kernel.sparse_attention import (fused_int4_page_bounds, fused_int4_sparse_paged_decode_attention,
                                              fused_page_select)
    from iris_kernel.step import SparseDecodeStep

    rng, a = _setup(dtype)
    _, b = _setup(dtype)
    for t in (a, b):
        _prefill_bounds(t)
    step = SparseDecodeStep(*a["cache"], a["bounds"], a["step"], a["bt"], a["lens"], a["cos"], a["sin"],
                            num_q_heads=HQ, sections=SECTIONS, rotary_dim=D, max_pages=KEEP)
    for x, y in zip((*a["cache"], a["bounds"], a["step"]), (*b["cache"], b["bounds"], b["step"])):
        assert torch.equal(x, y)  # building the step has changed nothing
    for _ in range(9):  # 250 -> 259 and 15 -> 24 begin new pages
        query, key, value, pos, slots = _tokens(rng, dtype, b["lens"], b["bt"])
        for t in (a, b):
            t["lens"].add_((t["lens"] > 0).int())
        out = step(query, key, value, pos, slots, check=True).clone()
        rotated = fused_mrope_int4_paged_append(key, value, pos, slots, b["cos"], b["sin"], *b["cache"], query,
                                                sections=SECTIONS, rotary_dim=D, page_size=16)
        fused_int4_page_bounds(b["cache"][0], b["cache"][2], b["bt"], b["lens"], b["bounds"], b["step"],
                               first_token=b["lens"] - 1)
        lists, counts = fused_page_select(rotated, b["bounds"], b["step"], b["bt"], b["lens"], max_pages=KEEP)
        eager = fused_int4_sparse_paged_decode_attention(rotated, *b["cache"], b["bt"], b["lens"], lists, counts)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        for x, y in zip((*a["cache"], a["bounds"], a["step"]), (*b["cache"], b["bounds"], b["step"])):
            assert torch.equal(x, y)
    # the last step against the plain forms, from the cache as it is now
    cache = [x.cpu().numpy() for x in b["cache"]]
    bt, lens = b["bt"].cpu().numpy(), b["lens"].cpu().numpy()
    bounds, bstep = np.zeros(b["bounds"].shape, np.int8), np.zeros(b["step"].shape, np.float32)
    R.bounds_ref(cache[0], cache[2], bt, lens, None, bounds, bstep)
    used = np.concatenate([bt[i, :-(-int(n) // 16)] for i, n in enumerate(lens)])
    assert np.array_equal(b["bounds"].cpu().numpy()[used], bounds[used])
    want, n = R.select_ref(R.scores_ref(R.f32(rotated), bounds, bstep, bt, HKV), lens, KEEP, 1, 1)
    assert np.array_equal(lists.cpu().numpy(), want) and np.array_equal(counts.cpu().numpy(), n)
    ref, _ = R.attend_ref(R.f32(rotated), *cache, bt, lens, want, n)
    half_ulp = 2.0 ** (-11 if dtype == torch.float16 else -8)
    biggest = 7 * float(cache[3].max())
    assert (np.abs(out.double().cpu().numpy() - ref) <= half_ulp * np.abs(ref) + 2.0 ** -14 * biggest).all()
    assert not out[2].any()  # the idle row


def test_graph_step_reports_a_rejected_append():
    from iris_kernel.step import SparseDecodeStep

    rng, t = _setup(torch.float16, 1)
    _prefill_bounds(t)
    step = SparseDecodeStep(*t["cache"], t["bounds"], t["step"], t["bt"], t["lens"], t["cos"], t["sin"],
                            num_q_heads=HQ, sections=SECTIONS, rotary_dim=D, max_pages=KEEP)
    before = [x.clone() for x in t["cache"]]
    query, key, value, pos, slots = _tokens(rng, torch.float16, t["lens"], t["bt"])
    with pytest.raises(ValueError):
        step(query, key, value, pos, torch.full_like(slots, 5), check=True)  # one slot for all
    for x, y in zip(before, t["cache"]):
        assert torch.equal(x, y)
    with pytest.raises(ValueError):
        SparseDecodeStep(*t["cache"], t["bounds"], t["step"], t["bt"], t["lens"], t["cos"], t["sin"], num_q_heads=HQ,
                         sections=SECTIONS, rotary_dim=D, max_pages=KEEP, recent_pages=0)


def test_selection_finds_the_pages_that_matter():
    """Keys of a few pages point along the query, far above the others': their
    weight is all but the whole (the rest has below 2^-11 of it), so attention
    over the selection is the dense attention within the dense decode's own
    tolerance (max-abs 2e-3 / relative 1e-2)."""
    from iris_kernel.fused_attention import fused_int4_paged_decode_attention
    from iris_kernel.sparse_attention import (fused_int4_page_bounds, fused_int4_sparse_paged_decode_attention,
                                              fused_page_select)

    rng = np.random.default_rng(3)
    n, pages = 64 * 16, 64
    key = 0.3 * rng.standard_normal((pages, 16, HKV, D)).astype(np.float32)
    query = rng.standard_normal((1, HQ, D)).astype(np.float32)
    query = query / np.abs(query).max()
    query[0, 1:HQ // HKV], query[0, HQ // HKV + 1:] = query[0, 0], query[0, HQ // HKV]  # one direction a KV head
    chosen = [5, 17, 40]
    for page in chosen:
        for h in range(HKV):
            key[page, :, h] += 10.0 * query[0, h * (HQ // HKV)]
    kq, ks = R.quantise(key)
    vq, vs = R.quantise(rng.standard_normal((pages, 16, HKV, D)).astype(np.float32))
    cache = [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (R.pack(kq), R.pack(vq), ks, vs)]
    bt = torch.from_numpy(rng.permutation(pages).astype(np.int32)).cuda().view(1, pages)
    inverse = {int(p): c for c, p in enumerate(bt[0].tolist())}
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    q = R.to_type(query, torch.float16).cuda()
    bounds = torch.zeros(pages, HKV, 2, D, dtype=torch.int8, device="cuda")
    bstep = torch.zeros(pages, HKV, device="cuda")
    fused_int4_page_bounds(cache[0], cache[2], bt, lens, bounds, bstep)
    lists, counts = fused_page_select(q, bounds, bstep, bt, lens, max_pages=8)
    for h in range(HKV):
        assert {inverse[p] for p in chosen} <= set(lists[0, h].tolist())
    x = (R.f32(q)[0, 0] @ R.dequant(R.pack(kq), ks)[:, :, 0].reshape(-1, D).T) * D ** -0.5
    weight = np.exp(x - x.max())
    inside = np.zeros(pages, bool)
    inside[chosen] = True
    assert weight.reshape(pages, 16)[~inside].sum() < 2.0 ** -11 * weight.sum()
    sparse = fused_int4_sparse_paged_decode_attention(q, *cache, bt, lens, lists, counts).float()
    dense = fused_int4_paged_decode_attention(q, *cache, bt, lens).float()
    assert ((sparse - dense).abs() <= 2e-3 + 1e-2 * dense.abs()).all()
