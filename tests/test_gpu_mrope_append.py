"""fused_mrope_int4_paged_append and fused_int4_paged_gather: bit for bit
against a plain fp32 implementation (the products of 16-bit values are exact
in fp32, every later rounding is part of the definition), odd sizes, strides,
paddings, non-finite values, refusals, and batches that must not be written."""
import numpy as np
import pytest
import torch

import _sparse_refs as R

pytestmark = pytest.mark.gpu


def _case(seed, T=7, hq=4, hkv=2, dim=128, rotary=None, sections=(16, 24, 24), dtype=torch.float16, pages=9, page=16,
          top=300, pad=0.15):
    rng = np.random.default_rng(seed)
    rotary = dim if rotary is None else rotary
    half = rotary // 2
    ang = np.arange(top)[:, None] * 10000.0 ** (-np.arange(half) / half)
    slots = rng.permutation(pages * page)[:T].astype(np.int32)
    slots[rng.random(T) < pad] = -1

    def dev(x):
        return to(x).cuda()

    def to(x):
        return R.to_type(x, dtype)

    key = rng.standard_normal((T, hkv, dim)).astype(np.float32)
    key[rng.random(key.shape) < 0.01] *= 20
    kd, vd, ks, vs = R.random_cache(rng, pages * page // 16 + 1, hkv, dim)
    cache = [x.reshape(-1, *x.shape[2:])[:pages * page].reshape(pages, page, *x.shape[2:]) for x in (kd, vd, ks, vs)]
    return dict(key=dev(key), value=dev(rng.standard_normal((T, hkv, dim))), query=dev(rng.standard_normal((T, hq, dim))),
                positions=torch.from_numpy(rng.integers(0, top, (len(sections), T)).astype(np.int32)).cuda(),
                slots=torch.from_numpy(slots).cuda(), cos=dev(np.cos(ang)), sin=dev(np.sin(ang)),
                cache=[torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in cache], sections=tuple(sections),
                rotary=rotary, page=page)


def _run(c, query=True, key_out=True, **kw):
    from iris_kernel.fused_kv import fused_mrope_int4_paged_append

    rotated = torch.empty(c["key"].shape, dtype=c["key"].dtype, device="cuda") if key_out else None
    out = fused_mrope_int4_paged_append(c["key"], c["value"], c["positions"], c["slots"], c["cos"], c["sin"],
                                        *c["cache"], c["query"] if query else None, sections=c["sections"],
                                        rotary_dim=c["rotary"], page_size=c["page"], key_out=rotated, **kw)
    torch.cuda.synchronize()
    return out, rotated


def _expect(c, interleaved=False):
    """(cache arrays, rotated queries, rotated keys)."""
    pos, slots = c["positions"].cpu().numpy(), c["slots"].cpu().numpy()
    live = slots >= 0
    args = (np.where(live, pos, 0), R.f32(c["cos"]), R.f32(c["sin"]), c["sections"], interleaved, c["rotary"])
    with np.errstate(all="ignore"):
        key, query = R.rotate(R.f32(c["key"]), *args), R.rotate(R.f32(c["query"]), *args)
    cache = [x.cpu().numpy().copy() for x in c["cache"]]
    for x, data, scale in ((key, 0, 2), (R.f32(c["value"]), 1, 3)):
        q, s = R.quantise(x)
        cache[data].reshape(-1, *cache[data].shape[2:])[slots[live]] = R.pack(q)[live]
        cache[scale].reshape(-1, *cache[scale].shape[2:])[slots[live]] = s[live]
    zero = live[:, None, None]
    return cache, np.where(zero, query, 0), np.where(zero, key, 0)


def _same_bits(got, want):
    """Equal bit for bit, NaN equal to NaN."""
    got, want = got.detach().cpu(), want if isinstance(want, torch.Tensor) else torch.from_numpy(want)
    assert got.dtype == want.dtype and got.shape == want.shape
    if got.is_floating_point():
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(got), nan)
        got, want = got.masked_fill(nan, 0), want.masked_fill(nan, 0)
    assert torch.equal(got, want)


def _check(c, interleaved=False, **kw):
    cache, query, key = _expect(c, interleaved)
    q, k = _run(c, interleaved=interleaved, **kw)
    for got, want in zip(c["cache"], cache):
        _same_bits(got, want)
    _same_bits(q, R.to_type(query, c["key"].dtype))
    _same_bits(k, R.to_type(key, c["key"].dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T", [1, 7, 128, 129, 300])
def test_matches_the_plain_form(T, interleaved, dtype):
    _check(_case(T, T=T, sections=(24, 20, 20), dtype=dtype, pages=24), interleaved)


@pytest.mark.parametrize("dim,rotary,sections", [
    (64, 64, (32,)), (64, 32, (4, 6, 6)), (64, 16, (1, 7)), (128, 48, (5, 9, 10)), (128, 128, (1, 62, 1)),
    (128, 128, (0, 64, 0)), (192, 192, (40, 30, 20, 6)), (256, 128, (16, 24, 24)), (320, 320, (100, 60)),
    (512, 512, (64, 96, 96))])
@pytest.mark.parametrize("interleaved", [False, True])
def test_head_dims_and_partial_rotation(dim, rotary, sections, interleaved):
    _check(_case(dim + rotary, T=5, hq=3, hkv=1, dim=dim, rotary=rotary, sections=sections), interleaved)
    _check(_case(dim + rotary, T=140, hq=3, hkv=3, dim=dim, rotary=rotary, sections=sections, pages=12), interleaved)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (5, 5), (24, 3), (64, 16)])
def test_head_counts(hq, hkv):
    _check(_case(hq, T=9, hq=hq, hkv=hkv))
    _check(_case(hq, T=150, hq=hq, hkv=hkv, pages=12))


def test_page_size_other_than_16():
    _check(_case(3, T=40, pages=7, page=11))


def test_without_queries_or_rotated_keys():
    c = _case(5)
    cache, query, _ = _expect(c)
    out, rotated = _run(c, query=False, key_out=False)
    assert out is None and rotated is None
    for got, want in zip(c["cache"], cache):
        _same_bits(got, want)
    c = _case(6)
    out = torch.empty_like(c["query"])
    assert _run(c, key_out=False, query_out=out)[0] is out
    _same_bits(out, R.to_type(_expect(c)[1], torch.float16))


@pytest.mark.parametrize("T", [6, 200])
def test_slices_of_a_fused_projection(T):
    c = _case(7, T=T, hq=4, hkv=2, pages=15)
    fused = torch.cat([c["query"], c["key"], c["value"]], dim=1).contiguous()
    c["query"], c["key"], c["value"] = fused[:, :4], fused[:, 4:6], fused[:, 6:]
    wide = torch.full((c["positions"].shape[0], T + 13), -5, dtype=torch.int32, device="cuda")
    wide[:, :T] = c["positions"]
    c["positions"] = wide[:, :T]
    _check(c)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [8, 136])
def test_values_that_are_not_finite_or_very_large(T, dtype):
    """A NaN or infinity takes its whole group with it and no other; finite
    bf16 groups too large for an fp16 scale saturate."""
    c = _case(8, T=T, dtype=dtype, pages=12, pad=0.0)
    big = 3.0e38 if dtype == torch.bfloat16 else 65504.0
    for x in (c["key"], c["value"]):
        x[0, 0, 3] = float("nan")
        x[1, 0, 40] = float("inf")
        x[2, 0, 70] = -float("inf")
        x[3, 0, :32] = big
        x[4, 0] = 0.0
        x[5, 0, ::2] = 2.0 ** -20
    _check(c)


def test_half_way_quotients_round_to_even():
    """x / scale = k + 1/2 exactly (scale a power of two): no rotation."""
    c = _case(9, T=4, hkv=2, hq=2, pad=0.0)
    c["cos"].fill_(1.0)
    c["sin"].zero_()
    for x in (c["key"], c["value"]):
        x[:] = (torch.arange(x.numel(), device="cuda") % 14 - 6.5).view(x.shape).to(x.dtype) * 0.25
        x[..., ::32] = 1.75
    _check(c)


def test_several_batches_and_padding_only():
    c = _case(10, T=5)
    c["slots"].fill_(-1)
    c["positions"].fill_(1 << 30)  # never looked at
    c["key"].fill_(float("nan"))
    before = [x.clone() for x in c["cache"]]
    q, k = _run(c)
    assert not q.any() and not k.any()
    for a, b in zip(before, c["cache"]):
        assert torch.equal(a, b)
    c = _case(11, T=0)
    q, k = _run(c)
    assert q.shape == (0, 4, 128)


@pytest.mark.parametrize("T", [20, 200])
@pytest.mark.parametrize("what,error", [("duplicate", ValueError), ("slot", IndexError), ("negative", IndexError),
                                        ("position", IndexError)])
def test_a_bad_batch_writes_nothing(T, what, error):
    c = _case(12, T=T, pages=15, pad=0.0)
    if what == "duplicate":
        c["slots"][T - 1] = c["slots"][0].clone()
    elif what == "slot":
        c["slots"][T // 2] = 15 * 16
    else:
        c["positions"][2, T // 2] = -1 if what == "negative" else 300
    before = [x.clone() for x in c["cache"]]
    with pytest.raises(error):
        _run(c)
    for a, b in zip(before, c["cache"]):
        assert torch.equal(a, b)
    _check(_case(13, T=T, pages=15))  # the next batch is written


@pytest.mark.parametrize("T", [20, 200, 2100])
def test_slots_past_the_cache_are_an_index_error_even_twice(T):
    c = _case(30, T=T, pages=140, pad=0.0)
    c["slots"][3] = c["slots"][T - 1] = 140 * 16
    with pytest.raises(IndexError):
        _run(c)


@pytest.mark.parametrize("T", [2048, 2049, 5000])
def test_large_batches(T):
    """Both forms of the duplicate check, and a duplicate far away."""
    c = _case(31, T=T, hq=2, hkv=1, dim=64, sections=(16, 8, 8), pages=330)
    _check(c)
    c = _case(32, T=T, hq=1, hkv=1, dim=64, sections=(16, 8, 8), pages=330, pad=0.0)
    before = [x.clone() for x in c["cache"]]
    c["slots"][T - 1] = c["slots"][7].clone()
    with pytest.raises(ValueError):
        _run(c)
    for x, y in zip(before, c["cache"]):
        assert torch.equal(x, y)


def test_positions_shared_by_the_axes_and_a_single_head():
    """One row of positions expanded over the axes, as text tokens have them,
    is the rotation with one axis."""
    c = _case(33, T=12, hq=2, hkv=1, pad=0.0)
    one = {**c, "positions": c["positions"][:1], "sections": (64,), "cache": [x.clone() for x in c["cache"]]}
    c["positions"] = c["positions"][:1].expand(3, -1)
    q, k = _run(c)
    q1, k1 = _run(one)
    _same_bits(q, q1.cpu())
    _same_bits(k, k1.cpu())
    for x, y in zip(c["cache"], one["cache"]):
        _same_bits(x, y.cpu())


def test_on_a_side_stream():
    c = _case(14, T=150, pages=12)
    want = _expect(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q, k = _run(c)
    for got, w in zip(c["cache"], want[0]):
        _same_bits(got, w)
    _same_bits(q, R.to_type(want[1], torch.float16))


def test_refusals():
    c = _case(15)

    def call(error, **change):
        with pytest.raises(error):
            _run({**c, **change}, **change.get("kw", {}))

    call(TypeError, key=c["key"].float(), value=c["value"].float())
    call(TypeError, value=c["value"].bfloat16())
    call(TypeError, positions=c["positions"].long())
    call(TypeError, cos=c["cos"].bfloat16())
    call(ValueError, positions=c["positions"][:2])
    call(ValueError, sections=(16, 24, 23))
    call(ValueError, sections=(-1, 33, 32))
    call(ValueError, sections=(13, 13, 13, 13, 12))
    call(ValueError, slots=c["slots"][:3])
    call(ValueError, key=c["key"].transpose(0, 1).contiguous().transpose(0, 1))
    call(ValueError, value=c["value"][:, :1])
    call(ValueError, cos=c["cos"][:, :32])
    call(ValueError, cache=[c["cache"][0][..., :32], *c["cache"][1:]])
    call(NotImplementedError, rotary=136)
    call(NotImplementedError, rotary=40)
    call(ValueError, page=8)
    flat = torch.zeros(c["key"].numel() + 1, dtype=torch.float16, device="cuda")
    call(ValueError, key=flat[1:].view(c["key"].shape))  # not on a 16-byte boundary
    call(ValueError, key=c["key"].cpu())
    with pytest.raises(ValueError):
        _run(c, key_out=False, query_out=c["query"])  # a rotation in place would read what it has overwritten
    with pytest.raises(NotImplementedError):
        _run(c, group_size=64)
    with pytest.raises(ValueError):
        _run(c, query=False, query_out=torch.empty_like(c["query"]))


@pytest.mark.parametrize("what", ["the same", "half over", "key", "k_data", "v_scale", "cos"])
def test_outputs_that_overlap_are_refused(what):
    """Rotated keys in the rotated queries' place, or in memory that the call
    reads or stores to: nothing is written."""
    from iris_kernel.fused_kv import fused_mrope_int4_paged_append

    c = _case(34, hq=2, hkv=2)
    n = c["query"].numel()

    def call(query_out, key_out):
        fused_mrope_int4_paged_append(c["key"], c["value"], c["positions"], c["slots"], c["cos"], c["sin"], *c["cache"],
                                      c["query"], sections=c["sections"], rotary_dim=c["rotary"], page_size=c["page"],
                                      query_out=query_out, key_out=key_out)
        torch.cuda.synchronize()

    room = torch.full((2 * n,), 3.0, dtype=torch.float16, device="cuda")
    query_out = room[:n].view(c["query"].shape)
    places = {"the same": query_out, "half over": room[n // 2:n // 2 + n].view(c["query"].shape), "key": c["key"]}
    if what in places:
        key_out = places[what]
    else:  # the output in the other tensor's memory
        big = torch.zeros(40960, dtype=torch.float16, device="cuda")
        key_out = big[:n].view(c["query"].shape)
        if what == "cos":
            c["cos"] = big[:c["cos"].numel()].view(c["cos"].shape).copy_(c["cos"])
        else:
            i = ["k_data", "v_data", "k_scale", "v_scale"].index(what)
            x = c["cache"][i]
            c["cache"][i] = big.view(x.dtype)[:x.numel()].view(x.shape).copy_(x)
    before = [x.clone() for x in c["cache"]]
    for outputs in ((query_out, key_out), (key_out, query_out)):
        with pytest.raises(ValueError, match="overlap"):
            call(*outputs)
    torch.cuda.synchronize()
    assert bool((room == 3).all())
    for x, y in zip(before, c["cache"]):
        assert torch.equal(x, y)
    call(query_out, room[n:].view(c["query"].shape))  # one right after the other
    assert not bool((room == 3).any())


# ------------------------------------------------------------------ read back
def _table(rng, lens, page, width=None):
    counts = [-(-n // page) for n in lens]
    ids = rng.permutation(sum(counts) + 3).astype(np.int32)
    bt = np.full((len(lens), width or max(1, max(counts))), -7, np.int32)  # unused columns are never read
    at = 0
    for b, n in enumerate(counts):
        bt[b, :n] = ids[at:at + n]
        at += n
    return bt, sum(counts) + 3


def _gather_expect(cache, bt, lens, first, dtype, page):
    out = []
    for data, scale in ((cache[0], cache[2]), (cache[1], cache[3])):
        rows = [R.dequant(data[bt[b, t // page], t % page], scale[bt[b, t // page], t % page])
                for b, n in enumerate(lens) for t in range(first[b], n)]
        out.append(R.to_type(np.stack(rows) if rows else np.zeros((0, *data.shape[2:-1], data.shape[-1] * 2)), dtype))
    return out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hkv,dim,page,lens,first", [
    (1, 64, 16, [1], [0]), (2, 128, 16, [37, 0, 16, 17, 1], [0, 0, 3, 16, 0]), (3, 32, 16, [50, 49], [49, 0]),
    (8, 128, 16, [200, 0, 0, 333], None), (1, 96, 7, [30, 15], [8, 0]), (5, 512, 16, [19], [2])])
def test_gather_matches_the_cache(hkv, dim, page, lens, first, dtype):
    from iris_kernel.fused_kv import fused_int4_paged_gather

    rng = np.random.default_rng(hkv * dim)
    bt, pages = _table(rng, lens, page)
    cache = R.random_cache(rng, pages * page // 16 + 1, hkv, dim)
    cache = [np.ascontiguousarray(x.reshape(-1, *x.shape[2:])[:pages * page].reshape(pages, page, *x.shape[2:]))
             for x in cache]
    start = first or [0] * len(lens)
    counts = [n - f for n, f in zip(lens, start)]
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    dev = [torch.from_numpy(x).cuda() for x in (*cache, bt, cu)]
    wider = torch.full((len(lens), bt.shape[1] + 5), -9, dtype=torch.int32, device="cuda")
    wider[:, :bt.shape[1]] = dev[4]
    kw = dict(first_token=torch.tensor(first, dtype=torch.int32, device="cuda")) if first else {}
    want = _gather_expect(cache, bt, lens, start, dtype, page)
    for table in (dev[4], wider[:, :bt.shape[1]]):
        got = fused_int4_paged_gather(*dev[:4], table, dev[5], num_tokens=int(cu[-1]), dtype=dtype, page_size=page, **kw)
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            _same_bits(g, w)
    # rows past the last sequence are zeros; the outputs can be given
    rest = torch.full((int(cu[-1]) + 21, hkv, dim), 7.0, dtype=dtype, device="cuda")
    k, v = fused_int4_paged_gather(*dev[:4], dev[4], dev[5], rest, num_tokens=int(cu[-1]) + 21, dtype=dtype,
                                   page_size=page, **kw)
    assert k is rest and not k[int(cu[-1]):].any() and not v[int(cu[-1]):].any()
    _same_bits(k[:int(cu[-1])], want[0])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 8, 16])
def test_gather_into_rows_at_any_16_bytes(offset, dtype):
    """Outputs that start 0, 16 or 32 bytes into their memory: the narrow and the wide stores."""
    from iris_kernel.fused_kv import fused_int4_paged_gather

    rng = np.random.default_rng(7 + offset)
    lens, hkv, dim = [45, 0, 18], 3, 96
    bt, pages = _table(rng, lens, 16)
    cache = R.random_cache(rng, pages + 1, hkv, dim)
    cache = [np.ascontiguousarray(x[:pages]) for x in cache]
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    dev = [torch.from_numpy(x).cuda() for x in (*cache, bt, cu)]
    want = _gather_expect(cache, bt, lens, [0, 0, 0], dtype, 16)
    n = int(cu[-1]) * hkv * dim
    room = torch.full((2, n + 64), 5.0, dtype=dtype, device="cuda")
    key, value = (room[i, 32 * i + offset:32 * i + offset + n].view(-1, hkv, dim) for i in range(2))
    fused_int4_paged_gather(*dev[:4], dev[4], dev[5], key, value, num_tokens=int(cu[-1]))
    _same_bits(key, want[0])
    _same_bits(value, want[1])
    for i in range(2):  # and nothing around them
        assert bool((room[i, :32 * i + offset] == 5).all()) and bool((room[i, 32 * i + offset + n:] == 5).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gather_of_extreme_scales(dtype):
    """Every nibble with the smallest, the largest and the non-finite scales."""
    from iris_kernel.fused_kv import fused_int4_paged_gather

    values = np.array([0.0, 2.0 ** -24, 2.0 ** -14, 3.0 / 7, 9375.0, 65504.0, np.inf, np.nan, -0.5], np.float16)
    n = len(values)
    data = np.broadcast_to(R.pack(np.tile(np.arange(-8, 8, dtype=np.int8), 2)), (1, n, 1, 16)).copy()
    scale = values.reshape(1, n, 1, 1).copy()
    dev = [torch.from_numpy(x).cuda() for x in (data, data, scale, scale, np.zeros((1, 1), np.int32),
                                                 np.array([0, n], np.int32))]
    with np.errstate(invalid="ignore", over="ignore"):
        want = _gather_expect((data, data, scale, scale), np.zeros((1, 1), np.int32), [n], [0], dtype, n)
    for got, w in zip(fused_int4_paged_gather(*dev, num_tokens=n, dtype=dtype, page_size=n), want):
        _same_bits(got, w)


def test_gather_errors_and_refusals():
    from iris_kernel.fused_kv import fused_int4_paged_gather

    rng = np.random.default_rng(1)
    cache = [torch.from_numpy(x).cuda() for x in R.random_cache(rng, 4, 2, 64)]

    def call(bt, cu, n, **kw):
        out = fused_int4_paged_gather(*cache, torch.tensor(bt, dtype=torch.int32, device="cuda"),
                                      torch.tensor(cu, dtype=torch.int32, device="cuda"), num_tokens=n, **kw)
        torch.cuda.synchronize()
        return out

    call([[0, 3]], [0, 32], 32)
    with pytest.raises(IndexError):
        call([[0, 4]], [0, 32], 32)  # no such page
    with pytest.raises(IndexError):
        call([[-1, 0]], [0, 32], 32)
    with pytest.raises(ValueError):
        call([[0, 1]], [0, 33], 33)  # the table is too short
    with pytest.raises(ValueError):
        call([[0, 1], [2, 3]], [0, 20, 10], 20)  # offsets that fall
    with pytest.raises(ValueError):
        call([[0, 1]], [5, 20], 20)  # offsets that do not start at 0
    with pytest.raises(ValueError):
        call([[0, 1]], [0, 5], 5, first_token=torch.tensor([-1], dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError):
        call([[0, 1]], [0, 5], 5, dtype=torch.float32)
    with pytest.raises(ValueError):
        call([[0, 1]], [0, 5, 6], 5)
    with pytest.raises(ValueError):
        call([[0, 1]], [0, 5], -1)
    with pytest.raises(NotImplementedError):
        call([[0, 1]], [0, 5], 5, group_size=16)
    with pytest.raises(ValueError):
        call([[0, 1]], [0, 5], 5, page_size=8)
    assert call([[0, 1]], [0, 0], 0)[0].shape == (0, 2, 64)


def test_offsets_past_32_bits():
    """Pages more than 2^31 bytes into the cache are written and read."""
    from iris_kernel.fused_kv import fused_int4_paged_gather

    hkv, dim, pages = 16, 128, 140_000  # 16 KB of keys a page: 2.3 GB
    c = _case(20, T=9, hq=1, hkv=hkv, dim=dim, pages=9, pad=0.0)
    want, _, key = _expect(c)
    big = [torch.zeros((pages, *x.shape[1:]), dtype=x.dtype, device="cuda") for x in c["cache"]]
    for x, small in zip(big, c["cache"]):
        x[-9:] = small
    c["cache"] = big
    c["slots"] = c["slots"] + (pages - 9) * 16
    _run(c)
    for got, w in zip(big, want):
        _same_bits(got[-9:], w)
    bt = torch.tensor([[pages - 1, pages - 9]], dtype=torch.int32, device="cuda")
    k, v = fused_int4_paged_gather(*big, bt, torch.tensor([0, 32], dtype=torch.int32, device="cuda"), num_tokens=32)
    ref = np.concatenate([R.dequant(want[0][8], want[2][8]), R.dequant(want[0][0], want[2][0])])
    _same_bits(k, R.to_type(ref, torch.float16))


def test_gather_outputs_that_overlap_are_refused():
    from iris_kernel.fused_kv import fused_int4_paged_gather

    rng = np.random.default_rng(8)
    cache = [torch.from_numpy(x).cuda() for x in R.random_cache(rng, 4, 2, 64)]
    bt, cu = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[0, 3]], [0, 20]))
    room = torch.zeros(3 * 20 * 128, dtype=torch.float16, device="cuda")
    at = [room[i * 1280:i * 1280 + 2560].view(20, 2, 64) for i in range(3)]
    for key, value in ((at[0], at[0]), (at[0], at[1]), (at[1], at[0])):
        with pytest.raises(ValueError, match="overlap"):
            fused_int4_paged_gather(*cache, bt, cu, key, value, num_tokens=20)
    inside = cache[0].view(-1).view(torch.float16)[:1280].view(10, 2, 64)  # the cache's own bytes
    with pytest.raises(ValueError, match="overlap"):
        fused_int4_paged_gather(*cache, bt, cu, inside, num_tokens=10)
    with pytest.raises(ValueError, match="overlap"):
        fused_int4_paged_gather(*cache, bt, cu, None, inside, num_tokens=10)
    key, value = fused_int4_paged_gather(*cache, bt, cu, at[0], at[2], num_tokens=20)
    for got, want in zip((key, value), fused_int4_paged_gather(*cache, bt, cu, num_tokens=20)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("cu", [[-5, 10], [-5, 0, 10], [-8, -5, 10], [1, 1, 10], [0, 8, 3, 10], [0, 3, -2, 10],
                                [0] * 400 + [9, 8, 10]])
def test_gather_offsets_that_do_not_rise_from_0(cu):
    from iris_kernel.fused_kv import fused_int4_paged_gather

    rng = np.random.default_rng(9)
    cache = [torch.from_numpy(x).cuda() for x in R.random_cache(rng, 4, 2, 64)]
    bt = torch.tensor([[0, 3]], dtype=torch.int32, device="cuda").expand(len(cu) - 1, 2)
    with pytest.raises(ValueError):
        fused_int4_paged_gather(*cache, bt, torch.tensor(cu, dtype=torch.int32, device="cuda"), num_tokens=10)
    cu = [0] + sorted(abs(x) for x in cu[1:])
    fused_int4_paged_gather(*cache, bt, torch.tensor(cu, dtype=torch.int32, device="cuda"), num_tokens=10)


def test_gather_names_its_own_arguments():
    from iris_kernel.fused_kv import fused_int4_paged_gather

    rng = np.random.default_rng(10)
    cache = [torch.from_numpy(x).cuda() for x in R.random_cache(rng, 4, 2, 64)]
    bt, cu, first = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[0, 3]], [0, 10], [-1]))
    with pytest.raises(ValueError, match="first_token"):
        fused_int4_paged_gather(*cache, bt, cu, num_tokens=10, first_token=first)
    with pytest.raises(ValueError, match="cu_seqlens"):
        fused_int4_paged_gather(*cache, bt, cu + 2, num_tokens=12)
