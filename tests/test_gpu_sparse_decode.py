"""Page bounds and page selection, bit for bit against their definition, and
the attention over selected pages against 64 bits.

Tolerance of the attention, per output: half a unit in the last place of the
output's type (2^-11 or 2^-8 of the value), and 2^-14 of the largest value in
the page list: p * scale is held in two 16-bit terms (2^-18 or better), and a logit of up to
128 products, summed in fp32 with at most 2^-22 of the running sum lost an
addition and sums below 16, is off by less than 2^-15, which moves p and the
normaliser by 2^-15.5 each.  The lse, a logit plus a logarithm, by 2^-14."""
import numpy as np
import pytest
import torch

import _sparse_refs as R

pytestmark = pytest.mark.gpu

I32 = torch.int32


def _dev(*xs):
    out = [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in xs]
    return out if len(out) > 1 else out[0]


def _table(rng, lens, width=None, spare=2):
    counts = [-(-n // 16) for n in lens]
    ids = rng.permutation(sum(counts) + spare).astype(np.int32)
    bt = np.full((len(lens), width or max(1, max(counts))), -3, np.int32)  # columns past the end are never read
    at = 0
    for b, n in enumerate(counts):
        bt[b, :n] = ids[at:at + n]
        at += n
    return bt, sum(counts) + spare


# -------------------------------------------------------------------- bounds
def _bounds(kd, ks, bt, lens, bounds, step, **kw):
    from iris_kernel.sparse_attention import fused_int4_page_bounds

    fused_int4_page_bounds(kd, ks, bt, lens, bounds, step, **kw)
    torch.cuda.synchronize()


@pytest.mark.parametrize("hkv,dim", [(1, 64), (3, 64), (2, 128), (8, 128), (17, 128)])
@pytest.mark.parametrize("lens,first", [([1], None), ([37, 0, 16, 17, 300], None), ([37, 0, 16, 17, 300], [30, 0, 16, 16, 5]),
                                        ([500], [499])])
def test_bounds_match_the_definition(hkv, dim, lens, first):
    rng = np.random.default_rng(hkv * dim + len(lens))
    bt, pages = _table(rng, lens)
    kd, _, ks, _ = R.random_cache(rng, pages, hkv, dim)
    kd[bt[0, 0], :, 0] = 0  # a page of zero keys in head 0
    ks[rng.random(ks.shape) < 0.05] = np.float16(2.0 ** -14)
    bounds = rng.integers(-127, 128, (pages, hkv, 2, dim)).astype(np.int8)
    step = rng.random((pages, hkv)).astype(np.float32)
    values = np.full(bounds.shape, 3.0, np.float16)
    dev = _dev(kd, ks, bt, np.array(lens, np.int32), bounds, step)
    val = _dev(values)
    fd = None if first is None else torch.tensor(first, dtype=I32, device="cuda")
    _bounds(*dev, first_token=fd, values=val)
    was = bounds.copy()
    R.bounds_ref(kd, ks, bt, lens, first, bounds, step)
    assert np.array_equal(dev[4].cpu().numpy(), bounds)
    assert np.array_equal(dev[5].cpu().numpy(), step)
    # the values of the pages that were computed, and only those
    touched = {int(bt[b, c]) for b, n in enumerate(lens) for c in range((first[b] if first else 0) // 16, -(-n // 16))}
    for page in range(pages):
        want = (bounds[page].astype(np.float32) * step[page][:, None, None]).astype(np.float16)
        if page not in touched:
            assert np.array_equal(bounds[page], was[page])
            want = values[page]
        assert np.array_equal(val[page].cpu().numpy(), want)


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_bounds_of_scales_that_are_not_finite(bad):
    """Such a scale opens its head's bounds of its page; one past the end of the
    sequence changes nothing."""
    rng = np.random.default_rng(3)
    bt, pages = _table(rng, [40])
    kd, _, ks, _ = R.random_cache(rng, pages, 4, 128)
    ks[bt[0, 1], 5, 2, 3] = bad
    ks[bt[0, 2], 8:] = bad  # tokens 40 .. 47
    bounds, step = np.zeros((pages, 4, 2, 128), np.int8), np.zeros((pages, 4), np.float32)
    dev = _dev(kd, ks, bt, np.array([40], np.int32), bounds, step)
    _bounds(*dev)
    R.bounds_ref(kd, ks, bt, [40], None, bounds, step)
    assert np.isinf(step[bt[0, 1], 2]) and np.isfinite(step).sum() == step.size - 1
    assert np.array_equal(dev[4].cpu().numpy(), bounds) and np.array_equal(dev[5].cpu().numpy(), step)


def test_bounds_hold_every_key():
    rng = np.random.default_rng(4)
    bt, pages = _table(rng, [333])
    kd, _, ks, _ = R.random_cache(rng, pages, 2, 64)
    dev = _dev(kd, ks, bt, np.array([333], np.int32), np.zeros((pages, 2, 2, 64), np.int8),
               np.zeros((pages, 2), np.float32))
    _bounds(*dev)
    bounds, step = dev[4].cpu().numpy().astype(np.float64), dev[5].cpu().numpy().astype(np.float64)
    for col in range(21):
        page, tok = bt[0, col], min(16, 333 - 16 * col)
        key = R.dequant(kd[page, :tok], ks[page, :tok], np.float64)
        unit = step[page][:, None] * (1 + 2.0 ** -22)  # the step itself is rounded
        assert (bounds[page, :, 0] * unit <= key.min(0) + 1e-12).all()
        assert (bounds[page, :, 1] * unit >= key.max(0) - 1e-12).all()


def test_bounds_errors_and_refusals():
    rng = np.random.default_rng(5)
    kd, _, ks, _ = R.random_cache(rng, 4, 2, 64)
    base = dict(kd=kd, ks=ks, bt=np.array([[0, 1]], np.int32), lens=np.array([20], np.int32),
                bounds=np.zeros((4, 2, 2, 64), np.int8), step=np.zeros((4, 2), np.float32))

    def call(error, **change):
        dev = _dev(*{**base, **change}.values())
        if error is None:
            return _bounds(*dev)
        with pytest.raises(error):
            _bounds(*dev)

    call(None)
    call(None, lens=np.array([0], np.int32))
    call(IndexError, bt=np.array([[0, 4]], np.int32))
    call(IndexError, bt=np.array([[-1, 0]], np.int32))
    call(ValueError, lens=np.array([33], np.int32))
    call(ValueError, lens=np.array([-1], np.int32))
    call(TypeError, lens=np.array([20], np.int64))
    call(TypeError, bounds=np.zeros((4, 2, 2, 64), np.int16))
    call(ValueError, bounds=np.zeros((4, 2, 2, 32), np.int8))
    call(ValueError, step=np.zeros((4, 3), np.float32))
    call(ValueError, bt=np.array([[0, 1], [2, 3]], np.int32))
    call(NotImplementedError, kd=kd[..., :16].copy())
    call(None)


# ----------------------------------------------------------------- selection
def _select(query, bounds, step, bt, lens, **kw):
    from iris_kernel.sparse_attention import fused_page_select

    out = fused_page_select(query, bounds, step, bt, lens, **kw)
    torch.cuda.synchronize()
    return [x.cpu().numpy() for x in out]


def _check_select(seed, hq, hkv, dim, lens, keep, sink=1, recent=1, dtype=torch.float16, width=None, pages=None,
                  spread=127, change=None):
    rng = np.random.default_rng(seed)
    if pages is None:
        bt, pages = _table(rng, lens, width)
    else:  # few physical pages under a long table: many equal scores
        bt = rng.integers(0, pages, (len(lens), width)).astype(np.int32)
    bounds = np.sort(rng.integers(-spread, spread + 1, (pages, hkv, 2, dim)), axis=2).astype(np.int8)
    step = (0.01 + 0.02 * rng.random((pages, hkv))).astype(np.float32)
    query = R.to_type(rng.standard_normal((len(lens), hq, dim)), dtype)
    if change:
        change(query, bounds, step, bt)
    lists, counts = _select(query.cuda(), *_dev(bounds, step, bt, np.array(lens, np.int32)), max_pages=keep,
                            sink_pages=sink, recent_pages=recent)
    scores = R.scores_ref(R.f32(query), bounds, step, np.maximum(bt, 0), hkv)
    want, n = R.select_ref(scores, lens, keep, sink, recent)
    assert np.array_equal(counts, n)
    assert np.array_equal(lists, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,dim", [(1, 1, 64), (4, 4, 128), (6, 2, 64), (32, 4, 128), (9, 1, 128), (32, 2, 64)])
def test_selection_matches_the_definition(hq, hkv, dim, dtype):
    _check_select(hq, hq, hkv, dim, [777, 1, 0, 160, 161, 2000], 10, dtype=dtype)


@pytest.mark.parametrize("keep,sink,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (2, 1, 1), (7, 3, 4), (7, 0, 0), (64, 2, 9),
                                              (125, 1, 1), (126, 1, 1), (400, 1, 1)])
def test_budgets_and_kept_ends(keep, sink, recent):
    _check_select(keep, 8, 2, 64, [2000, 1999, 16, 1984], keep, sink, recent)


@pytest.mark.parametrize("width", [2048, 2049, 8193, 33000])
def test_long_tables_with_many_equal_scores(width):
    """Each key layout of the selection, three physical pages: ties go to the
    lowest page."""
    _check_select(width, 2, 2, 64, [16 * width - 3, 16 * width], 300, width=width, pages=3)
    _check_select(width, 2, 2, 64, [16 * width - 3], 300, width=width, pages=4000)


@pytest.mark.parametrize("pages", [200, 500, 1000, 2000, 8000, 33000])
def test_scores_of_all_sizes_and_scores_that_differ_in_their_last_bits(pages):
    """Each key layout: half of the scores lie within 40 units in the last
    place, the others are spread over 2^120, and the budget ends among the
    former."""
    def change(query, bounds, step, bt):
        rng = np.random.default_rng(pages)
        bounds[:] = bounds[0]
        near = rng.permutation(len(step))[:len(step) // 2]
        step[:] = np.exp2(rng.uniform(-60, 60, step.shape)).astype(np.float32)
        step[near] = (1 + rng.integers(0, 40, (len(near), step.shape[1])) * 2.0 ** -23).astype(np.float32)

    _check_select(pages, 2, 2, 64, [16 * pages - 5], pages // 4 + 7 * (pages // 16), change=change)


@pytest.mark.parametrize("pages", [200, 500, 1000, 2000, 8000, 20000, 33000])
@pytest.mark.parametrize("top", ["ordinary", "infinite"])
def test_scores_that_overflow(pages, top):
    """Each key layout: most scores are minus infinity (a finite step times a
    negative sum), some lie just above it, a few are ordinary or plus infinity;
    the budget ends among each of them, and where one kind ends."""
    n, few = pages, 3 + pages // 100
    near = pages // 10

    def change(query, bounds, step, bt):
        rng = np.random.default_rng(pages)
        query[:] = query.abs().clamp(min=0.5)
        kind = rng.permutation(n)
        low, high = bt[0, kind[few + near:]], bt[0, kind[:few]]
        bounds[:] = -100  # of a positive query: a negative sum
        step[:] = (4e32 * (1 - rng.random(step.shape) / 64)).astype(np.float32)  # sums below 8.2e5: finite
        step[low] = 3e38
        bounds[high] = 100
        step[high] = np.inf if top == "infinite" else 0.25

    for keep in (2 + few // 2, 2 + few, 2 + few + near // 2, few + near, 2 + few + near, few + near + (n - few - near) // 2,
                 n - 1):
        _check_select(pages, 2, 2, 64, [16 * n - 5], keep, change=change)


def test_all_scores_equal_or_zero():
    _check_select(1, 4, 2, 64, [1600], 9, spread=0)  # every bound 0

    def zero(query, bounds, step, bt):
        query[:] = 0

    _check_select(2, 4, 2, 64, [1600], 9, change=zero)


def test_values_that_are_not_finite():
    """A page with an infinite step comes first; a query head that is not
    finite has no say."""
    def change(query, bounds, step, bt):
        step[bt[0, 50:53]] = np.inf
        step[bt[0, 60], 1] = np.nan
        query[0, 0, 3] = float("nan")
        query[0, 2, 5] = float("inf")
        query[0, 3, 5] = -float("inf")

    _check_select(3, 4, 2, 64, [1600], 9, change=change)

    def many(query, bounds, step, bt):
        step[:] = np.inf  # more such pages than there is room for: the lowest, and the kept ends

    _check_select(4, 4, 2, 64, [1600], 9, sink=2, recent=3, change=many)


def test_selection_errors_and_refusals():
    from iris_kernel.sparse_attention import fused_page_select

    rng = np.random.default_rng(6)
    bt, pages = _table(rng, [400])
    good = dict(query=torch.randn(1, 4, 64, device="cuda").half(),
                bounds=torch.zeros(pages, 2, 2, 64, dtype=torch.int8, device="cuda"),
                step=torch.ones(pages, 2, device="cuda"), bt=_dev(bt), lens=torch.tensor([400], dtype=I32, device="cuda"))

    def call(error, max_pages=4, kw=None, **change):
        a = {**good, **change}
        with pytest.raises(error):
            fused_page_select(*a.values(), max_pages=max_pages, **(kw or {}))

    call(ValueError, lens=torch.tensor([401], dtype=I32, device="cuda"))  # the table is too short
    call(ValueError, lens=torch.tensor([-1], dtype=I32, device="cuda"))
    call(IndexError, bt=_dev(np.where(bt == bt[0, 3], pages, bt).astype(np.int32)))
    call(ValueError, max_pages=0)
    call(ValueError, max_pages=1)  # one page at each end
    call(ValueError, kw=dict(sink_pages=-1))
    call(TypeError, query=good["query"].float())
    call(ValueError, query=good["query"][:, :3])
    call(ValueError, query=torch.randn(1, 4, 128, device="cuda").half())
    call(NotImplementedError, query=torch.randn(1, 34, 64, device="cuda").half())
    call(TypeError, step=good["step"].half())
    call(TypeError, lens=good["lens"].long())
    call(ValueError, lens=torch.tensor([1, 1], dtype=I32, device="cuda"))
    call(NotImplementedError, kw=dict(page_size=32))
    fused_page_select(*good.values(), max_pages=4)
    empty = fused_page_select(good["query"][:0], good["bounds"], good["step"], good["bt"][:0], good["lens"][:0],
                              max_pages=4)
    assert empty[0].shape == (0, 2, 4)


# ----------------------------------------------------------------- attention
def _attend(args, **kw):
    from iris_kernel.sparse_attention import fused_int4_sparse_paged_decode_attention

    out = fused_int4_sparse_paged_decode_attention(*args, return_lse=True, **kw)
    torch.cuda.synchronize()
    return out


def _case(seed, hq, hkv, dim, lens, keep, dtype=torch.float16, width=None):
    """Random lists: distinct pages, the last one mostly among them."""
    rng = np.random.default_rng(seed)
    bt, pages = _table(rng, lens, width)
    cache = R.random_cache(rng, pages, hkv, dim)
    lists = np.full((len(lens), hkv, keep), -1, np.int32)
    counts = np.zeros((len(lens), hkv), np.int32)
    for b, n in enumerate(lens):
        total = -(-n // 16)
        for h in range(hkv):
            got = rng.permutation(total)[:min(total, keep)]
            if len(got) and h % 2 == 0:
                got[0] = total - 1 if total - 1 not in got else got[0]
            lists[b, h, :len(got)] = np.sort(got)
            counts[b, h] = len(got)
    query = R.to_type(rng.standard_normal((len(lens), hq, dim)), dtype)
    return dict(query=query, cache=list(cache), bt=bt, lens=np.array(lens, np.int32), lists=lists, counts=counts)


def _check_attend(c, scale=None, **kw):
    args = [c["query"].cuda(), *_dev(*c["cache"], c["bt"], c["lens"], c["lists"], c["counts"])]
    out, lse = _attend(args, softmax_scale=scale, **kw)
    want, want_lse = R.attend_ref(R.f32(c["query"]), *c["cache"], np.maximum(c["bt"], 0), c["lens"], c["lists"],
                                  c["counts"], scale)
    half_ulp = 2.0 ** (-11 if c["query"].dtype == torch.float16 else -8)
    biggest = 7 * float(np.nanmax(np.where(np.isfinite(c["cache"][3]), c["cache"][3], 0).astype(np.float64)))
    got = out.double().cpu().numpy()
    assert out.dtype == c["query"].dtype and np.isfinite(got).all()
    assert (np.abs(got - want) <= half_ulp * np.abs(want) + 2.0 ** -14 * biggest).all()
    empty = np.isneginf(want_lse)
    got_lse = lse.double().cpu().numpy()
    assert np.array_equal(np.isneginf(got_lse), empty)
    assert (np.abs(got_lse[~empty] - want_lse[~empty]) <= 2.0 ** -14).all()
    assert not got[empty].any()
    return args, out, lse


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (8, 2), (24, 3), (9, 1), (32, 2)])
def test_attention_matches_64_bits(hq, hkv, dim, dtype):
    _check_attend(_case(hq + dim, hq, hkv, dim, [1, 15, 16, 17, 0, 333, 1000], 13, dtype))


@pytest.mark.parametrize("keep", [1, 2, 4, 5, 31, 33, 64, 129, 300])
def test_list_lengths(keep):
    """Fewer pages than warps, every cluster size, several look-ups a warp."""
    _check_attend(_case(keep, 8, 1, 128, [5000], keep))
    _check_attend(_case(keep, 16, 1, 64, [5000, 77], keep))


@pytest.mark.parametrize("batch", [1, 30, 60, 120, 300])
def test_cluster_sizes(batch):
    _check_attend(_case(batch, 4, 2, 64, [200 + 7 * i for i in range(batch)], 12))


def test_lists_with_holes_repeats_and_pages_past_the_end():
    c = _case(11, 8, 2, 128, [100, 40], 12)
    c["lists"][0, 0] = [-1, 3, -1, 99, 6, 6, 0, -5, 2, 7, 1, 1]
    c["counts"][0, 0] = 10  # the last two do not count
    c["lists"][0, 1] = -1
    c["counts"][0, 1] = 12  # nothing but holes
    c["counts"][1, 0] = 0
    c["counts"][1, 1] = 99  # more than there is room for
    _check_attend(c)


def test_bytes_past_the_end_do_not_matter():
    """Tokens after the last one hold NaN and infinite scales and full nibbles."""
    c = _case(12, 8, 2, 128, [37, 1, 130], 9)
    for b, n in enumerate(c["lens"]):
        page = c["bt"][b, (n - 1) // 16]
        for x in c["cache"][:2]:
            x[page, n % 16:] = 0x77
        c["cache"][2][page, n % 16:] = np.nan
        c["cache"][3][page, n % 16:] = np.inf
        for h in range(2):
            c["lists"][b, h, 0] = (n - 1) // 16
            c["lists"][b, h, 1:] = -1
            c["counts"][b, h] = 1
    _check_attend(c)


@pytest.mark.parametrize("scale", [0.01, 1.0, 20.0])
def test_softmax_scales(scale):
    """Also logits in the hundreds: one token holds almost all the weight, and
    the logits' own error grows with them (tolerances at the default scale are
    compared at scale <= 1; at 20 only that the result is that token's value)."""
    c = _case(13, 4, 1, 128, [600], 30)
    if scale <= 1.0:
        c["query"] = (c["query"].float() * 0.08 / max(scale, 0.08)).half()
        _check_attend(c, scale)
        return
    args = [c["query"].cuda(), *_dev(*c["cache"], c["bt"], c["lens"], c["lists"], c["counts"])]
    out, _ = _attend(args, softmax_scale=scale)
    want, _ = R.attend_ref(R.f32(c["query"]), *c["cache"], c["bt"], c["lens"], c["lists"], c["counts"], scale)
    assert (np.abs(out.double().cpu().numpy() - want) <= 2.0 ** -9 * np.abs(want) + 2.0 ** -9).all()


def test_values_that_are_not_finite_show():
    """A NaN key scale reaches the outputs of its head and no others'."""
    c = _case(14, 4, 2, 64, [64], 4)
    c["cache"][2][c["bt"][0, 1], 3, 1] = np.nan
    c["lists"][0] = [0, 1, 2, 3]
    c["counts"][:] = 4
    args = [c["query"].cuda(), *_dev(*c["cache"], c["bt"], c["lens"], c["lists"], c["counts"])]
    out, lse = _attend(args)
    assert torch.isfinite(out[0, :2]).all() and torch.isfinite(lse[0, :2]).all()
    assert torch.isnan(out[0, 2:]).all() and torch.isnan(lse[0, 2:]).all()


def test_all_pages_equal_the_dense_decode():
    """With every page listed, the dense decode's output (within its own
    tolerance, max-abs 2e-3 / relative 1e-2)."""
    from iris_kernel.fused_attention import fused_int4_paged_decode_attention

    c = _case(15, 32, 8, 128, [513, 1, 160], 40)
    args, out, _ = _check_attend(c)
    args[5] = args[5].clamp(min=0)
    dense = fused_int4_paged_decode_attention(*args[:7]).float()
    assert ((out.float() - dense).abs() <= 2e-3 + 1e-2 * dense.abs()).all()


def test_two_runs_and_a_side_stream_give_the_same_bits():
    c = _case(16, 16, 2, 128, [2000, 900], 50)
    args, out, lse = _check_attend(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again, lse2 = _attend(args)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    given = torch.full_like(out, 5.0)
    assert _attend(args[:9], output=given)[0] is given and torch.equal(out, given)


def test_pages_past_32_bits():
    """Pages more than 2^31 bytes into the cache."""
    c = _case(17, 16, 16, 128, [90], 6)
    pages = 140_000  # 16 KB of keys a page
    big = []
    for x in c["cache"]:
        y = torch.zeros((pages, *x.shape[1:]), dtype=torch.from_numpy(x).dtype, device="cuda")
        y[-x.shape[0]:] = torch.from_numpy(x).cuda()
        big.append(y)
    shift = pages - c["cache"][0].shape[0]
    args, out, lse = _check_attend(c)
    far = [args[0], *big, args[5] + shift, *args[6:]]
    out2, lse2 = _attend(far)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    # and their bounds
    rows = c["cache"][0].shape[0]
    near_b = _dev(np.zeros((rows, 16, 2, 128), np.int8), np.zeros((rows, 16), np.float32))
    _bounds(args[1], args[3], args[5], args[6], *near_b)
    far_b = [torch.zeros((pages, 16, 2, 128), dtype=torch.int8, device="cuda"), torch.zeros((pages, 16), device="cuda")]
    _bounds(big[0], big[2], args[5] + shift, args[6], *far_b)
    assert torch.equal(far_b[0][-rows:], near_b[0]) and torch.equal(far_b[1][-rows:], near_b[1])
    got = _select(args[0], *far_b, args[5] + shift, args[6], max_pages=3)
    want = _select(args[0], *near_b, args[5], args[6], max_pages=3)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_attention_errors_and_refusals():
    c = _case(18, 4, 2, 64, [100], 5)
    good = [c["query"].cuda(), *_dev(*c["cache"], c["bt"], c["lens"], c["lists"], c["counts"])]
    names = ["query", "kd", "vd", "ks", "vs", "bt", "lens", "lists", "counts"]

    def call(error, kw=None, **change):
        args = [change.get(n, x) for n, x in zip(names, good)]
        with pytest.raises(error):
            _attend(args, **(kw or {}))

    call(IndexError, bt=torch.full_like(good[5], 1 << 20))
    call(IndexError, bt=torch.full_like(good[5], -1))
    call(ValueError, bt=good[5][:, :1].contiguous(), lists=torch.full_like(good[7], 6))  # the table is too short
    call(ValueError, lens=torch.tensor([-1], dtype=I32, device="cuda"))
    call(TypeError, query=good[0].float())
    call(TypeError, kd=good[1].to(torch.int8))
    call(TypeError, ks=good[3].float())
    call(TypeError, lists=good[7].long())
    call(ValueError, counts=good[8][:, :1])
    call(ValueError, lists=good[7][:, :, :0])
    call(ValueError, lists=good[7][:, :1])
    call(ValueError, query=good[0][:, :3])
    call(ValueError, query=good[0].transpose(1, 2).contiguous().transpose(1, 2))
    call(ValueError, vd=good[2][:1])
    call(ValueError, query=good[0].cpu())
    call(NotImplementedError, query=torch.zeros(1, 34, 64, device="cuda").half())
    call(NotImplementedError, kw=dict(group_size=64))
    call(NotImplementedError, kw=dict(page_size=32))
    call(ValueError, kw=dict(output=torch.empty(1, 4, 128, dtype=torch.float16, device="cuda")))
    call(RuntimeError, kw=dict(softmax_scale=-1.0))
    _attend(good)
    none = _attend([good[0][:0], *good[1:5], good[5][:0], good[6][:0], good[7][:0], good[8][:0]])
    assert none[0].shape == (0, 4, 64) and none[1].shape == (0, 4)


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_key_group_that_is_not_finite_always_shows(dim, bad):
    """Its nibbles are zeros, as the append leaves them: the key is NaN, and so
    is every output of its head, whatever the query; other heads do not change."""
    lens = [200 + i for i in range(24)]
    c = _case(24, 8, 2, dim, lens, 14)
    rng = np.random.default_rng(24)
    total = [-(-n // 16) for n in lens]
    for b in range(24):
        c["lists"][b] = -1
        c["lists"][b, :, :total[b]] = np.arange(total[b])
        c["counts"][b] = total[b]
        page, tok, k = c["bt"][b, rng.integers(0, total[b] - 1)], rng.integers(0, 16), rng.integers(0, dim // 32)
        c["cache"][2][page, tok, 1, k] = bad
        c["cache"][0][page, tok, 1, 16 * k:16 * k + 16] = 0
    args = [c["query"].cuda(), *_dev(*c["cache"], c["bt"], c["lens"], c["lists"], c["counts"])]
    out, lse = _attend(args)
    assert torch.isnan(out[:, 4:]).all() and torch.isnan(lse[:, 4:]).all()
    assert torch.isfinite(out[:, :4]).all() and torch.isfinite(lse[:, :4]).all()


def _close(c, scale=None):
    """The attention against 64 bits, every output on its own: half a unit in
    the last place (FP16: or 2^-25) and 2^-14 of the sum of the magnitudes that
    are added up for it (the errors of p and the normaliser, as above)."""
    args = [c["query"].cuda(), *_dev(*c["cache"], c["bt"], c["lens"], c["lists"], c["counts"])]
    out, lse = _attend(args, softmax_scale=scale)
    rest = (c["bt"], c["lens"], c["lists"], c["counts"], scale)
    kd, vd, ks, vs = c["cache"]
    want, want_lse = R.attend_ref(R.f32(c["query"]), kd, vd, ks, vs, *rest)
    magnitude, _ = R.attend_ref(R.f32(c["query"]), kd, R.pack(np.abs(R.unpack(vd))), ks, vs, *rest)
    half = c["query"].dtype == torch.float16
    rounding = np.maximum(2.0 ** -11 * np.abs(want), 2.0 ** -25) if half else 2.0 ** -8 * np.abs(want)
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= rounding + 2.0 ** -14 * magnitude).all()
    assert (np.abs(got_lse - want_lse) <= 2.0 ** -14).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
def test_small_elements_of_a_query_with_a_large_one(dim, dtype):
    """The largest element meets zero keys; the logits are the odd dims', 2^-14
    (BF16: 2^-18) of it, in the other groups."""
    c = _case(22, 4, 2, dim, [700], 20, dtype)
    small = 2.0 ** (-4 if dtype == torch.float16 else -8)
    rng = np.random.default_rng(22)
    query = np.zeros((1, 4, dim), np.float32)
    query[..., 33::2] = small * rng.uniform(1, 2, query[..., 33::2].shape) * rng.choice([-1, 1], query[..., 33::2].shape)
    query[..., 0] = 1024
    c["query"] = R.to_type(query, dtype)
    keys = R.unpack(c["cache"][0])
    keys[..., :32] = 0
    c["cache"][0] = R.pack(keys)
    _close(c, 1.5 / (small * 3 * 0.28 * 1.5 * (dim // 2 - 16) ** 0.5))


@pytest.mark.parametrize("exponent", [-130, -120, 100, 108, 116])
def test_queries_near_the_ends_of_bf16(exponent):
    """Logits too small to tell the tokens apart give their mean; logits far
    beyond an exponential's range give the one largest's value."""
    c = _case(23, 6, 2, 128, [300, 40], 19, torch.bfloat16)
    c["query"] = (c["query"].double() * 2.0 ** exponent).to(torch.bfloat16)
    args = [c["query"].cuda(), *_dev(*c["cache"], c["bt"], c["lens"], c["lists"], c["counts"])]
    out, lse = _attend(args)
    want, want_lse = R.attend_ref(c["query"].double().numpy(), *c["cache"], np.maximum(c["bt"], 0), c["lens"],
                                  c["lists"], c["counts"])
    got = out.double().cpu().numpy()
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -14 * 7 * float(c["cache"][3].max())).all()
    assert (np.abs(lse.double().cpu().numpy() - want_lse) <= 2.0 ** -14 + 2.0 ** -18 * np.abs(want_lse)).all()


SIZES = {
    "one small group": lambda t, k, n: 5e-4 if k == 1 else 0.28,
    "all small": lambda t, k, n: 5e-4,
    "the smallest": lambda t, k, n: 2.0 ** -14,
    "smallest beside largest": lambda t, k, n: 9000.0 if k == 0 else 2.0 ** -14,
    "rising": lambda t, k, n: 2.0 ** (-14 + 24 * t / n),
    "falling": lambda t, k, n: 2.0 ** (10 - 24 * t / n),
    "small first token": lambda t, k, n: np.where(t == 0, 2.0 ** -12, 2.0 ** -2),
}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,dim", [(2, 2, 64), (4, 1, 128), (8, 1, 128), (16, 1, 64), (12, 1, 128)])
@pytest.mark.parametrize("sizes", SIZES)
def test_small_values_are_as_exact_as_large_ones(sizes, hq, hkv, dim, dtype):
    """One token holds a quarter of the weight or more, 2047 others about 2^-11 of
    its weight each; the values' group scales are small in all groups, in some,
    or change along the sequence."""
    n = 2048
    c = _case(21, hq, hkv, dim, [n], n // 16, dtype)
    query = R.f32(c["query"]).reshape(1, hkv, hq // hkv, dim)
    query[:] = query[:, :, :1] * (1 + np.arange(hq // hkv)[:, None] / 64)  # one direction a KV head
    c["query"] = R.to_type(query.reshape(1, hq, dim), dtype)
    kd, _, ks, vs = c["cache"]
    at = c["bt"][0, 0]
    kd[at, 0] = R.pack((3 * np.sign(query[0, :, 0])).astype(np.int8))
    ks[at, 0] = 0.28 * (1.0 if dim == 128 else 2.0 ** 0.5)
    for page, col in zip(c["bt"][0], range(n // 16)):
        for k in range(dim // 32):
            vs[page, :, :, k] = np.broadcast_to(SIZES[sizes](16 * col + np.arange(16), k, n), 16).astype(np.float16)[:, None]
    _close(c)


def test_outputs_that_overlap_are_refused():
    """An output over part of the query or in the cache's memory, a list in the
    counts' place; the output in the query's own place is the output."""
    from iris_kernel.sparse_attention import fused_page_select

    c = _case(25, 8, 2, 128, [100, 333], 9)
    args, out, lse = _check_attend(c)
    room = torch.zeros(3 * out.numel(), dtype=out.dtype, device="cuda")
    args[0] = room[:out.numel()].view(out.shape).copy_(args[0])
    for at in (out.numel() // 2, 8):
        with pytest.raises(ValueError, match="overlap"):
            _attend(args, output=room[at:at + out.numel()].view(out.shape))
    with pytest.raises(ValueError, match="overlap"):
        _attend(args, output=args[3].view(-1)[:out.numel()].view(out.shape))
    own, lse2 = _attend(args, output=args[0])
    assert own is args[0] and torch.equal(own, out) and torch.equal(lse, lse2)

    ints = torch.zeros(64, dtype=I32, device="cuda")
    index = _dev(np.zeros((c["bt"].max() + 1, 2, 2, 128), np.int8), np.ones((c["bt"].max() + 1, 2), np.float32))
    for lists, counts in ((ints[:16], ints[:4]), (ints[:16], ints[12:16])):
        with pytest.raises(ValueError, match="overlap"):
            fused_page_select(out, *index, args[5], args[6], lists.view(2, 2, 4), counts.view(2, 2), max_pages=4)
    fused_page_select(out, *index, args[5], args[6], ints[:16].view(2, 2, 4), ints[16:20].view(2, 2), max_pages=4)


def test_a_negative_length_says_so():
    """These operators take a length of 0: the message is not the dense decode's."""
    from iris_kernel.sparse_attention import fused_page_select

    c = _case(26, 4, 2, 64, [100], 5)
    args = [c["query"].cuda(), *_dev(*c["cache"], c["bt"], c["lens"], c["lists"], c["counts"])]
    pages = args[1].shape[0]
    index = _dev(np.zeros((pages, 2, 2, 64), np.int8), np.zeros((pages, 2), np.float32))
    lens = torch.tensor([-1], dtype=I32, device="cuda")
    with pytest.raises(ValueError, match="negative"):
        _bounds(args[1], args[3], args[5], lens, *index)
    with pytest.raises(ValueError, match="negative"):
        fused_page_select(args[0], *index, args[5], lens, max_pages=4)
    with pytest.raises(ValueError, match="negative"):
        _attend([*args[:6], lens, *args[7:]])


@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("hq,dim", [(2, 64), (8, 128), (16, 128), (32, 64)])
def test_a_value_group_that_is_not_finite_shows_in_its_dims(hq, dim, bad):
    """NaN in the 32 dims of that head's outputs, and nowhere else; the other
    dims, of ordinary scales and of scales of 2 and more, are what they are
    without it."""
    for large in (1.0, 40.0):
        c = _case(27, hq, 2, dim, [300, 90], 19)
        c["cache"][3] = (c["cache"][3].astype(np.float32) * large).astype(np.float16)
        for b in range(2):
            total = -(-int(c["lens"][b]) // 16)
            c["lists"][b] = -1
            c["lists"][b, :, :total] = np.arange(total)
            c["counts"][b] = total
        args, out, lse = _check_attend(c)
        page, k = c["bt"][0, 4], dim // 32 - 1
        vd, vs = args[2].clone(), args[4].clone()
        vd[page, 9, 1, 16 * k:16 * k + 16] = 0
        vs[page, 9, 1, k] = float(bad)
        got, lse2 = _attend([*args[:2], vd, args[3], vs, *args[5:]])
        nan = torch.zeros_like(out, dtype=torch.bool)
        nan[0, hq // 2:, 32 * k:32 * k + 32] = True
        assert torch.equal(torch.isnan(got), nan) and torch.equal(lse2, lse)
        assert torch.equal(got[~nan], out[~nan])
