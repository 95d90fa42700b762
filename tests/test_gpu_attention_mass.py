"""Accumulated attention weights against 64 bits (tolerances: _varlen_refs)."""
import numpy as np
import pytest
import torch

import _sparse_refs as R
import _varlen_refs as V
from test_gpu_varlen_attention import BF16, F16, Case, _dev, close

pytestmark = pytest.mark.gpu


def _run(c, mass, first=None, decay=1.0, lse=None, query=None, cu=None):
    """(kernel's weights, the definition's, how far they may be off); lse: the attention's own, rounded keys and all."""
    from iris_kernel.varlen_attention import fused_int4_paged_attention_mass

    a = c.args()
    lse = c.run()[1] if lse is None else lse
    got = _dev(mass)
    fused_int4_paged_attention_mass(a[0], lse, a[1], a[3], a[5], a[6], got, a[7], first_token=_dev(first), decay=decay,
                                    **c.options())
    torch.cuda.synchronize()
    how = dict(c.how)
    if "softmax_scale" in how:
        how["scale"] = how.pop("softmax_scale")
    return got, *V.mass_ref(R.f32(c.query), lse.cpu().numpy(), c.cache, c.bt, c.lens, c.cu, mass, first, decay, **how)


def _mass(c, seed=1):
    return np.random.default_rng(seed).exponential(size=(c.cache[0].shape[0], c.cache[0].shape[2], 16)).astype(np.float32)


def _check(c, **kw):
    got, want, far = _run(c, _mass(c), **kw)
    close(got, want, far)
    return got, want


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (6, 2), (8, 8), (40, 2), (150, 1)])
@pytest.mark.parametrize("lens", [[1], [0, 17, 2048], [4097, 1, 16, 128, 129]])
def test_single_tokens(lens, hq, hkv, dim, dtype):
    c = Case([1] * len(lens), lens, hq, hkv, dim, dtype, seed=hq + len(lens), offsets=False).spoil_tails()
    _check(c, first=np.maximum(c.lens - 1, 0), decay=0.9)


@pytest.mark.parametrize("new,lens", [([7, 1, 20], [7, 300, 1000]), ([32, 32], [500, 32]), ([200], [200]), ([0, 5, 0], [30, 60, 0])])
@pytest.mark.parametrize("hq,hkv,dim", [(8, 2, 64), (3, 1, 128)])
def test_windows_of_queries(new, lens, hq, hkv, dim):
    c = Case(new, lens, hq, hkv, dim, seed=len(new)).spoil_tails()
    got, want = _check(c)
    again = _run(c, _mass(c))[0]
    assert torch.equal(got, again)
    _check(c, first=np.array([max(0, n - m - 3) for m, n in zip(new, lens)], np.int32), decay=0.5)


def test_weights_of_rows_add_up_to_one():
    c = Case([40], [700], 4, 2, 128, seed=3)
    got, _ = _check(c)
    pages = c.bt[0][np.arange(700) // 16]
    total = got.cpu().numpy()[pages, :, np.arange(700) % 16].sum(0)
    assert np.abs(total / 80 - 1).max() < 2.0 ** -10  # (the attention's keys are rounded)


def test_masks_cap_and_bias():
    rng = np.random.default_rng(11)
    new, lens = [200, 1, 90], [333, 20, 90]
    first = np.concatenate([np.sort(rng.integers(0, 300, 200)), [7], np.repeat([0, 31, 64], 30)]).astype(np.int32)
    first[5], first[40], first[199], first[-1] = 2 ** 31 - 1, -9, 333, 2 ** 30
    slopes = (2.0 ** -np.arange(1, 7)).astype(np.float32)
    for how in (dict(window=30), dict(window=200, prefix_lens=np.array([140, 3, 0], np.int32)), dict(logit_cap=3.0),
                dict(slopes=slopes), dict(first_visible=first),
                dict(first_visible=first, window=90, prefix_lens=np.array([33, 3, 50], np.int32), slopes=slopes, logit_cap=20.0)):
        _check(Case(new, lens, 6, 2, 128, BF16, seed=12, **how).spoil_tails(), decay=0.75)
        _check(Case(new, lens, 6, 2, 64, F16, seed=13, **how).spoil_tails())


def test_tokens_and_pages_of_others_stay():
    c = Case([4], [70], 4, 2, 64, seed=5)
    mass = _mass(c)
    got, _, _ = _run(c, mass)
    got = got.cpu().numpy()
    other = np.setdiff1d(np.arange(mass.shape[0]), c.bt[0, :5])
    assert np.array_equal(got[other], mass[other]) and np.array_equal(got[c.bt[0, 4], :, 6:], mass[c.bt[0, 4], :, 6:])


@pytest.mark.parametrize("lo,hi", [(2.0 ** -14, 2.0 ** -14), (2.0 ** -24, 2.0 ** -20), (9000.0, 65504.0)])
def test_scales_of_all_sizes(lo, hi):
    c = Case([20, 1], [300, 130], 4, 2, 64, seed=21)
    c.cache[2][...] = np.exp(c.rng.uniform(np.log(lo), np.log(hi), c.cache[2].shape)).astype(np.float16)
    c.query = R.to_type(R.f32(c.query) * (30.0 / hi if hi > 1 else 1000.0), F16)
    _, want_lse, _, _ = c.want()
    _check(c, lse=torch.from_numpy(want_lse.astype(np.float32)).cuda())


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_scales_that_are_not_finite(bad):
    c = Case([60], [260], 4, 2, 64, seed=23, window=100)
    _, want_lse, _, _ = c.want()
    lse = torch.from_numpy(want_lse.astype(np.float32)).cuda()
    c.cache[2][c.bt[0, 230 // 16], 230 % 16, 0, 1] = bad
    c.cache[2][c.bt[0, 3 // 16], 3 % 16] = bad  # seen by no row
    got, want, far = _run(c, _mass(c), lse=lse)
    want[c.bt[0, 230 // 16], 0, 230 % 16] = np.nan
    close(got, want, far)


def test_an_lse_that_is_too_small_and_rows_that_saw_nothing():
    c = Case([5], [50], 2, 1, 64, seed=6)
    lse = torch.full((5, 2), -200.0, device="cuda")
    lse[3] = float("-inf")
    got, _, _ = _run(c, _mass(c), lse=lse)
    n = got.cpu().numpy()[c.bt[0][np.arange(50) // 16], 0, np.arange(50) % 16]
    assert np.array_equal(n, [8.0] * 46 + [6.0, 4.0, 2.0, 2.0])


def test_errors():
    from iris_kernel.varlen_attention import fused_int4_paged_attention_mass as f

    c = Case([5, 9], [40, 60], 4, 2, 64, seed=18)
    a = c.args()
    lse = c.run()[1]
    good = [a[0], lse, a[1], a[3], a[5], a[6], _dev(_mass(c)), a[7]]
    for at, x, error in ((1, lse[:3], ValueError), (1, lse.half(), TypeError), (6, good[6][:, :1], ValueError),
                         (6, good[6].double(), TypeError), (7, a[7][:2], ValueError), (7, None, ValueError)):
        with pytest.raises(error):
            f(*good[:at], x, *good[at + 1:])
    for kw in (dict(decay=1.5), dict(decay=-0.1), dict(decay=float("nan")), dict(window=-2), dict(first_token=a[7])):
        with pytest.raises(ValueError):
            f(*good, **kw)
    with pytest.raises(ValueError, match="overlap"):
        f(*good[:1], good[6].flatten()[:56].view(14, 4), *good[2:])
    for at, x, error in ((5, [40, -1], ValueError), (5, [40, 65], ValueError), (5, [4, 60], ValueError),
                         (7, [0, 15, 14], ValueError), (4, [[0, 99, 1, 2], [3, 4, 5, 6]], IndexError)):
        with pytest.raises(error):
            f(*good[:at], torch.tensor(x, dtype=torch.int32, device="cuda"), *good[at + 1:])
    _check(c)


@pytest.mark.parametrize("place", [1, 18])
@pytest.mark.parametrize("bad", [-1, 2 ** 31 - 1])
def test_a_bad_page_id_writes_to_no_page(place, bad):
    from iris_kernel.varlen_attention import fused_int4_paged_attention_mass as f

    c = Case([3], [300], 4, 2, 64, seed=27)
    a = c.args()
    lse, mass = c.run()[1], _mass(c)
    table = c.bt.copy()
    table[table == 0] = table[0, place]  # page 0 is nobody's
    table[0, place] = bad
    got = _dev(mass)
    with pytest.raises(IndexError):
        f(a[0], lse, a[1], a[3], _dev(table), a[6], got, a[7])
    torch.cuda.synchronize()
    others = np.setdiff1d(np.arange(mass.shape[0]), table[0, :19])
    assert 0 in others and np.array_equal(got.cpu().numpy()[others], mass[others])
    mine = table[0, :18 if place == 18 else 19][np.arange(18 if place == 18 else 19) != place]
    assert (got.cpu().numpy()[mine] != mass[mine]).any(axis=(1, 2)).all()
