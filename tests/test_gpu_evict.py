"""Eviction, bit for bit against its definition."""
import numpy as np
import pytest
import torch

import _sparse_refs as R
import _varlen_refs as V

pytestmark = pytest.mark.gpu


def _dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def _batch(lens, hkv, dim, seed=0, width=None):
    rng = np.random.default_rng(seed)
    bt, pages = V.table(rng, lens, width)
    cache = list(R.random_cache(rng, pages, hkv, dim))
    return bt, cache, np.exp(2 * rng.standard_normal((pages, hkv, 16))).astype(np.float32)


def _evict(bt, cache, mass, lens, **kw):
    from iris_kernel.fused_kv import fused_int4_paged_evict

    dev = [_dev(x) for x in (*cache, mass)]
    out = fused_int4_paged_evict(*dev, _dev(bt), _dev(np.array(lens, np.int32)), **kw)
    torch.cuda.synchronize()
    return dev, out


def _check(lens, hkv, dim, budget, sink, recent, seed=0, change=None, width=None):
    bt, cache, mass = _batch(lens, hkv, dim, seed, width)
    if change is not None:
        change(mass, bt)
    dev, (new, kept) = _evict(bt, cache, mass, lens, budget=budget, sink_tokens=sink, recent_tokens=recent, return_kept=True)
    want_new, want_kept = V.evict_ref(cache, mass, bt, lens, budget, sink, recent)
    assert np.array_equal(new.cpu().numpy(), want_new)
    assert np.array_equal(kept.cpu().numpy(), want_kept)
    for x, w in zip(dev, (*cache, mass)):
        assert x.cpu().numpy().tobytes() == w.tobytes()


@pytest.mark.parametrize("hkv,dim", [(1, 64), (3, 128), (8, 64)])
@pytest.mark.parametrize("lens,budget,sink,recent", [
    ([17], 16, 4, 4), ([33, 5, 0, 32, 400], 32, 1, 16), ([1000, 999], 100, 0, 0), ([70], 64, 0, 64), ([70], 64, 64, 0),
    ([300], 50, 20, 30), ([129, 128], 127, 3, 100), ([2], 1, 0, 0), ([2], 1, 1, 0), ([2], 1, 0, 1), ([5000], 4999, 4, 4000),
    ([700], 30, 0, 29)])
def test_against_the_definition(lens, budget, sink, recent, hkv, dim):
    _check(lens, hkv, dim, budget, sink, recent, seed=budget + hkv)


@pytest.mark.parametrize("lens,budget,recent", [([20000], 3000, 200), ([9000, 100], 1000, 999), ([6000], 5999, 5000)])
def test_over_clusters(lens, budget, recent):
    _check(lens, 2, 128, budget, 4, min(recent, budget - 4), seed=budget)


def test_more_tokens_than_shared_memory_holds():
    _check([350000], 1, 64, 2000, 4, 100, seed=1)


@pytest.mark.parametrize("fill", ["equal", "zeros", "two values", "specials", "last bits"])
def test_ties_and_special_weights(fill):
    def change(mass, bt):
        rng = np.random.default_rng(5)
        if fill == "equal":
            mass[...] = 0.25
        elif fill == "zeros":
            mass[...] = np.where(rng.random(mass.shape) < 0.5, 0.0, -0.0)
        elif fill == "two values":
            mass[...] = np.where(rng.random(mass.shape) < 0.4, 1.0, 2.0)
        elif fill == "specials":
            mass[...] = rng.choice(np.array([np.nan, np.inf, -np.inf, -1.0, 1e-45, 3e38, -np.nan], np.float32), mass.shape)
        else:
            mass[...] = (np.float32(1.0).view(np.int32) + rng.integers(0, 40, mass.shape)).astype(np.int32).view(np.float32)

    _check([777, 90], 2, 64, 100, 3, 20, change=change)
    _check([9999], 1, 128, 1500, 3, 20, change=change)


def test_again_and_again():
    """A decode loop's use: one token too many each time."""
    lens, bt, cache, mass = [65, 65], *_batch([80, 80], 2, 64, 3)
    for step in range(3):
        dev, new = _evict(bt, cache, mass, lens, budget=64, sink_tokens=2, recent_tokens=16)
        V.evict_ref(cache, mass, bt, lens, 64, 2, 16)
        assert new.tolist() == [64, 64]
        for x, w in zip(dev, (*cache, mass)):
            assert x.cpu().numpy().tobytes() == w.tobytes()


def test_wide_tables_and_given_outputs():
    from iris_kernel.fused_kv import fused_int4_paged_evict

    bt, cache, mass = _batch([200, 40], 2, 64, 4, width=5000)
    dev = [_dev(x) for x in (*cache, mass)]
    wide = torch.full((2, 6000), -7, dtype=torch.int32, device="cuda")
    wide[:, 500:5500] = _dev(bt)
    new, kept = torch.empty(2, dtype=torch.int32, device="cuda"), torch.empty(2, 2, 64, dtype=torch.int32, device="cuda")
    got = fused_int4_paged_evict(*dev, wide[:, 500:5500], _dev(np.array([200, 40], np.int32)), new, kept, budget=64,
                                 sink_tokens=4, recent_tokens=40)
    assert got[0] is new and got[1] is kept
    want_new, want_kept = V.evict_ref(cache, mass, bt, [200, 40], 64, 4, 40)
    assert np.array_equal(new.cpu().numpy(), want_new) and np.array_equal(kept.cpu().numpy(), want_kept)


def test_errors_leave_the_sequence_alone():
    from iris_kernel import _runtime
    from iris_kernel.fused_kv import fused_int4_paged_evict

    bt, cache, mass = _batch([200, 100], 2, 64, 6, width=13)
    for lens, table, error in (([200, -1], bt, ValueError), ([209, 100], bt, ValueError),
                               ([200, 100], np.where(bt == bt[0, 9], 10 ** 6, bt), IndexError),
                               ([200, 100], np.where(bt == bt[0, 0], -1, bt), IndexError)):
        dev = [_dev(x) for x in (*cache, mass)]
        new = torch.zeros(2, dtype=torch.int32, device="cuda")
        with pytest.raises(error):
            fused_int4_paged_evict(*dev, _dev(table.astype(np.int32)), _dev(np.array(lens, np.int32)), new, budget=64,
                                   sink_tokens=4, recent_tokens=8)
        good = 1 if lens[1] == 100 else 0
        want = [x.copy() for x in (*cache, mass)]
        one = [bt[good:good + 1], [lens[good]]]
        V.evict_ref(want[:4], want[4], *one, 64, 4, 8)
        assert new.tolist() == [64 if b == good else lens[b] for b in range(2)]
        for x, w in zip(dev, want):
            assert x.cpu().numpy().tobytes() == w.tobytes()
    dev = [_dev(x) for x in (*cache, mass)]
    args = [*dev, _dev(bt), _dev(np.array([200, 100], np.int32))]
    for kw in (dict(budget=0), dict(budget=10, sink_tokens=4, recent_tokens=7), dict(budget=10, sink_tokens=-1),
               dict(budget=100, recent_tokens=-1)):
        with pytest.raises(ValueError):
            fused_int4_paged_evict(*args, **kw)
    with pytest.raises(NotImplementedError):
        fused_int4_paged_evict(*args, budget=100, page_size=8)
    with pytest.raises(ValueError, match="overlap"):
        fused_int4_paged_evict(*args, args[6], budget=100)
    _runtime.check_errors()


def test_a_budget_that_no_sequence_can_pass():
    bt, cache, mass = _batch([200, 40], 2, 64, 4)
    dev, new = _evict(bt, cache, mass, [200, 40], budget=2 ** 31 - 1)
    assert new.tolist() == [200, 40]
    for x, w in zip(dev, (*cache, mass)):
        assert x.cpu().numpy().tobytes() == w.tobytes()
