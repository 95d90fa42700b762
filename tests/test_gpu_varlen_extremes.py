"""Attention of new tokens at the ends of its arguments' ranges, against 64 bits."""
import numpy as np
import pytest
import torch

import _sparse_refs as R
import _varlen_refs as V
from test_gpu_varlen_attention import BF16, F16, Case, _dev, close

pytestmark = pytest.mark.gpu

LOWEST = -2 ** 31


@pytest.mark.parametrize("prefix", [[LOWEST, LOWEST + 31], [LOWEST + 200, LOWEST + 1000], [2 ** 31 - 1, LOWEST]])
@pytest.mark.parametrize("window", [0, 30])
def test_prefixes_that_are_far_below_zero(prefix, window):
    """No prefix, however far below 0 it lies."""
    how = dict(prefix_lens=np.array(prefix, np.int32), window=window)
    Case([150, 20], [700, 40], 4, 2, 64, seed=7, **how).spoil_tails().check()
    Case([1, 1], [700, 40], 4, 2, 128, seed=8, **how).spoil_tails().check()


# ---- logits near and past 2^24, where fp32 holds whole numbers only
ONE = float(np.float32(0.6931472))  # its product with log2(e) is 1 in fp32: logits in log2 units are the sums q.k


def _towering(new, lens, hq, exponent, extra, offsets):
    """Two tokens of 300 count: 3 with logit `base` and 200, in another tile, with base + extra; base has the given
    exponent and differs from row to row.  Every step on the way is exact in fp32."""
    c = Case(new, lens, hq, 1, 64, seed=exponent, offsets=offsets, softmax_scale=ONE)
    rows = c.query.shape[0] * hq
    q0 = (1024 + np.arange(rows) * 7 % 1024) * 2.0 ** (exponent - 24)
    base = q0 * 2.0 ** 14
    assert (base < 2.0 ** (exponent + 1)).all() and (base >= 2.0 ** exponent).all()
    assert (np.float32(base + extra) == base + extra).all()
    query = np.zeros((rows, 64), np.float32)
    query[:, 0], query[:, 32] = q0, extra
    c.query = R.to_type(query.reshape(-1, hq, 64), F16)
    for b in range(len(lens)):
        pages = c.bt[b, np.arange(lens[b]) // 16], np.arange(lens[b]) % 16
        c.cache[0][pages] = 0
        c.cache[2][pages] = 1.0
        for j in (3, 200):
            at = c.bt[b, j // 16], j % 16, 0
            c.cache[0][at][0] = 1        # dim 0: 1 times 2^14
            c.cache[2][at][0] = 2.0 ** 14
            c.cache[0][at][16] = int(j == 200)  # dim 32
    return c, base.reshape(-1, hq)


@pytest.mark.parametrize("new,lens,hq,offsets", [([1] * 12, [300] * 12, 8, False), ([5] * 4, [300] * 4, 4, True), ([40], [300], 8, True)])
@pytest.mark.parametrize("exponent,extra", [(23, 8), (24, 8), (24, -8), (25, 8), (25, 4), (26, 8), (26, -8), (26, 0), (27, 0),
                                            (27, 16), (27, -16), (28, 0), (28, 32), (29, 0), (29, 64)])
def test_logits_that_tower(new, lens, hq, offsets, exponent, extra):
    """Finite logits give finite outputs: no probability passes what fp16 holds, however coarse the logits have become."""
    c, base = _towering(new, lens, hq, exponent, extra, offsets)
    out, lse = c.run()
    seq = np.repeat(np.arange(len(lens)), new)
    value = [R.dequant(c.cache[1][c.bt[seq, j // 16], j % 16, 0], c.cache[3][c.bt[seq, j // 16], j % 16, 0], np.float64) for j in (3, 200)]
    w = 1.0 / (1.0 + 2.0 ** -float(extra))  # the second token's
    want = ((1 - w) * value[0] + w * value[1])[:, None].repeat(hq, 1)
    most = ((1 - w) * np.abs(value[0]) + w * np.abs(value[1]))[:, None]
    # probabilities and values in fp16, the output in fp16, fp32's sums
    far = most * (2 * 2.0 ** -11 + 2.0 ** -18) + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    close(out, want, np.broadcast_to(far, want.shape))
    want_lse = base + max(extra, 0) + np.log2(1 + 2.0 ** -abs(extra))
    close(lse, want_lse, np.abs(want_lse) * 2.0 ** -22)


# ---- values of very different sizes
def _alike(c, got, rows, quiet):
    """`rows` have what they would have if the tokens `quiet` had no value: those are not seen, or weigh nothing."""
    out, lse = got
    for b, j in quiet:
        c.cache[3][c.bt[b, j // 16], j % 16] = 0
    want, want_lse, far, far_lse = c.want()
    close(out[rows], want[rows], far[rows])
    close(lse[rows], want_lse[rows], far_lse[rows])


def _sized(c, b, tokens, lo, hi):
    """Values of a few sizes in [lo, hi]."""
    for j in tokens:
        c.cache[3][c.bt[b, j // 16], j % 16] = np.exp(c.rng.uniform(np.log(lo), np.log(hi), c.cache[3].shape[2:])).astype(np.float16)


@pytest.mark.parametrize("small", [2.0 ** -9, 2.0 ** -19])
@pytest.mark.parametrize("new,hq,dim,dtype", [([60], 8, 64, BF16), ([200], 4, 128, F16), ([3], 8, 128, BF16), ([1], 4, 64, F16)])
def test_unseen_values_do_not_matter(new, hq, dim, dtype, small):
    """Large values that a window has left behind, in the same page as what is seen and before it."""
    n = 260
    c = Case(new, [n], hq, 2, dim, dtype, seed=41, window=50)
    edge = n - new[0] - 49  # the first token that any row sees
    _sized(c, 0, range(edge), 9000.0, 60000.0)
    _sized(c, 0, range(edge, n), small / 8, small)
    _alike(c, c.run(), slice(None), [(0, j) for j in range(edge)])


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
def test_documents_with_values_of_different_sizes(dim, dtype):
    """Two documents that share tiles and runs, one with values 2^30 times the other's: each has its own bits."""
    n, cut = 300, 150
    first = np.where(np.arange(n) < cut, 0, cut).astype(np.int32)
    for large in (range(cut), range(cut, n)):
        c = Case([n], [n], 4, 2, dim, dtype, seed=42, first_visible=first)
        rest = sorted(set(range(n)) - set(large))
        _sized(c, 0, large, 9000.0, 60000.0)
        _sized(c, 0, rest, 2.0 ** -20, 2.0 ** -16)
        got = c.run()
        _alike(c, [x.clone() for x in got], np.array(rest), [(0, j) for j in large])


@pytest.mark.parametrize("new", [[100], [2], [1]])
def test_large_values_that_weigh_nothing(new):
    """A bias puts the large values' tokens 2^-60 and further down: what is left of them is below the small ones' last bit."""
    n = 400
    slopes = np.array([1.0, 2.0, 1.0, 0.7], np.float32)
    c = Case(new, [n], 4, 2, 64, BF16, seed=43, slopes=slopes, sharp=0.1)
    far = range(n - new[0] - 150)
    _sized(c, 0, far, 9000.0, 60000.0)
    _sized(c, 0, range(far.stop, n), 2.0 ** -19, 2.0 ** -17)
    _alike(c, c.run(), slice(None), [(0, j) for j in far])


@pytest.mark.parametrize("new,offsets", [([40], True), ([5], True), ([1], False)])
def test_values_that_decide_by_their_size(new, offsets):
    """Tokens of next to no weight with values so large that the output is theirs."""
    n = 300
    c = Case(new, [n], 4, 1, 64, F16, seed=44, offsets=offsets, softmax_scale=1.0)
    query = np.zeros((new[0], 4, 64), np.float32)
    query[..., 0] = 1.0
    c.query = R.to_type(query, F16)
    for j in range(n):
        at = c.bt[0, j // 16], j % 16, 0
        c.cache[0][at] = 0
        light = j % 3 == 0 and j < 250
        c.cache[0][at][0] = 0 if light else 7  # logits 0, or 17.5: 2^-25 of the weight
        c.cache[2][at] = 2.5
        c.cache[3][at] = np.float16(2.0 ** 14 if light else 2.0 ** -16)
    out, lse = c.run()
    want, want_lse, far, far_lse = c.want()
    # (relative to the sum of what tokens contribute: probabilities and values in fp16)
    x, _, seen = V._sequence(R.f32(c.query), c.cache, c.bt, c.lens, c.cu, 0, 0, **V._options(dict(scale=1.0)))
    w = np.where(seen, np.exp(x - np.log(np.exp(x).sum(-1, keepdims=True))), 0.0)
    pages = c.bt[0, np.arange(n) // 16], np.arange(n) % 16, 0
    most = (w @ np.abs(R.dequant(c.cache[1][pages], c.cache[3][pages], np.float64))).transpose(1, 0, 2)
    close(out, want, most * (2 * 2.0 ** -11 + 2.0 ** -15) + np.abs(want) * 2.0 ** -11 + 2.0 ** -25)
    close(lse, want_lse, far_lse)


@pytest.mark.parametrize("exponent", [-10, -4, 0, 12])
@pytest.mark.parametrize("new,lens", [([70], [400]), ([5, 1], [300, 130])])
def test_every_nibble_and_full_mantissas(new, lens, exponent):
    """-8, which the append does not write but the format has, times scales just below a power of two."""
    c = Case(new, lens, 4, 2, 64, BF16, seed=45, sharp=2.0 ** -max(exponent, 0))
    for x in c.cache[:2]:
        x[...] = c.rng.integers(0, 256, x.shape)
    for x in c.cache[2:]:
        x[...] = ((2.0 - c.rng.integers(1, 9, x.shape) * 2.0 ** -10) * 2.0 ** exponent).astype(np.float16)
    c.check()


@pytest.mark.parametrize("new,lens,offsets", [([1, 1], [400, 300], False), ([5, 2], [300, 500], True), ([40], [300], True)])
@pytest.mark.parametrize("q0", [64.0, -128.0])
def test_logits_far_below_those_that_count(new, lens, offsets, q0):
    """A row whose first tile lies at -2^22 to -2^24, and the rest where logits usually are: nothing is lost on the way."""
    c = Case(new, lens, 8, 2, 64, BF16, seed=46, offsets=offsets)
    c.query[..., 0] = -abs(q0)
    for b in range(len(lens)):
        at = c.bt[b, np.arange(lens[b]) // 16], np.arange(lens[b]) % 16
        c.cache[0][at[0], at[1], :, 0] &= 0xf0  # dim 0: nothing ...
        for j in range(128):                   # ... but in the first tile
            c.cache[0][c.bt[b, j // 16], j % 16, :, 0] |= 7
            c.cache[2][c.bt[b, j // 16], j % 16, :, 0] = 62000.0 if q0 < 0 else 65504.0
    out, lse = c.run()
    c.how["first_visible"] = np.full(c.query.shape[0], 128, np.int32)
    want, want_lse, far, far_lse = c.want()
    close(out, want, far)
    close(lse, want_lse, far_lse)


def test_a_bias_that_falls_to_far_below():
    """The nearest token decides, and its logit is the log-sum-exp to the last bits."""
    for new, lens, offsets in (([1], [400], False), ([3], [300], True), ([60], [300], True)):
        slopes = np.array([2e4, 5e4, 1e5, 3e4], np.float32)
        Case(new, lens, 4, 2, 64, BF16, seed=47, offsets=offsets, slopes=slopes).check()
