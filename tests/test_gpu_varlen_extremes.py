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
