"""Attention and its accumulated weights beside each other."""
import numpy as np
import pytest
import torch

import _varlen_refs as V
from test_gpu_attention_mass import _run
from test_gpu_varlen_attention import BF16, F16, Case, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,lens,hq,hkv,dim", [([40], [700], 4, 2, 128), ([200, 9], [600, 333], 8, 2, 64), ([1, 1], [900, 60], 8, 1, 128)])
def test_weights_of_rows_add_up_to_one_as_far_as_exact_keys_allow(new, lens, hq, hkv, dim, dtype):
    """Both operators take keys exactly, so a row's weights miss 1 by what fp32 loses: the logits of both by 2^-18 and
    2^-20 of sum |q k| * scale, the log-sum-exp by 2^-18 of its own size and of 1, the sums by 2^-20."""
    c = Case(new, lens, hq, hkv, dim, dtype, seed=3)
    mass = np.zeros((c.cache[0].shape[0], hkv, 16), np.float32)
    got = _run(c, mass)[0].double().cpu().numpy()
    for b, n in enumerate(lens):
        pages = c.bt[b][np.arange(n) // 16]
        for h in range(hkv):
            x, size, seen = V._sequence(c.query.float().numpy(), c.cache, c.bt, c.lens, c.cu, b, h, **V._options({}))
            lse = np.log2(np.exp(x).sum(-1))
            off = np.expm1(size.max() * (2.0 ** -18 + 2.0 ** -20) + np.log(2.0) * 2.0 ** -18 * (1 + np.abs(lse).max())) + 2.0 ** -20
            rows = (hq // hkv) * new[b]
            total = got[pages, h, np.arange(n) % 16].sum()
            assert off < 2.0 ** -11 and abs(total / rows - 1) <= off, f"{abs(total / rows - 1):.2e} of {off:.2e}"


@pytest.mark.parametrize("rows,hq,dim", [(190, 64, 64), (700, 64, 128), (3, 33, 64), (1000, 1, 64)])
def test_sums_over_many_rows(rows, hq, dim):
    """Thousands of weights of one size: what each addition to a sum of fp32 loses must not add up.  A weight is off by
    2^-22 (the exponential), 8 of them added by 2^-21, and sums of those by 2^-22 however many they are."""
    c = Case([rows], [rows], hq, 1, dim, F16, seed=5, sharp=0.0, prefix_lens=np.array([rows], np.int32))
    lse = torch.full((rows, hq), float(np.log2(rows)), device="cuda")
    got, want, _ = _run(c, np.zeros((c.cache[0].shape[0], 1, 16), np.float32), lse=lse)
    close(got, want, want * 2.0 ** -20)
