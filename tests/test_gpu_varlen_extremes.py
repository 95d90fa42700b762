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
