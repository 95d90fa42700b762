"""Attention of new tokens right behind what writes its inputs, with nothing in between that waits."""
import numpy as np
import pytest
import torch

import _sparse_refs as R
from test_gpu_varlen_attention import Case, _dev

pytestmark = pytest.mark.gpu

I32 = torch.int32


@pytest.fixture
def deferred():
    from iris_kernel import set_validation_mode

    set_validation_mode("deferred")
    yield
    set_validation_mode("sync")


@pytest.mark.parametrize("new,lens", [([1, 70, 3, 1, 33], [700, 70, 50, 1, 2000]), ([1, 4, 2], [4096, 90, 2]), ([300, 40], [300, 900])])
def test_behind_an_append(new, lens, deferred):
    """Rows of both kinds (few and many a sequence) read what the append before them has just written: cache, queries,
    lengths, offsets, page tables.  Every round has other values in the same places."""
    from iris_kernel import _runtime
    from iris_kernel.fused_kv import fused_mrope_int4_paged_append
    from iris_kernel.varlen_attention import fused_int4_paged_varlen_attention

    hq, hkv, dim, rounds = 8, 2, 64, 6
    c = Case(new, lens, hq, hkv, dim, seed=51)
    total = int(c.cu[-1])
    rng = np.random.default_rng(52)
    seq = np.repeat(np.arange(len(new)), new)
    place = np.concatenate([n - m + np.arange(m) for m, n in zip(new, lens)])
    slots = _dev((c.bt[seq, place // 16] * 16 + place % 16).astype(np.int32))
    positions = torch.arange(total, dtype=I32, device="cuda")[None].contiguous()
    ang = np.arange(total)[:, None] * 100.0 ** (-np.arange(dim // 2) / (dim // 2))
    cos, sin = (R.to_type(fn(ang), torch.float16).cuda() for fn in (np.cos, np.sin))
    inputs = [[R.to_type(rng.standard_normal((total, h, dim)) * s, torch.float16).cuda() for h, s in ((hkv, 1), (hkv, 1), (hq, 2))]
              for _ in range(rounds)]
    given = [_dev(c.lens), _dev(c.cu), _dev(c.bt)]
    kw = dict(sections=(dim // 2,), rotary_dim=dim, page_size=16)

    def run(wait):
        cache = [_dev(x) for x in c.cache]
        rotated = torch.empty(total, hq, dim, dtype=torch.float16, device="cuda")
        lens_, cu_, bt_ = (torch.empty_like(x) for x in given)
        out = []
        for key, value, query in inputs:
            for x, y in zip((lens_, cu_, bt_), given):
                x.zero_()
                x.copy_(y)
            fused_mrope_int4_paged_append(key, value, positions, slots, cos, sin, *cache, query, query_out=rotated, **kw)
            if wait:
                torch.cuda.synchronize()
            out += fused_int4_paged_varlen_attention(rotated, *cache, bt_, lens_, cu_, return_lse=True)
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        _runtime.check_errors(0)
        return out

    want = run(True)
    assert not torch.equal(want[0], want[2])
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(run(False), want))
