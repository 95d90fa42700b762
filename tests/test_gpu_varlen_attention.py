"""Attention of new tokens over the INT4 cache against 64 bits (tolerances: _varlen_refs)."""
import numpy as np
import pytest
import torch

import _sparse_refs as R
import _varlen_refs as V

pytestmark = pytest.mark.gpu

F16, BF16, I32 = torch.float16, torch.bfloat16, torch.int32


def _dev(x):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()


class Case:
    """A batch: `new` tokens and `lens` cached tokens of each sequence."""

    def __init__(self, new, lens, hq, hkv, dim, dtype=F16, seed=0, width=None, sharp=1.0, offsets=True, **how):
        rng = self.rng = np.random.default_rng(seed)
        self.lens, self.dtype, self.how = np.array(lens, np.int32), dtype, how
        self.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.offsets = offsets
        self.bt, pages = V.table(rng, lens, width)
        self.cache = list(R.random_cache(rng, pages, hkv, dim))
        self.query = R.to_type(sharp * rng.standard_normal((int(self.cu[-1]), hq, dim)), dtype)

    def spoil_tails(self):
        """What lies behind a sequence's last token in its last page is never seen."""
        for b, n in enumerate(self.lens):
            if n % 16:
                for x in self.cache[2:]:
                    x[self.bt[b, n // 16], n % 16:] = np.nan
                for x in self.cache[:2]:
                    x[self.bt[b, n // 16], n % 16:] = 0x88
        return self

    def args(self):
        return [self.query.cuda(), *map(_dev, self.cache), _dev(self.bt), _dev(self.lens),
                _dev(self.cu) if self.offsets else None]

    def options(self):
        return {k: _dev(v) if isinstance(v, np.ndarray) else v for k, v in self.how.items()}

    def run(self, **kw):
        from iris_kernel.varlen_attention import fused_int4_paged_varlen_attention

        out = fused_int4_paged_varlen_attention(*self.args(), return_lse=True, **self.options(), **kw)
        torch.cuda.synchronize()
        return out

    def want(self):
        how = dict(self.how)
        if "softmax_scale" in how:
            how["scale"] = how.pop("softmax_scale")
        return V.attend_ref(R.f32(self.query), self.cache, self.bt, self.lens, self.cu, self.dtype, **how)

    def check(self, got=None):
        out, lse = self.run() if got is None else got
        want, want_lse, far, far_lse = self.want()
        close(out, want, far)
        close(lse, want_lse, far_lse)
        return out, lse


def close(got, want, far):
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want)), "NaN in other places"
    fin = np.isfinite(want)
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)]), "infinities in other places"
    off = np.abs(got[fin] - want[fin])
    assert (off <= far[fin]).all(), f"off by {off.max():.3e}, {(off - far[fin]).max():.3e} too much"


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,lens", [([1], [1]), ([1, 1, 1], [5, 128, 129]), ([7, 1, 20], [7, 300, 1000]),
                                      ([64], [64]), ([130, 3], [130, 260]), ([300, 65], [300, 999])])
def test_causal(new, lens, dim, dtype):
    Case(new, lens, 8, 2, dim, dtype, seed=len(new) + dim).spoil_tails().check()


@pytest.mark.parametrize("hq,hkv", [(1, 1), (6, 2), (5, 1), (16, 16), (32, 2), (40, 8), (130, 1), (300, 1)])
@pytest.mark.parametrize("new,lens", [([1, 1], [77, 400]), ([9, 33], [200, 33])])
def test_head_groups(hq, hkv, new, lens):
    Case(new, lens, hq, hkv, 64, seed=hq).spoil_tails().check()
    if set(new) == {1}:
        Case(new, lens, hq, hkv, 128, seed=hq, offsets=False).spoil_tails().check()


@pytest.mark.parametrize("lens", [[1], [0, 17, 2048], [4097, 1, 16, 15], [20000]])
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
def test_single_tokens(lens, dim, dtype):
    c = Case([1] * len(lens), lens, 8, 2, dim, dtype, seed=sum(lens), offsets=False).spoil_tails()
    out, lse = c.check()
    again = c.run()
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])  # the same bits
    idle = np.flatnonzero(c.lens == 0)
    assert not out[idle].any() and torch.isneginf(lse[idle]).all()


def test_a_long_context_shared_by_many_blocks():
    Case([3], [40000], 8, 1, 128, seed=5).spoil_tails().check()
    Case([40], [9000], 16, 2, 64, BF16, seed=6, sharp=3.0).spoil_tails().check()


@pytest.mark.parametrize("cap", [0.5, 30.0, 1e4])
@pytest.mark.parametrize("sharp", [0.01, 1.0, 30.0])
def test_cap(cap, sharp):
    Case([40, 1], [290, 33], 4, 2, 128, seed=3, logit_cap=cap, sharp=sharp).spoil_tails().check()


@pytest.mark.parametrize("window", [1, 2, 63, 128, 129, 1000, 2 ** 31 - 1])
@pytest.mark.parametrize("new,lens", [([1, 1], [500, 40]), ([150, 20], [700, 20]), ([400], [400])])
def test_window(window, new, lens):
    Case(new, lens, 4, 2, 64, seed=window % 97, window=window).spoil_tails().check()


@pytest.mark.parametrize("prefix", [[0, 0], [1, 300], [128, 40], [10 ** 6, 129], [-5, 7]])
@pytest.mark.parametrize("window", [0, 30, 257])
def test_prefix(prefix, window):
    Case([150, 20], [700, 40], 4, 2, 64, seed=7, prefix_lens=np.array(prefix, np.int32), window=window).spoil_tails().check()
    Case([1, 1], [700, 40], 4, 2, 128, seed=8, prefix_lens=np.array(prefix, np.int32), window=window).spoil_tails().check()


@pytest.mark.parametrize("bias,cap,window,prefix", [(False, 0.0, 0, 0), (True, 0.0, 0, 0), (True, 20.0, 90, 33), (False, 5.0, 0, 140)])
def test_documents(bias, cap, window, prefix):
    """Rows that see nothing among them: first visible tokens past their own place, or past everything."""
    rng = np.random.default_rng(11)
    new, lens = [200, 1, 90], [333, 20, 90]
    first = np.concatenate([np.sort(rng.integers(0, 300, 200)), [7], np.repeat([0, 31, 64], 30)]).astype(np.int32)
    first[5], first[40], first[199], first[-1] = 2 ** 31 - 1, -9, 333, 2 ** 30
    how = dict(first_visible=first, window=window, logit_cap=cap)
    if bias:
        how["slopes"] = (2.0 ** -np.arange(1, 7)).astype(np.float32)
    if prefix:
        how["prefix_lens"] = np.array([prefix, 3, prefix], np.int32)
    c = Case(new, lens, 6, 2, 128, BF16, seed=12, **how).spoil_tails()
    out, lse = c.check()
    assert not out[5].any() and torch.isneginf(lse[5]).all()


@pytest.mark.parametrize("slope", [0.0, 0.05, 8.0, -0.01])
def test_bias(slope):
    slopes = (slope * np.array([1, 0.5, 0.25, 2])).astype(np.float32)
    Case([100, 1], [600, 257], 4, 1, 64, seed=4, slopes=slopes, prefix_lens=np.array([580, 0], np.int32)).spoil_tails().check()


def test_softmax_scale_and_sharp_rows():
    for sharp, scale in ((1.0, 1.0), (200.0, None), (1e-3, 1e-3), (40.0, 0.5)):
        Case([50, 2], [300, 300], 4, 2, 64, seed=9, sharp=sharp, softmax_scale=scale).check()


@pytest.mark.parametrize("lo,hi", [(2.0 ** -14, 2.0 ** -14), (2.0 ** -24, 2.0 ** -20), (9000.0, 65504.0), (2.0 ** -14, 65504.0)])
@pytest.mark.parametrize("which", ["values", "keys"])
def test_scales_of_all_sizes(lo, hi, which):
    """A run's power of two keeps large scales from overflowing and small ones from losing bits."""
    c = Case([70, 1], [400, 130], 4, 2, 64, seed=21)
    x = c.cache[3 if which == "values" else 2]
    x[...] = np.exp(c.rng.uniform(np.log(lo), np.log(hi), x.shape)).astype(np.float16)
    if which == "keys":
        c.query = R.to_type(R.f32(c.query) * min(1.0, 30.0 / hi) if hi > 1 else R.f32(c.query) * 1000.0, F16)
    c.check()


def test_values_whose_size_changes_from_run_to_run():
    """Values that grow along the sequence, and ones that shrink: the rows' power follows the largest."""
    for order in (1, -1):
        c = Case([40], [600], 4, 2, 128, seed=22)
        for j in range(600):
            c.cache[3][c.bt[0, j // 16], j % 16] = np.float16(2.0 ** (-12 + (j if order > 0 else 599 - j) // 40))
        c.check()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_scales_that_are_not_finite(bad):
    """A key's spoils the rows that see it, a value's the 32 dims of those; unseen ones do nothing."""
    c = Case([60, 1], [260, 200], 4, 2, 64, seed=23, window=100, first_visible=np.array([0] * 30 + [150] * 30 + [0], np.int32))
    c.cache[2][c.bt[0, 230 // 16], 230 % 16, 0, 1] = bad   # seen by rows from place 230 on, head 0
    c.cache[3][c.bt[0, 140 // 16], 140 % 16, 1, 1] = bad   # seen by the rows in whose window and document it lies
    c.cache[2][c.bt[0, 3 // 16], 3 % 16] = bad             # left behind by every window
    c.cache[3][c.bt[1, 60 // 16], 60 % 16] = bad
    out, lse = c.run()
    want, want_lse, far, far_lse = c.want()
    seen = V.visible(200 + np.arange(60), c.how["first_visible"][:60], 0, 100, 260)
    rows = np.flatnonzero(seen[:, 230])
    assert 0 < len(rows) < 60
    want[rows, :2], want_lse[rows, :2] = np.nan, np.nan
    close(out, want, far)
    close(lse, want_lse, far_lse)
    assert np.isnan(want[:60, 2:, 32:]).any() and not np.isnan(want[:60, 2:, :32]).any() and not np.isnan(want[60]).any()


def test_queries_that_are_not_finite():
    c = Case([6], [200], 2, 1, 64, BF16, seed=24)
    c.query[1, 0, 5], c.query[4, 1, 63] = float("inf"), float("nan")
    out, lse = c.run()
    want, want_lse, far, far_lse = c.want()
    want[1, 0], want[4, 1], want_lse[1, 0], want_lse[4, 1] = (np.nan,) * 4
    close(out, want, far)
    close(lse, want_lse, far_lse)


@pytest.mark.parametrize("size", [1e-30, 2.0 ** -130, 1e30])
def test_bf16_queries_of_all_sizes(size):
    c = Case([20], [150], 2, 1, 128, BF16, seed=25, softmax_scale=1.0)
    c.query = R.to_type(R.f32(c.query) * np.float32(size), BF16)
    if size > 1:
        c.cache[2][...] = np.float16(2.0 ** -24)  # logits of 1e23: one token takes all
    out, lse = c.run()
    want, want_lse, far, far_lse = c.want()
    if size < 1:
        close(out, want, far)
        close(lse, want_lse, far_lse)
    else:
        x = np.abs(lse.double().cpu().numpy() - want_lse) / np.abs(want_lse)
        assert x.max() < 2.0 ** -10 and torch.isfinite(out).all()


def test_strided_query_and_output_in_its_place():
    from iris_kernel.varlen_attention import fused_int4_paged_varlen_attention

    c = Case([33, 140], [50, 300], 4, 2, 64, seed=13)
    out, lse = c.check()
    a = c.args()
    wide = torch.randn(a[0].shape[0], 8, 64, device="cuda").half()
    wide[:, 2:6] = a[0]
    assert torch.equal(fused_int4_paged_varlen_attention(wide[:, 2:6], *a[1:]), out)
    assert fused_int4_paged_varlen_attention(*a, a[0]) is a[0]
    assert torch.equal(a[0], out)


def test_rows_behind_the_last_sequence_are_zeros():
    c = Case([5, 9], [40, 60], 4, 2, 64, seed=14)
    out, lse = c.run()
    c.query = torch.cat([c.query, c.query[:6]])
    given = torch.full(c.query.shape, 7.0, dtype=F16, device="cuda")
    got, got_lse = c.run(output=given)
    assert got is given and torch.equal(got[:14], out) and torch.equal(got_lse[:14], lse)
    assert not got[14:].any() and torch.isneginf(got_lse[14:]).all()


def test_sequences_without_new_tokens_and_idle_ones():
    c = Case([0, 5, 0, 4, 3], [30, 60, 0, 0, 3], 4, 2, 64, seed=15)
    out, lse = c.check()
    assert not out[5:9].any() and torch.isneginf(lse[5:9]).all()


def test_many_sequences():
    rng = np.random.default_rng(16)
    new = rng.integers(0, 40, 300).tolist()
    Case(new, [n + int(h) for n, h in zip(new, rng.integers(0, 200, 300))], 2, 1, 64, seed=17).spoil_tails().check()


def test_errors():
    from iris_kernel.varlen_attention import fused_int4_paged_varlen_attention as f

    def bad(error, match, **change):
        c = Case([5, 9], [40, 60], 4, 2, 64, seed=18)
        for k, v in change.items():
            setattr(c, k, np.array(v, np.int32))
        with pytest.raises(error, match=match):
            c.run()

    bad(ValueError, "must not be negative", lens=[40, -1])
    bad(ValueError, "enough pages", lens=[40, 65])
    bad(ValueError, "count the new tokens", lens=[4, 60])
    bad(ValueError, "cu_seqlens", cu=[1, 5, 14])
    bad(ValueError, "cu_seqlens", cu=[0, 15, 14])
    bad(ValueError, "cu_seqlens", cu=[0, 5, 15])
    bad(IndexError, "page id", bt=[[0, 99, 1, 2], [3, 4, 5, 6]])
    bad(IndexError, "page id", bt=[[0, -1, 1, 2], [3, 4, 5, 6]])
    c = Case([5, 9], [40, 60], 4, 2, 64, seed=18)
    c.check()  # and the device is as it was
    a = c.args()
    with pytest.raises(ValueError, match="one row a sequence"):
        f(*a[:7])
    with pytest.raises(ValueError, match="overlap"):
        f(*a[:7], a[7], a[1].view(torch.float16).flatten()[:14 * 4 * 64].view(14, 4, 64))
    with pytest.raises(ValueError, match="slopes"):
        f(*a, slopes=torch.ones(2, device="cuda"))
    with pytest.raises(TypeError):
        f(*a, first_visible=torch.zeros(14, device="cuda"))
    for kw in (dict(window=-1), dict(logit_cap=-1.0), dict(logit_cap=float("nan")), dict(logit_cap=3e38),
               dict(softmax_scale=-0.5)):
        with pytest.raises(ValueError):
            f(*a, **kw)
    with pytest.raises(NotImplementedError):
        f(*a, page_size=32)


def test_an_empty_batch():
    from iris_kernel.varlen_attention import fused_int4_paged_varlen_attention as f

    c = Case([5], [40], 4, 2, 64, seed=19)
    a = c.args()
    out, lse = f(a[0][:0], *a[1:5], a[5][:0], a[6][:0], None, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    out = f(a[0][:0], *a[1:7], torch.zeros(2, dtype=I32, device="cuda"))
    assert out.shape == (0, 4, 64)


def test_another_stream_and_a_graph():
    from iris_kernel import set_validation_mode
    from iris_kernel.varlen_attention import fused_int4_paged_varlen_attention as f

    cases = [Case([1] * 3, [9000, 30, 700], 8, 2, 128, seed=20, offsets=False), Case([90, 3], [90, 6000], 8, 2, 64, seed=21)]
    want = [c.check()[0] for c in cases]
    args = [c.args() for c in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [f(*a) for a in args]
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    set_validation_mode("deferred")
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = [f(*a) for a in args]
        for a in args:
            a[0].mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        for a, g in zip(args, got):
            assert torch.equal(g, f(*a))
    finally:
        set_validation_mode("sync")


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
def test_few_and_many_rows_together(dim, dtype):
    """Decode steps, drafts and prompts in one batch, short and long contexts."""
    new, lens = [1, 300, 4, 0, 8, 9, 1, 33], [9000, 300, 700, 50, 8, 2000, 1, 40]
    Case(new, lens, 8, 2, dim, dtype, seed=31).spoil_tails().check()
    Case(new, lens, 8, 2, dim, dtype, seed=32, window=150, prefix_lens=np.array([40, 290, 0, 9, 8, 777, 1, 0], np.int32),
         logit_cap=30.0).spoil_tails().check()
    Case(new, lens, 3, 1, dim, dtype, seed=33, slopes=np.array([0.5, 0.01, 0.0], np.float32),
         first_visible=np.repeat([100, 7, 0, 3, 1990, 0, 5], [1, 300, 4, 8, 9, 1, 33]).astype(np.int32)).spoil_tails().check()


@pytest.mark.parametrize("hq", [3, 9, 17, 32])
@pytest.mark.parametrize("lens", [[5], [130, 5000]])
def test_single_tokens_of_wide_groups(hq, lens):
    for how in ({}, dict(logit_cap=5.0), dict(slopes=(0.1 * np.arange(hq)).astype(np.float32)), dict(window=77)):
        Case([1] * len(lens), lens, hq, 1, 64 if hq % 2 else 128, seed=hq, offsets=False, **how).spoil_tails().check()
        Case([1] * len(lens), lens, hq, 1, 128 if hq % 2 else 64, seed=hq, offsets=True, **how).spoil_tails().check()


@pytest.mark.parametrize("how", [dict(logit_cap=1e-30), dict(logit_cap=1e20), dict(softmax_scale=1e-38), dict(logit_cap=1e-3, softmax_scale=1e30)])
def test_extreme_caps_and_scales(how):
    """A cap far below the logits, one far above them, logits that vanish: finite, and as the definition has it."""
    for new, lens in (([40], [300]), ([1, 3], [200, 33])):
        Case(new, lens, 4, 2, 64, seed=34, **how).check()


def test_keys_are_exact():
    """The log-sum-exp of a row that sees one token is its logit: fp32's, not fp16's."""
    for new, lens in (([200], [200]), ([1, 1], [300, 40])):
        c = Case(new, lens, 4, 2, 128, seed=35, window=1)
        out, lse = c.run()
        want = c.want()[1]
        assert np.abs(lse.double().cpu().numpy() - want).max() < 2.0 ** -19 * max(1.0, np.abs(want).max())
