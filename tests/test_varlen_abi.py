"""Host-side refusals of attention over new tokens, its weights and eviction: a bad
size, pointer or workspace ends in its status code before any CUDA call, and the
wrappers refuse CPU tensors.  CPU only."""
import math

import pytest
import torch

from iris_kernel import _lib
from iris_kernel._lib import lib

EINVAL, EUNSUPPORTED, EALIGN, EWORKSPACE = 1, 2, 3, 5
P = 64  # stands for an aligned pointer: no refused call reads it


def _attend(**kw):
    a = dict(query=P, query_stride=512, k_data=P, v_data=P, k_scale=P, v_scale=P, block_table=P, stride=4, seq_lens=P, cu=P,
             slopes=None, prefix=None, first=None, output=P, lse=None, tokens=8, batch=2, hq=8, hkv=2, head_dim=64,
             num_pages=4, page_size=16, max_pages=4, window=0, cap=0.0, scale=0.1, dtype=_lib.DTYPE_FP16, workspace=None,
             workspace_bytes=0, error=P, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.iris_b200_int4_paged_varlen_attention(*a.values())


SHARED = [
    (dict(tokens=-1), EINVAL), (dict(batch=-1), EINVAL), (dict(hq=7), EINVAL), (dict(hkv=0), EINVAL), (dict(window=-1), EINVAL),
    (dict(cap=-1.0), EINVAL), (dict(cap=math.nan), EINVAL), (dict(cap=2e20), EINVAL), (dict(scale=0.0), EINVAL), (dict(scale=math.nan), EINVAL),
    (dict(dtype=2), EINVAL), (dict(cu=None), EINVAL), (dict(batch=0), EINVAL), (dict(num_pages=0), EINVAL),
    (dict(max_pages=0), EINVAL), (dict(query=None), EINVAL), (dict(k_scale=None), EINVAL), (dict(seq_lens=None), EINVAL),
    (dict(page_size=32), EUNSUPPORTED), (dict(head_dim=96), EUNSUPPORTED), (dict(head_dim=256), EUNSUPPORTED),
    (dict(tokens=1 << 29), EUNSUPPORTED), (dict(max_pages=1 << 27), EUNSUPPORTED), (dict(num_pages=1 << 31), EUNSUPPORTED),
    (dict(query=P + 8), EALIGN), (dict(query_stride=516), EALIGN), (dict(k_data=P + 4), EALIGN), (dict(k_scale=P + 4), EALIGN),
]


@pytest.mark.parametrize("kw, status", SHARED + [
    (dict(output=None), EINVAL), (dict(v_data=None), EINVAL), (dict(output=P + 8), EALIGN), (dict(v_data=P + 8), EALIGN),
])
def test_attention_status(kw, status):
    assert _attend(**kw) == status


def test_attention_of_no_tokens_is_done_at_once():
    assert _attend(tokens=0, query=None, output=None) == 0


def test_attention_workspace():
    """Where blocks share rows: bounded by what is shared, none where nothing is."""
    need = lib.iris_b200_varlen_attention_workspace_bytes
    shape = (8, 2, 64, 1000, 0, 0)
    assert need(0, 2, *shape, 1, 0) == 0 and need(8, 0, *shape, 1, 0) == 0
    one = need(1, 1, 8, 2, 64, 5000, 0, 0, 0, 0)  # a long context: parts of its 4 columns a KV head
    assert one > 0 and one % (2 * 4 * 65 * 4) == 0
    assert need(1, 1, 8, 2, 64, 8, 0, 0, 0, 0) == 0  # one tile
    # prompts of many tokens: only the few rows that a sequence of theirs might have are shared
    assert need(8192, 2, 32, 8, 128, 256, 0, 0, 1, 0) < 16 << 20


@pytest.mark.parametrize("change", [
    dict(max_pages=0), dict(max_pages=-5), dict(max_pages=-(2 ** 31)), dict(max_pages=1 << 27), dict(max_pages=2 ** 31 - 1),
    dict(head_dim=0), dict(head_dim=-64), dict(head_dim=96), dict(window=-3), dict(tokens=1 << 29), dict(tokens=2 ** 63 - 1),
    dict(batch=-1), dict(hq=7), dict(hkv=0), dict(hq=0), dict(offsets=0)])
def test_attention_workspace_of_what_is_refused(change):
    """A size is asked for before the call that refuses the sizes: no workspace, and the process goes on."""
    a = dict(tokens=8, batch=2, hq=8, hkv=2, head_dim=64, max_pages=5000, window=0, prefix=0, offsets=1, device=0)
    need = lib.iris_b200_varlen_attention_workspace_bytes
    assert need(*a.values()) > 0
    a.update(change)
    assert need(*a.values()) == 0


def _mass(**kw):
    a = dict(query=P, query_stride=512, lse=P, k_data=P, k_scale=P, block_table=P, stride=4, seq_lens=P, cu=P, slopes=None,
             prefix=None, first=None, first_token=None, mass=P, tokens=8, batch=2, hq=8, hkv=2, head_dim=64, num_pages=4,
             page_size=16, max_pages=4, window=0, cap=0.0, scale=0.1, decay=1.0, dtype=_lib.DTYPE_FP16, error=P, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.iris_b200_int4_paged_attention_mass(*a.values())


@pytest.mark.parametrize("kw, status", SHARED + [(dict(lse=None), EINVAL), (dict(mass=None), EINVAL), (dict(mass=P + 2), EALIGN)])
def test_mass_status(kw, status):
    assert _mass(**kw) == status


def test_mass_without_sequences_is_done_at_once():
    assert _mass(tokens=0, batch=0) == 0


def _evict(**kw):
    a = dict(k_data=P, v_data=P, k_scale=P, v_scale=P, mass=P, block_table=P, stride=4, seq_lens=P, new_lens=P, kept=None,
             batch=2, hkv=2, head_dim=64, num_pages=4, page_size=16, max_pages=4, budget=32, sink=4, recent=8, workspace=P,
             workspace_bytes=1 << 20, error=P, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.iris_b200_int4_paged_evict(*a.values())


@pytest.mark.parametrize("kw, status", [
    (dict(batch=-1), EINVAL), (dict(hkv=0), EINVAL), (dict(budget=0), EINVAL), (dict(sink=-1), EINVAL), (dict(recent=-1), EINVAL),
    (dict(sink=33), EINVAL), (dict(sink=20, recent=13), EINVAL), (dict(num_pages=0), EINVAL), (dict(max_pages=0), EINVAL),
    (dict(mass=None), EINVAL), (dict(new_lens=None), EINVAL), (dict(v_scale=None), EINVAL), (dict(page_size=8), EUNSUPPORTED),
    (dict(head_dim=32), EUNSUPPORTED), (dict(batch=1 << 28, hkv=8), EUNSUPPORTED), (dict(k_data=P + 8), EALIGN),
    (dict(k_scale=P + 2), EALIGN), (dict(mass=P + 4), EALIGN), (dict(workspace=None), EWORKSPACE),
    (dict(workspace_bytes=767), EWORKSPACE), (dict(workspace=P + 2), EALIGN),
])
def test_evict_status(kw, status):
    assert _evict(**kw) == status


APART = {k: (i + 1) << 20 for i, k in enumerate(
    ("k_data", "v_data", "k_scale", "v_scale", "mass", "block_table", "seq_lens", "new_lens", "kept", "workspace"))}


@pytest.mark.parametrize("out,size", [("new_lens", 2 * 4), ("kept", 2 * 2 * 32 * 4)])
@pytest.mark.parametrize("other,other_size", [("seq_lens", 2 * 4), ("block_table", (4 + 4) * 4), ("mass", 4 * 2 * 16 * 4),
                                              ("k_data", 4 * 16 * 2 * 32), ("v_scale", 4 * 16 * 2 * 4), ("workspace", 768), (None, 0)])
def test_evict_outputs_apart(out, size, other, other_size):
    """An output in what the kernel's other clusters still read, or in the other output, is refused: the first byte and the last."""
    other = other or {"new_lens": "kept", "kept": "new_lens"}[out]
    other_size = other_size or {"new_lens": 2 * 4, "kept": 2 * 2 * 32 * 4}[other]
    at = APART[other]
    for where in (at, at + other_size - 4, at - size + 4):
        assert _evict(**dict(APART, **{out: where}), workspace_bytes=768) == EINVAL
    if out == "new_lens" and other == "seq_lens" and not torch.cuda.is_available():  # (no GPU here: what is accepted ends at the launch)
        for where in (at + other_size, at - size):
            assert _evict(**dict(APART, **{out: where}), workspace_bytes=768) not in (0, EINVAL)


def test_evict_workspace():
    need = lib.iris_b200_evict_workspace_bytes
    assert need(2, 2, 32, 8) == 2 * 2 * 2 * 24 * 4
    assert need(0, 2, 32, 8) == 0 and need(2, 2, 32, 32) == 0
    assert _evict(batch=0) == 0
    assert _evict(budget=2 ** 31 - 1, mass=P + 4, workspace=None, workspace_bytes=0) == EALIGN  # not EWORKSPACE


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-CUDA error path")
def test_wrappers_require_cuda():
    from iris_kernel.fused_kv import fused_int4_paged_evict
    from iris_kernel.varlen_attention import fused_int4_paged_attention_mass, fused_int4_paged_varlen_attention

    q, d, s = torch.zeros(1, 2, 64).half(), torch.zeros(1, 16, 2, 32, dtype=torch.uint8), torch.zeros(1, 16, 2, 2).half()
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_int4_paged_varlen_attention(q, d, d, s, s, i[None], i)
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_int4_paged_attention_mass(q, torch.zeros(1, 2), d, s, i[None], i, torch.zeros(1, 2, 16))
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_int4_paged_evict(d, d, s, s, torch.zeros(1, 2, 16), i[None], i, budget=8)
    with pytest.raises(TypeError, match="torch.Tensor"):
        fused_int4_paged_varlen_attention(None, d, d, s, s, i[None], i)
