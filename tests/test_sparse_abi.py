"""Host-side refusals of the sparse decode's C entries and wrappers: a bad size,
pointer or workspace ends in its status code before any CUDA call, and the
wrappers refuse CPU tensors.  CPU only."""
import ctypes

import pytest
import torch

from iris_kernel import _lib
from iris_kernel._lib import lib

EINVAL, EUNSUPPORTED, EALIGN, EWORKSPACE = 1, 2, 3, 5
P = 64  # stands for an aligned pointer: no refused call reads it


def _append(**kw):
    sections = kw.pop("sections", (16, 24, 24))
    a = dict(key=P, key_stride=1024, value=P, value_stride=1024, query=P, query_stride=4096, positions=P,
             positions_stride=8, sections=(ctypes.c_int32 * max(len(sections), 1))(*sections), num_axes=len(sections),
             interleaved=0, slots=P, cos=P, sin=P, k_data=P, v_data=P, k_scale=P, v_scale=P, query_out=P, key_out=None,
             num_tokens=8, hq=32, hkv=8, head_dim=128, rotary_dim=128, max_position=64, num_pages=4, page_size=16,
             dtype=_lib.DTYPE_FP16, workspace=None, workspace_bytes=0, error=P, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.iris_b200_mrope_int4_paged_append(*a.values())


@pytest.mark.parametrize("kw, status", [
    (dict(num_tokens=-1), EINVAL), (dict(hkv=0), EINVAL), (dict(page_size=0), EINVAL), (dict(dtype=2), EINVAL),
    (dict(sections=()), EINVAL), (dict(sections=(13, 13, 13, 13, 12)), EINVAL), (dict(sections=(16, 24, 23)), EINVAL),
    (dict(sections=(-1, 41, 24)), EINVAL), (dict(head_dim=96), EUNSUPPORTED), (dict(head_dim=576), EUNSUPPORTED),
    (dict(rotary_dim=136), EUNSUPPORTED), (dict(rotary_dim=24, sections=(12,)), EUNSUPPORTED),
    (dict(num_pages=1 << 28), EUNSUPPORTED), (dict(num_tokens=1 << 31), EUNSUPPORTED), (dict(hq=0), EINVAL),
    (dict(query=None), EINVAL), (dict(query_out=None), EINVAL), (dict(key=None), EINVAL), (dict(v_scale=None), EINVAL),
    (dict(key=P + 2), EALIGN), (dict(key_out=P + 8), EALIGN), (dict(value_stride=1026), EALIGN),
    (dict(k_data=P + 1), EALIGN), (dict(num_tokens=8192, num_pages=1024), EWORKSPACE),
    (dict(num_tokens=8192, num_pages=1024, workspace=P, workspace_bytes=8), EWORKSPACE),
])
def test_append_status(kw, status):
    assert _append(**kw) == status


def test_append_of_no_tokens_is_done_at_once():
    assert _append(num_tokens=0, key=None, value=None, slots=None) == 0


def test_append_workspace():
    """None for batches that are validated without a bitmap, a bit a slot for the others."""
    need = lib.iris_b200_mrope_append_workspace_bytes
    for tokens in (0, 1, 128, 129, 2048):
        assert need(tokens, 1 << 20, 16) == 0
    for tokens in (2049, 1 << 20):
        assert need(tokens, 1000, 16) == 1000 * 16 // 8
    assert need(4096, 0, 16) == 0


def _gather(**kw):
    a = dict(k_data=P, v_data=P, k_scale=P, v_scale=P, block_table=P, stride=4, cu=P, first=None, key=P, value=P,
             num_tokens=8, batch=2, hkv=8, head_dim=128, num_pages=4, page_size=16, max_pages_per_seq=4,
             dtype=_lib.DTYPE_BF16, error=P, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.iris_b200_int4_paged_gather(*a.values())


@pytest.mark.parametrize("kw, status", [
    (dict(num_tokens=-1), EINVAL), (dict(hkv=0), EINVAL), (dict(page_size=0), EINVAL), (dict(dtype=7), EINVAL),
    (dict(batch=0), EINVAL), (dict(head_dim=48), EUNSUPPORTED), (dict(head_dim=544), EUNSUPPORTED),
    (dict(hkv=1 << 20), EUNSUPPORTED), (dict(cu=None), EINVAL), (dict(value=None), EINVAL), (dict(key=P + 8), EALIGN),
    (dict(v_data=P + 2), EALIGN), (dict(k_scale=P + 1), EALIGN),
])
def test_gather_status(kw, status):
    assert _gather(**kw) == status


def _bounds(**kw):
    a = dict(k_data=P, k_scale=P, block_table=P, stride=4, seq_lens=P, first=None, bounds=P, step=P, values=None,
             batch=2, hkv=8, head_dim=128, num_pages=4, page_size=16, max_pages_per_seq=4, error=P, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.iris_b200_int4_page_bounds(*a.values())


@pytest.mark.parametrize("kw, status", [
    (dict(batch=-1), EINVAL), (dict(page_size=32), EUNSUPPORTED), (dict(head_dim=256), EUNSUPPORTED),
    (dict(num_pages=0), EINVAL), (dict(batch=65536), EUNSUPPORTED), (dict(bounds=None), EINVAL),
    (dict(bounds=P + 8), EALIGN), (dict(values=P + 8), EALIGN), (dict(step=P + 2), EALIGN), (dict(k_data=P + 4), EALIGN),
])
def test_bounds_status(kw, status):
    assert _bounds(**kw) == status


def _select(**kw):
    a = dict(query=P, bounds=P, step=P, block_table=P, stride=64, seq_lens=P, page_list=P, page_count=P, batch=2, hq=32,
             hkv=8, head_dim=128, num_pages=128, page_size=16, max_pages_per_seq=64, max_pages=8, sink=1, recent=1,
             dtype=_lib.DTYPE_FP16, workspace=P, workspace_bytes=1 << 20, error=P, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.iris_b200_page_select(*a.values())


@pytest.mark.parametrize("kw, status", [
    (dict(batch=-1), EINVAL), (dict(hq=33), EINVAL), (dict(max_pages=0), EINVAL), (dict(sink=5, recent=4), EINVAL),
    (dict(sink=(1 << 31) - 1, recent=(1 << 31) - 1), EINVAL), (dict(sink=-1), EINVAL), (dict(dtype=5), EINVAL),
    (dict(hq=136), EUNSUPPORTED), (dict(head_dim=96), EUNSUPPORTED), (dict(hq=1024, hkv=1024), EUNSUPPORTED),
    (dict(num_pages=0), EINVAL), (dict(page_list=None), EINVAL), (dict(query=P + 2), EALIGN),
    (dict(workspace=None), EWORKSPACE), (dict(workspace_bytes=64), EWORKSPACE), (dict(workspace=P + 4), EALIGN),
])
def test_select_status(kw, status):
    assert _select(**kw) == status


def test_select_workspace_holds_a_score_per_page():
    assert lib.iris_b200_page_select_workspace_bytes(0, 8, 64) == 0
    for batch, hkv, pages in ((1, 1, 1), (3, 8, 257), (64, 8, 8192)):
        assert lib.iris_b200_page_select_workspace_bytes(batch, hkv, pages) >= 4 * batch * hkv * pages


def _sparse(**kw):
    a = dict(query=P, k_data=P, v_data=P, k_scale=P, v_scale=P, block_table=P, stride=64, seq_lens=P, page_list=P,
             page_count=P, output=P, lse=None, batch=2, hq=32, hkv=8, head_dim=128, num_pages=128, page_size=16,
             max_pages_per_seq=64, max_pages=8, scale=0.1, dtype=_lib.DTYPE_FP16, workspace=P, workspace_bytes=1 << 30,
             error=P, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.iris_b200_int4_sparse_paged_decode(*a.values())


@pytest.mark.parametrize("kw, status", [
    (dict(batch=-1), EINVAL), (dict(hq=33), EINVAL), (dict(max_pages=0), EINVAL), (dict(scale=0.0), EINVAL),
    (dict(scale=float("nan")), EINVAL), (dict(dtype=5), EINVAL), (dict(page_size=8), EUNSUPPORTED),
    (dict(head_dim=32), EUNSUPPORTED), (dict(hq=136), EUNSUPPORTED),
    (dict(batch=1 << 16, max_pages=1 << 12), EUNSUPPORTED), (dict(num_pages=0), EINVAL), (dict(output=None), EINVAL),
    (dict(query=P + 8), EALIGN), (dict(k_scale=P + 2), EALIGN), (dict(workspace=P + 8), EALIGN), (dict(lse=P + 2), EALIGN),
])
def test_sparse_decode_status(kw, status):
    assert _sparse(**kw) == status


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-CUDA error path")
def test_wrappers_require_cuda():
    from iris_kernel.fused_kv import fused_int4_paged_gather, fused_mrope_int4_paged_append
    from iris_kernel.sparse_attention import (fused_int4_page_bounds, fused_int4_sparse_paged_decode_attention,
                                              fused_page_select)

    x = torch.zeros(1, 1, 64, dtype=torch.float16)
    data, scale = torch.zeros(1, 16, 1, 32, dtype=torch.uint8), torch.zeros(1, 16, 1, 2, dtype=torch.float16)
    one, table = torch.ones(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    rows = torch.zeros(1, 32, dtype=torch.float16)
    bounds, step = torch.zeros(1, 1, 2, 64, dtype=torch.int8), torch.zeros(1, 1)
    with pytest.raises(RuntimeError):
        fused_mrope_int4_paged_append(x, x, table, one, rows, rows, data, data, scale, scale, sections=(32,),
                                      rotary_dim=64, page_size=16)
    with pytest.raises(RuntimeError):
        fused_int4_paged_gather(data, data, scale, scale, table, torch.tensor([0, 1], dtype=torch.int32), num_tokens=1)
    with pytest.raises(RuntimeError):
        fused_int4_page_bounds(data, scale, table, one, bounds, step)
    with pytest.raises(RuntimeError):
        fused_page_select(x, bounds, step, table, one, max_pages=2)
    with pytest.raises(RuntimeError):
        fused_int4_sparse_paged_decode_attention(x, data, data, scale, scale, table, one, table.view(1, 1, 1), table)
