"""Sparse read path: decode attention over the pages that a cheap score selects.

Three operators, in the order of a decode step (none has a counterpart in
the reference):

* :func:`fused_int4_page_bounds` keeps, per physical page and KV head, the
  lowest and the highest stored key of every dim, in 8 bits;
* :func:`fused_page_select` bounds with them, for every page, the largest
  logit that a query can find there, and lists the best pages per sequence and
  KV head;
* :func:`fused_int4_sparse_paged_decode_attention` attends to those pages.

The index costs 2 D + 4 bytes per page and head to read where the dense
decode reads 18 D, and the attention reads max_pages pages whatever the
context's length.  The kernels are csrc/page_index.cu and csrc/sparse_decode.cu;
data-dependent errors go through the device error word (see ``_runtime``).
"""
from __future__ import annotations

import torch

from . import _lib, _runtime

_PAGE = 16


def _check_shape(page_size, head_dim):
    if page_size != _PAGE:
        raise NotImplementedError("sparse decode currently supports page_size=16")
    if head_dim not in (64, 128):
        raise NotImplementedError("sparse decode currently supports head_dim in {64, 128}")


def _check_query(query, num_kv_heads):
    if query.ndim != 3:
        raise ValueError("query must have shape [B, Hq, D]")
    code = _runtime.dtype_code("query", query.dtype)
    if not query.is_contiguous():
        raise ValueError("query must be contiguous")
    hq = query.shape[1]
    if num_kv_heads == 0 or hq == 0 or hq % num_kv_heads != 0:
        raise ValueError("num_query_heads must be divisible by num_kv_heads")
    if hq // num_kv_heads > 16:
        raise NotImplementedError("sparse decode supports at most 16 query heads per KV head")
    if query.data_ptr() % 16 != 0:
        raise ValueError("query must start on a 16-byte boundary")
    return code


def fused_int4_page_bounds(
    k_data: torch.Tensor,
    k_scale: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    bounds: torch.Tensor,
    bounds_step: torch.Tensor,
    *,
    first_token: torch.Tensor | None = None,
    values: torch.Tensor | None = None,
    page_size: int = 16,
    group_size: int = 32,
) -> None:
    """Bounds of the stored keys, in place: ``bounds [pages, Hkv, 2, D]`` int8
    (lowest, highest) in units of ``bounds_step [pages, Hkv]`` fp32, rounded
    outwards.  Call it after an append with ``first_token [B]`` int32, the
    first position that the append wrote in each sequence: the pages from that
    token's to the last one are computed anew from the cache.  None means
    every page.  ``values [pages, Hkv, 2, D]`` fp16, if given, receives what
    the codes of those pages stand for (rounded to FP16), for a score of the
    caller's own."""
    device = _runtime.require_device("k_data", k_data)
    if group_size != 32:
        raise NotImplementedError("sparse decode currently supports group_size=32")
    if k_data.ndim != 4:
        raise ValueError("k_data must be a rank-4 tensor")
    num_pages, cache_page_size, num_kv_heads, packed_dim = k_data.shape
    head_dim = 2 * packed_dim
    _check_shape(page_size, head_dim)
    if cache_page_size != page_size or num_kv_heads == 0:
        raise ValueError("packed cache shape does not match page_size")
    check = _runtime.check_tensor
    check("k_data", k_data, (num_pages, page_size, num_kv_heads, packed_dim), torch.uint8, device)
    check("k_scale", k_scale, (num_pages, page_size, num_kv_heads, head_dim // 32), torch.float16, device)
    check("bounds", bounds, (num_pages, num_kv_heads, 2, head_dim), torch.int8, device)
    check("bounds_step", bounds_step, (num_pages, num_kv_heads), torch.float32, device)
    if values is not None:
        check("values", values, (num_pages, num_kv_heads, 2, head_dim), torch.float16, device)
    batch = block_table.shape[0]
    width, table_stride = _runtime.check_block_table(block_table, batch, device)
    check("seq_lens", seq_lens, (batch,), torch.int32, device)
    if first_token is not None:
        check("first_token", first_token, (batch,), torch.int32, device)
    if batch == 0:
        return
    if num_pages == 0:
        raise IndexError("block_table contains an invalid physical page id")
    _runtime.launch(
        _lib.lib.iris_b200_int4_page_bounds, "iris_b200_int4_page_bounds", device,
        k_data.data_ptr(), k_scale.data_ptr(), block_table.data_ptr(), table_stride, seq_lens.data_ptr(),
        None if first_token is None else first_token.data_ptr(), bounds.data_ptr(), bounds_step.data_ptr(),
        None if values is None else values.data_ptr(), batch, num_kv_heads, head_dim, num_pages, page_size,
        width)


def fused_page_select(
    query: torch.Tensor,
    bounds: torch.Tensor,
    bounds_step: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    page_list: torch.Tensor | None = None,
    page_count: torch.Tensor | None = None,
    *,
    max_pages: int,
    sink_pages: int = 1,
    recent_pages: int = 1,
    page_size: int = 16,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The pages each sequence and KV head should attend to: ``page_list [B,
    Hkv, max_pages]`` int32, logical pages in rising order with -1 behind the
    last, and ``page_count [B, Hkv]`` int32.

    A page's score is the largest product that any key within its bounds could
    have with any of the KV head's query heads (held in 8 bits; the sum is a
    whole number, so a selection does not depend on the order of additions).
    The first ``sink_pages`` and the last ``recent_pages`` are always kept and
    count among the ``max_pages``; ties go to the lowest page.  The last page's
    bounds need not be up to date while ``recent_pages >= 1``.  An empty
    sequence keeps no page."""
    device = _runtime.require_device("query", query)
    if bounds.ndim != 4 or bounds.shape[2] != 2:
        raise ValueError("bounds must have shape [pages, Hkv, 2, D]")
    num_pages, num_kv_heads, _, head_dim = bounds.shape
    code = _check_query(query, num_kv_heads)
    _check_shape(page_size, head_dim)
    batch, num_q_heads, query_dim = query.shape
    if query_dim != head_dim:
        raise ValueError("bounds do not match the query's head_dim")
    if max_pages <= 0 or sink_pages < 0 or recent_pages < 0 or sink_pages + recent_pages > max_pages:
        raise ValueError("max_pages must be positive and hold sink_pages and recent_pages")
    check = _runtime.check_tensor
    check("bounds", bounds, bounds.shape, torch.int8, device)
    check("bounds_step", bounds_step, (num_pages, num_kv_heads), torch.float32, device)
    width, table_stride = _runtime.check_block_table(block_table, batch, device)
    check("seq_lens", seq_lens, (batch,), torch.int32, device)
    if page_list is None:
        page_list = torch.empty((batch, num_kv_heads, max_pages), dtype=torch.int32, device=device)
    else:
        check("page_list", page_list, (batch, num_kv_heads, max_pages), torch.int32, device)
    if page_count is None:
        page_count = torch.empty((batch, num_kv_heads), dtype=torch.int32, device=device)
    else:
        check("page_count", page_count, (batch, num_kv_heads), torch.int32, device)
    if batch == 0:
        return page_list, page_count
    if num_pages == 0:
        raise IndexError("block_table contains an invalid physical page id")
    need = _runtime.workspace_bytes(_lib.lib.iris_b200_page_select_workspace_bytes, batch, num_kv_heads, width)
    ws = _runtime.scratch(device, _runtime.stream_ptr(device), "page_select", need)
    _runtime.launch(
        _lib.lib.iris_b200_page_select, "iris_b200_page_select", device,
        query.data_ptr(), bounds.data_ptr(), bounds_step.data_ptr(), block_table.data_ptr(), table_stride,
        seq_lens.data_ptr(), page_list.data_ptr(), page_count.data_ptr(), batch, num_q_heads, num_kv_heads, head_dim,
        num_pages, page_size, width, max_pages, sink_pages, recent_pages, code, ws.data_ptr(), ws.numel())
    return page_list, page_count


def fused_int4_sparse_paged_decode_attention(
    query: torch.Tensor,
    k_data: torch.Tensor,
    v_data: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    page_list: torch.Tensor,
    page_count: torch.Tensor,
    output: torch.Tensor | None = None,
    *,
    page_size: int = 16,
    group_size: int = 32,
    softmax_scale: float | None = None,
    return_lse: bool = False,
):
    """Decode attention of ``query [B, Hq, D]`` (FP16 or BF16) over the listed
    pages of the INT4 cache: KV head ``h`` of sequence ``b`` attends to the
    first ``page_count[b, h]`` pages of ``page_list [B, Hkv, K]`` (int32,
    logical, as :func:`fused_page_select` gives them).  Negative entries and
    pages past the sequence's end count for nothing, a page listed twice
    counts twice; without a token the output is 0.

    Returns the output in the query's type, or ``(output, lse)`` with
    ``return_lse``: fp32 ``[B, Hq]``, log2-sum-exp2 of the scaled logits (-inf
    without a token), to merge with attention over other tokens.
    ``softmax_scale`` None (or 0.0) means ``D ** -0.5``."""
    device = _runtime.require_device("query", query)
    if group_size != 32:
        raise NotImplementedError("sparse decode currently supports group_size=32")
    if k_data.ndim != 4:
        raise ValueError("k_data/v_data must have identical rank-4 shapes")
    num_pages, cache_page_size, num_kv_heads, packed_dim = k_data.shape
    head_dim = 2 * packed_dim
    code = _check_query(query, num_kv_heads)
    _check_shape(page_size, head_dim)
    batch, num_q_heads, query_dim = query.shape
    if cache_page_size != page_size or query_dim != head_dim:
        raise ValueError("packed cache shape does not match query/page_size")
    check = _runtime.check_tensor
    data, scale = (num_pages, page_size, num_kv_heads, packed_dim), (num_pages, page_size, num_kv_heads, head_dim // 32)
    check("k_data", k_data, data, torch.uint8, device)
    check("v_data", v_data, data, torch.uint8, device)
    check("k_scale", k_scale, scale, torch.float16, device)
    check("v_scale", v_scale, scale, torch.float16, device)
    width, table_stride = _runtime.check_block_table(block_table, batch, device)
    check("seq_lens", seq_lens, (batch,), torch.int32, device)
    if page_list.ndim != 3 or page_list.shape[2] == 0:
        raise ValueError("page_list must have shape [B, Hkv, max_pages], max_pages >= 1")
    max_pages = page_list.shape[2]
    check("page_list", page_list, (batch, num_kv_heads, max_pages), torch.int32, device)
    check("page_count", page_count, (batch, num_kv_heads), torch.int32, device)
    if output is None:
        output = torch.empty_like(query)
    else:
        check("output", output, (batch, num_q_heads, head_dim), query.dtype, device)
    lse = torch.empty((batch, num_q_heads), dtype=torch.float32, device=device) if return_lse else None
    if batch > 0:
        if num_pages == 0:
            raise IndexError("block_table contains an invalid physical page id")
        need = _runtime.workspace_bytes(_lib.lib.iris_b200_sparse_decode_workspace_bytes, batch, num_q_heads,
                                        num_kv_heads, head_dim, max_pages, device.index)
        ws = _runtime.scratch(device, _runtime.stream_ptr(device), "sparse_decode", need)
        factor = head_dim ** -0.5 if softmax_scale is None or softmax_scale == 0.0 else float(softmax_scale)
        _runtime.launch(
            _lib.lib.iris_b200_int4_sparse_paged_decode, "iris_b200_int4_sparse_paged_decode", device,
            query.data_ptr(), k_data.data_ptr(), v_data.data_ptr(), k_scale.data_ptr(),
            v_scale.data_ptr(), block_table.data_ptr(), table_stride, seq_lens.data_ptr(),
            page_list.data_ptr(), page_count.data_ptr(), output.data_ptr(), None if lse is None else lse.data_ptr(),
            batch, num_q_heads, num_kv_heads, head_dim, num_pages, page_size, width, max_pages, factor,
            code, ws.data_ptr(), ws.numel())
    return (output, lse) if return_lse else output
