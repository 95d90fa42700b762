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
argument checks, outputs and calls are in csrc/bindings.cpp, data-dependent
errors go through the device error word (see ``_runtime``).
"""
from __future__ import annotations

import torch

from . import _runtime


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
    _runtime.ops().page_bounds(k_data, k_scale, block_table, seq_lens, bounds, bounds_step, first_token, values,
                               page_size, group_size)
    _runtime.finish(k_data)


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
    out = _runtime.ops().page_select(query, bounds, bounds_step, block_table, seq_lens, page_list, page_count,
                                     max_pages, sink_pages, recent_pages, page_size)
    _runtime.finish(query)
    return out


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
    ``softmax_scale`` None (or 0.0) means ``D ** -0.5``; a negative one is
    refused with a RuntimeError.  ``output`` may be the query itself."""
    out = _runtime.ops().sparse_decode(query, k_data, v_data, k_scale, v_scale, block_table, seq_lens, page_list,
                                       page_count, output, page_size, group_size, softmax_scale, return_lse)
    _runtime.finish(query)
    return out
