"""One layer's decode step as a single CUDA-graph replay.

A serving loop runs, per layer and step, the append of the new tokens' K/V
followed by the decode over the updated cache.  :class:`DecodeStep` captures
those two calls (five kernels) once and replays them, so a step costs one
graph launch instead of the Python and launch overhead of each call.
:class:`SparseDecodeStep` is the same for decode over selected pages,
:class:`BudgetDecodeStep` for a cache that is kept to a budget.  The
cache, block table, lengths and RoPE tables are bound when the step is built
(their contents may change between replays, their storage may not); the
per-step inputs go through static buffers.

Validation inside the graph is deferred: a replay never reads the error word
on the host.  ``step(..., check=True)`` (or ``iris_kernel.check_errors()``
later) raises what the kernels recorded; a batch the append check rejects is
not written.
"""
from __future__ import annotations

import torch

from . import _runtime
from .fused_attention import fused_int4_paged_decode_attention
from .fused_kv import fused_int4_paged_evict, fused_mrope_int4_paged_append, fused_rope_int4_paged_append
from .sparse_attention import (fused_int4_page_bounds, fused_int4_sparse_paged_decode_attention,
                               fused_page_select)
from .varlen_attention import fused_int4_paged_attention_mass, fused_int4_paged_varlen_attention


def _capture(graph, dev, calls):
    """Runs ``calls`` once (launch shapes, scratch buffers), then captures it."""
    mode = _runtime.validation_mode()
    _runtime.set_validation_mode("deferred")
    try:
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            calls()
        torch.cuda.current_stream(dev).wait_stream(side)
        torch.cuda.synchronize(dev)
        with torch.cuda.graph(graph, stream=side):
            calls()
        torch.cuda.synchronize(dev)
    finally:
        _runtime.set_validation_mode(mode)


class DecodeStep:
    def __init__(self, k_data, v_data, k_scale, v_scale, block_table, seq_lens, cos_cache, sin_cache, *,
                 num_q_heads: int, new_tokens: int, rotary_dim: int, page_size: int = 16, group_size: int = 32,
                 softmax_scale: float | None = None):
        dev = k_data.device
        batch = block_table.shape[0]
        num_kv_heads, head_dim = k_data.shape[2], k_data.shape[3] * 2
        self.cache = (k_data, v_data, k_scale, v_scale)
        self.block_table, self.seq_lens = block_table, seq_lens
        self.cos, self.sin = cos_cache, sin_cache
        self.kw_append = dict(rotary_dim=rotary_dim, group_size=group_size, page_size=page_size)
        self.kw_decode = dict(page_size=page_size, group_size=group_size, softmax_scale=softmax_scale)
        self.query = torch.zeros((batch, num_q_heads, head_dim), dtype=torch.float16, device=dev)
        self.key = torch.zeros((new_tokens, num_kv_heads, head_dim), dtype=torch.float16, device=dev)
        self.value = torch.zeros_like(self.key)
        self.positions = torch.zeros(new_tokens, dtype=torch.int32, device=dev)
        self.slots = torch.full((new_tokens,), -1, dtype=torch.int32, device=dev)  # warm-up writes nothing
        self.output = torch.empty_like(self.query)
        self.graph = torch.cuda.CUDAGraph()
        _capture(self.graph, dev, self._calls)

    def _calls(self):
        fused_rope_int4_paged_append(self.key, self.value, self.positions, self.slots, self.cos, self.sin,
                                     *self.cache, **self.kw_append)
        fused_int4_paged_decode_attention(self.query, *self.cache, self.block_table, self.seq_lens, self.output,
                                          **self.kw_decode)

    def __call__(self, query, key, value, positions, slots, *, check: bool = False) -> torch.Tensor:
        """Append ``key/value [T, Hkv, D]`` at ``positions``/``slots [T]`` and
        decode ``query [B, Hq, D]``; returns the step's output (a static
        buffer, overwritten by the next replay)."""
        self.query.copy_(query, non_blocking=True)
        self.key.copy_(key, non_blocking=True)
        self.value.copy_(value, non_blocking=True)
        self.positions.copy_(positions, non_blocking=True)
        self.slots.copy_(slots, non_blocking=True)
        self.graph.replay()
        if check:
            _runtime.check_errors(self.query.device)
        return self.output


class SparseDecodeStep:
    """One layer's sparse decode step as a single CUDA-graph replay: the new
    tokens' multi-axis rotary append (queries rotated in the same launch), the
    bounds of their pages, the selection of pages, and the attention over them.

    One new token per sequence.  The cache, its bounds, the block table, the
    lengths (which count the new token) and the rotary tables are bound when
    the step is built; the bounds have to hold the pages that are cached by
    then (:func:`iris_kernel.sparse_attention.fused_int4_page_bounds` after the
    prefill).  ``recent_pages`` is at least 1, so that the new token's page is
    always attended to.  A sequence of length 0 is an idle row of the batch:
    give it slot -1, its output is 0."""

    def __init__(self, k_data, v_data, k_scale, v_scale, bounds, bounds_step, block_table, seq_lens, cos_cache,
                 sin_cache, *, num_q_heads: int, sections: tuple, rotary_dim: int, max_pages: int,
                 interleaved: bool = False, sink_pages: int = 1, recent_pages: int = 1, page_size: int = 16,
                 group_size: int = 32, softmax_scale: float | None = None):
        if recent_pages < 1:
            raise ValueError("recent_pages must be at least 1")
        dev, dtype = k_data.device, cos_cache.dtype
        batch = block_table.shape[0]
        num_kv_heads, head_dim = k_data.shape[2], k_data.shape[3] * 2
        self.cache = (k_data, v_data, k_scale, v_scale)
        self.bounds, self.bounds_step = bounds, bounds_step
        self.block_table, self.seq_lens = block_table, seq_lens
        self.cos, self.sin = cos_cache, sin_cache
        self.kw_append = dict(sections=tuple(sections), rotary_dim=rotary_dim, interleaved=interleaved,
                              group_size=group_size, page_size=page_size)
        self.kw_select = dict(max_pages=max_pages, sink_pages=sink_pages, recent_pages=recent_pages,
                              page_size=page_size)
        self.kw_attend = dict(page_size=page_size, group_size=group_size, softmax_scale=softmax_scale)
        self.query = torch.zeros((batch, num_q_heads, head_dim), dtype=dtype, device=dev)
        self.key = torch.zeros((batch, num_kv_heads, head_dim), dtype=dtype, device=dev)
        self.value = torch.zeros_like(self.key)
        self.positions = torch.zeros((len(self.kw_append["sections"]), batch), dtype=torch.int32, device=dev)
        self.slots = torch.full((batch,), -1, dtype=torch.int32, device=dev)  # warm-up writes nothing
        self.first = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.rotated = torch.empty_like(self.query)
        self.page_list = torch.empty((batch, num_kv_heads, max_pages), dtype=torch.int32, device=dev)
        self.page_count = torch.empty((batch, num_kv_heads), dtype=torch.int32, device=dev)
        self.output = torch.empty_like(self.query)
        self.graph = torch.cuda.CUDAGraph()
        _capture(self.graph, dev, self._calls)

    def _calls(self):
        fused_mrope_int4_paged_append(self.key, self.value, self.positions, self.slots, self.cos, self.sin,
                                      *self.cache, self.query, query_out=self.rotated, **self.kw_append)
        torch.sub(self.seq_lens, 1, out=self.first)
        fused_int4_page_bounds(self.cache[0], self.cache[2], self.block_table, self.seq_lens, self.bounds,
                               self.bounds_step, first_token=self.first, page_size=self.kw_select["page_size"])
        fused_page_select(self.rotated, self.bounds, self.bounds_step, self.block_table, self.seq_lens,
                          self.page_list, self.page_count, **self.kw_select)
        fused_int4_sparse_paged_decode_attention(self.rotated, *self.cache, self.block_table, self.seq_lens,
                                                 self.page_list, self.page_count, self.output, **self.kw_attend)

    def __call__(self, query, key, value, positions, slots, *, check: bool = False) -> torch.Tensor:
        """Append ``key / value [B, Hkv, D]`` at ``positions [A, B]`` / ``slots
        [B]`` and attend with ``query [B, Hq, D]`` (not rotated yet); returns
        the step's output (a static buffer, overwritten by the next replay)."""
        self.query.copy_(query, non_blocking=True)
        self.key.copy_(key, non_blocking=True)
        self.value.copy_(value, non_blocking=True)
        self.positions.copy_(positions, non_blocking=True)
        self.slots.copy_(slots, non_blocking=True)
        self.graph.replay()
        if check:
            _runtime.check_errors(self.query.device)
        return self.output


class BudgetDecodeStep:
    """One layer's decode step over a cache that is kept to a budget, as a
    single CUDA-graph replay: the new tokens' multi-axis rotary append (queries
    rotated in the same launch), the attention over the cache, the weights that
    it gave added to ``mass [pages, Hkv, 16]``, and the eviction of what is over
    ``budget`` tokens in every sequence.

    One new token per sequence.  The cache, the weights, the block table, the
    lengths and the rotary tables are bound when the step is built.  ``seq_lens``
    counts the new token before a step and is ``min(seq_lens, budget)`` after it,
    which is also the place of the next token; positions go on as ever (keys
    carry their rotation).  Tables need room for ``budget + 1`` tokens.  A
    sequence of length 0 is an idle row of the batch: give it slot -1.  ``decay``
    forgets old weights; ``logit_cap``, ``slopes`` and ``window`` are the
    attention's (the latter two by place in the cache)."""

    def __init__(self, k_data, v_data, k_scale, v_scale, mass, block_table, seq_lens, cos_cache, sin_cache, *,
                 num_q_heads: int, sections: tuple, rotary_dim: int, budget: int, sink_tokens: int = 4,
                 recent_tokens: int = 64, decay: float = 1.0, interleaved: bool = False, logit_cap: float = 0.0,
                 slopes=None, window: int = 0, page_size: int = 16, group_size: int = 32,
                 softmax_scale: float | None = None):
        dev, dtype = k_data.device, cos_cache.dtype
        batch = block_table.shape[0]
        num_kv_heads, head_dim = k_data.shape[2], k_data.shape[3] * 2
        self.cache, self.mass = (k_data, v_data, k_scale, v_scale), mass
        self.block_table, self.seq_lens = block_table, seq_lens
        self.cos, self.sin = cos_cache, sin_cache
        self.kw_append = dict(sections=tuple(sections), rotary_dim=rotary_dim, interleaved=interleaved,
                              group_size=group_size, page_size=page_size)
        self.kw_attend = dict(page_size=page_size, group_size=group_size, softmax_scale=softmax_scale,
                              logit_cap=logit_cap, slopes=slopes, window=window)
        self.kw_evict = dict(budget=budget, sink_tokens=sink_tokens, recent_tokens=recent_tokens, page_size=page_size,
                             group_size=group_size)
        self.decay = decay
        self.query = torch.zeros((batch, num_q_heads, head_dim), dtype=dtype, device=dev)
        self.key = torch.zeros((batch, num_kv_heads, head_dim), dtype=dtype, device=dev)
        self.value = torch.zeros_like(self.key)
        self.positions = torch.zeros((len(self.kw_append["sections"]), batch), dtype=torch.int32, device=dev)
        self.slots = torch.full((batch,), -1, dtype=torch.int32, device=dev)
        self.first = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.new_lens = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.rotated = torch.empty_like(self.query)
        self.output = torch.empty_like(self.query)
        self.graph = torch.cuda.CUDAGraph()
        # the warm-up sees no tokens: it changes neither the cache nor its weights
        lens = seq_lens.clone()
        seq_lens.zero_()
        try:
            _capture(self.graph, dev, self._calls)
        finally:
            seq_lens.copy_(lens)

    def _calls(self):
        fused_mrope_int4_paged_append(self.key, self.value, self.positions, self.slots, self.cos, self.sin,
                                      *self.cache, self.query, query_out=self.rotated, **self.kw_append)
        _, lse = fused_int4_paged_varlen_attention(self.rotated, *self.cache, self.block_table, self.seq_lens, None,
                                                   self.output, return_lse=True, **self.kw_attend)
        torch.sub(self.seq_lens, 1, out=self.first)
        fused_int4_paged_attention_mass(self.rotated, lse, self.cache[0], self.cache[2], self.block_table,
                                        self.seq_lens, self.mass, first_token=self.first, decay=self.decay,
                                        **self.kw_attend)
        fused_int4_paged_evict(*self.cache, self.mass, self.block_table, self.seq_lens, self.new_lens, **self.kw_evict)
        self.seq_lens.copy_(self.new_lens)

    def __call__(self, query, key, value, positions, slots, *, check: bool = False) -> torch.Tensor:
        """Append ``key / value [B, Hkv, D]`` at ``positions [A, B]`` / ``slots
        [B]`` and attend with ``query [B, Hq, D]`` (not rotated yet); returns
        the step's output (a static buffer, overwritten by the next replay)."""
        self.query.copy_(query, non_blocking=True)
        self.key.copy_(key, non_blocking=True)
        self.value.copy_(value, non_blocking=True)
        self.positions.copy_(positions, non_blocking=True)
        self.slots.copy_(slots, non_blocking=True)
        self.graph.replay()
        if check:
            _runtime.check_errors(self.query.device)
        return self.output
