"""Attention of new tokens over the INT4 paged cache: whole prompts, chunks of
prompts, drafts of a few tokens, single tokens (none of it has a counterpart in
the reference).

The new tokens' keys and values are in the cache already
(:func:`iris_kernel.fused_kv.fused_mrope_int4_paged_append` or
:func:`iris_kernel.fused_kv.fused_rope_int4_paged_append`): sequence ``b``
counts ``seq_lens[b]`` cached tokens, of which its rows of the query are the
last.  Row ``i`` of ``n`` is at place ``pos = seq_lens[b] - n + i``.  The kernel
is csrc/varlen_attention.cu; argument checks, outputs and calls are in
csrc/bindings.cpp, data-dependent errors go through the device error word (see
``_runtime``).
"""
from __future__ import annotations

import torch

from . import _runtime


def fused_int4_paged_varlen_attention(
    query: torch.Tensor,
    k_data: torch.Tensor,
    v_data: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    output: torch.Tensor | None = None,
    *,
    page_size: int = 16,
    group_size: int = 32,
    softmax_scale: float | None = None,
    logit_cap: float = 0.0,
    slopes: torch.Tensor | None = None,
    window: int = 0,
    prefix_lens: torch.Tensor | None = None,
    first_visible: torch.Tensor | None = None,
    return_lse: bool = False,
):
    """Causal attention of ``query [T, Hq, D]`` (FP16 or BF16) over the cache.

    Sequence ``b`` has the rows ``cu_seqlens[b] .. cu_seqlens[b + 1]`` (int32
    ``[B + 1]``, rising from 0); None means one row a sequence, a decode step.
    Rows behind ``cu_seqlens[B]`` belong to none: output 0, lse -inf.

    The logit of a row at place ``pos`` and cached token ``j`` is
    ``softmax_scale * q.k``, capped to ``logit_cap * tanh(logit / logit_cap)``
    if ``logit_cap`` is not 0, less ``slopes[head] * |pos - j|`` (fp32 ``[Hq]``)
    if given.  A row sees token ``j`` of its sequence if ``j >=
    first_visible[row]`` (int32 ``[T]``: its document's first token, say) and
    either ``j < prefix_lens[b]`` (int32 ``[B]``: tokens that all rows see, also
    earlier ones and those that the window has left behind) or ``j <= pos`` and,
    with a ``window``, ``j > pos - window``.  A row that sees nothing has output
    0 and lse -inf; so has a sequence of length 0 (an idle row of the batch).

    Returns the output in the query's type, or ``(output, lse)`` with
    ``return_lse``: fp32 ``[T, Hq]``, log2-sum-exp2 of the logits, as
    :func:`fused_int4_paged_attention_mass` wants it.  ``softmax_scale`` None
    (or 0.0) means ``D ** -0.5``.  ``query`` may be a slice of a fused
    projection; ``output`` may be the query itself where that is dense."""
    out = _runtime.ops().varlen_attention(query, k_data, v_data, k_scale, v_scale, block_table, seq_lens, cu_seqlens,
                                          output, page_size, group_size, softmax_scale, logit_cap, slopes, window,
                                          prefix_lens, first_visible, return_lse)
    _runtime.finish(query)
    return out


def fused_int4_paged_attention_mass(
    query: torch.Tensor,
    lse: torch.Tensor,
    k_data: torch.Tensor,
    k_scale: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    mass: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    *,
    first_token: torch.Tensor | None = None,
    decay: float = 1.0,
    page_size: int = 16,
    group_size: int = 32,
    softmax_scale: float | None = None,
    logit_cap: float = 0.0,
    slopes: torch.Tensor | None = None,
    window: int = 0,
    prefix_lens: torch.Tensor | None = None,
    first_visible: torch.Tensor | None = None,
) -> None:
    """Adds to ``mass [pages, Hkv, 16]`` (fp32, in place) the attention weight
    that each cached token got from the query rows, summed over a KV head's
    query heads: what :func:`iris_kernel.fused_kv.fused_int4_paged_evict` goes
    by.

    ``query`` may hold all rows of an attention call or, with offsets to match,
    the last ones of every sequence (a prompt's last 32 tokens, say); ``lse
    [T, Hq]`` is what :func:`fused_int4_paged_varlen_attention` returned for
    them, and the other arguments are that call's.  Old weights are first
    multiplied by ``decay`` (0 to 1); tokens from ``first_token[b]`` on (int32
    ``[B]``; None: all) start from 0, as they must where their slots held other
    tokens before: None after a prompt, ``seq_lens - 1`` after a decode step.

    The fast use is the last rows: up to 128 of them a KV head (32 new tokens
    with four query heads each) are loaded once, more again for every tile of
    128 cached tokens (all rows of a prompt of 4096 tokens take five times as
    long as its attention).

    A weight is at most 1; a row whose lse is -inf gives nothing.  A page must
    belong to one sequence only; tokens behind a bad page id get no weight
    written."""
    _runtime.ops().attention_mass(query, lse, k_data, k_scale, block_table, seq_lens, mass, cu_seqlens, first_token, decay,
                                  page_size, group_size, softmax_scale, logit_cap, slopes, window, prefix_lens,
                                  first_visible)
    _runtime.finish(query)
