"""Plain CPU implementations, in 64 bits, of attention over new tokens, of the
weights it gives to cached tokens, and of eviction; and how far the kernels may
be from them.

Half a step of a rounding: fp16 2^-11, bf16 2^-8 of the value (`half_step`).

* Attention.  Keys enter the products exactly, as do queries; a logit is off by
  what fp32 sums lose: at most 32 steps of the tensor cores, each with 2^-23 of the
  running sum, so 2^-18 of sum_d |q_d k_jd| * scale (the cap and the bias do not
  make it more, and round with 2^-22 of their own size, which that covers or the
  2^-18 below); the largest over the visible tokens is delta.  Weights move by a
  factor of e^(2 delta) at most, each is rounded to fp16 (2^-11 of it, or 2^-25 of
  1/256 of the largest where it is tiny), and so is the value, nibble * scale.  The
  output is then rounded to its type.
* lse: delta / ln 2, and 2^-18 of its size and of 1 for fp32.
* Weights (mass): keys are exact there; a logit is off by 2^-20 of sum |q k| *
  scale and of its own size and the lse's; each weight by e to that, sums of
  fp32 by 2^-20 of the sum.  Each of a token's weights below 2^-126 may count as
  0 (the exponential flushes what fp32 holds with fewer bits), one a row and
  query head of the group.
"""
from __future__ import annotations

import math

import numpy as np
import torch

import _sparse_refs as R

PAGE = 16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def table(rng, lens, width=None, spare=2):
    """Scattered disjoint pages; columns past the end are never read."""
    counts = [-(-n // PAGE) for n in lens]
    ids = rng.permutation(sum(counts) + spare).astype(np.int32)
    bt = np.full((len(lens), width or max(1, max(counts))), -3, np.int32)
    at = 0
    for b, n in enumerate(counts):
        bt[b, :n] = ids[at:at + n]
        at += n
    return bt, sum(counts) + spare


def visible(pos, first, prefix, window, length):
    """[rows, length] truth values."""
    j = np.arange(length)[None]
    pos, first = np.asarray(pos)[:, None], np.asarray(first)[:, None]
    seen = j <= pos
    if window:
        seen &= j > pos - window
    seen |= j < prefix
    return seen & (j >= first)


def _sequence(query, cache, bt, lens, cu, b, h, *, scale, logit_cap, slopes, window, prefix_lens, first_visible):
    """Logits [group, rows, tokens] of KV head h's query heads (-inf: not visible), and sum |q k| * scale of each."""
    n, r0, r1 = int(lens[b]), int(cu[b]), int(cu[b + 1])
    hkv, dim = cache[0].shape[2], query.shape[2]
    group = query.shape[1] // hkv
    j = np.arange(n)
    pages = bt[b, j // PAGE]
    key = R.dequant(cache[0][pages, j % PAGE, h], cache[2][pages, j % PAGE, h], np.float64)
    q = query[r0:r1, h * group:(h + 1) * group].astype(np.float64).transpose(1, 0, 2)
    scale = dim ** -0.5 if scale is None else scale
    with np.errstate(all="ignore"):
        x = q @ key.T * scale
        size = np.abs(q) @ np.abs(key).T * scale
        if logit_cap:
            x = logit_cap * np.tanh(x / logit_cap)
    pos = n - (r1 - r0) + np.arange(r1 - r0)
    if slopes is not None:
        x = x - slopes[h * group:(h + 1) * group, None, None].astype(np.float64) * np.abs(pos[:, None] - j)
    seen = visible(pos, np.zeros(r1 - r0) if first_visible is None else first_visible[r0:r1],
                   0 if prefix_lens is None else int(prefix_lens[b]), window, n)
    return np.where(seen, x, -np.inf), np.where(seen, size, 0.0), seen


def _options(kw):
    return dict(dict(scale=None, logit_cap=0.0, slopes=None, window=0, prefix_lens=None, first_visible=None), **kw)


def attend_ref(query, cache, bt, lens, cu, dtype, **kw):
    """(output, lse, how far the output may be off, and the lse)."""
    kw = _options(kw)
    t, hq, dim = query.shape
    hkv = cache[0].shape[2]
    group = hq // hkv
    out, far = np.zeros((t, hq, dim)), np.zeros((t, hq, dim))
    lse, lse_far = np.full((t, hq), -np.inf), np.zeros((t, hq))
    half = half_step(torch.float16)
    for b, n in enumerate(lens):
        r0, r1 = int(cu[b]), int(cu[b + 1])
        if n <= 0 or r1 == r0:
            continue
        j = np.arange(n)
        pages = bt[b, j // PAGE]
        for h in range(hkv):
            x, size, seen = _sequence(query, cache, bt, lens, cu, b, h, **kw)
            value = R.dequant(cache[1][pages, j % PAGE, h], cache[3][pages, j % PAGE, h], np.float64)
            value = np.where(seen.any(0)[:, None], value, 0.0)
            with np.errstate(all="ignore"):
                top = x.max(-1, keepdims=True)
                top = np.where(top == -np.inf, 0.0, top)
                p = np.where(seen, np.exp(x - top), 0.0)
                total = p.sum(-1, keepdims=True)
                w = p / np.where(total == 0, 1.0, total)
                bad = ~np.isfinite(value)
                o = w @ np.where(bad, 0.0, value)
                hit = (seen.astype(float) @ bad.astype(float)) > 0  # [rows, dims]
                o = np.where(hit[None], np.nan, o)
                delta = size.max(-1, keepdims=True) * 2.0 ** -18
                most = np.abs(w) @ np.abs(np.where(bad, 0.0, value))
                big = np.abs(np.where(bad, 0.0, value)).max()
                f = most * (np.expm1(2 * delta) + 2 * half + 2.0 ** -18) + n * 2.0 ** -33 * big / np.maximum(total, 1.0)
                f = f + np.abs(o) * half_step(dtype) + 2.0 ** -25
                s = (top + np.log(total))[..., 0] / math.log(2.0)
                rows = slice(h * group, (h + 1) * group)
                out[r0:r1, rows], far[r0:r1, rows] = o.transpose(1, 0, 2), f.transpose(1, 0, 2)
                lse[r0:r1, rows] = s.T
                lse_far[r0:r1, rows] = (delta[..., 0] / math.log(2.0) + 2.0 ** -18 * (1 + np.abs(s))).T
    return out, lse, far, lse_far


def mass_ref(query, lse, cache, bt, lens, cu, mass, first_token, decay, **kw):
    """(the weights [pages, Hkv, 16] afterwards, how far they may be off)."""
    kw = _options(kw)
    hkv = cache[0].shape[2]
    group = query.shape[1] // hkv
    out, far = mass.astype(np.float64).copy(), np.zeros(mass.shape)
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        r0, r1 = int(cu[b]), int(cu[b + 1])
        j = np.arange(n)
        pages = bt[b, j // PAGE]
        for h in range(hkv):
            before = out[pages, h, j % PAGE] * decay
            before[(0 if first_token is None else int(first_token[b])):] = 0.0
            x, size, seen = _sequence(query, cache, bt, lens, cu, b, h, **kw)
            y = lse[r0:r1, h * group:(h + 1) * group].astype(np.float64).T[..., None] * math.log(2.0)
            with np.errstate(all="ignore"):
                w = np.where(seen, np.exp(np.minimum(x - y, 0.0)), 0.0)  # a weight is at most 1
                e = np.where(seen, np.expm1(2.0 ** -20 * (1 + size + np.abs(x) + np.abs(y))), 0.0)
                out[pages, h, j % PAGE] = before + w.sum((0, 1))
                far[pages, h, j % PAGE] = (w * e).sum((0, 1)) + 2.0 ** -20 * np.abs(out[pages, h, j % PAGE]) + w.shape[0] * w.shape[1] * 2.0 ** -126
    return out, far


def evict_ref(cache, mass, bt, lens, budget, sink, recent):
    """Moves the rows in place; (new lengths, kept [B, Hkv, budget])."""
    hkv = mass.shape[1]
    kept = np.full((len(lens), hkv, budget), -1, np.int32)
    heavy = budget - recent
    for b, n in enumerate(lens):
        n = int(n)
        if n <= budget:
            kept[b, :, :max(n, 0)] = np.arange(max(n, 0))
            continue
        j = np.arange(n)
        pages = bt[b, j // PAGE]
        for h in range(hkv):
            w = mass[pages, h, j % PAGE].astype(np.float64)
            w = np.where(np.isnan(w), np.inf, w)
            best = set(sorted(range(sink, n - recent), key=lambda i: (-w[i], i))[:heavy - sink])
            late = iter(sorted(i for i in best if i >= heavy))
            place = list(range(sink)) + [i if i in best else next(late) for i in range(sink, heavy)]
            place = np.array(place + list(range(n - recent, n)), np.int64)
            kept[b, h] = place
            src, dst = (pages[place], place % PAGE), (pages[:budget], np.arange(budget) % PAGE)
            for x in cache:
                x[dst[0], dst[1], h] = x[src[0], src[1], h]
            mass[dst[0], h, dst[1]] = mass[src[0], h, src[1]]
    return np.minimum(np.asarray(lens), budget).astype(np.int32), kept
