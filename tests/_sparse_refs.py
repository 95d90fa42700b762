"""Plain CPU implementations of the sparse decode's operators, written from
their definitions: fp32 where the definition rounds to fp32 (quantisation,
bounds, scores: compared bit for bit), 64 bits for the attention."""
from __future__ import annotations

import math

import numpy as np
import torch

PAGE, GROUP = 16, 32
TINY, TOP = np.float32(2.0 ** -14), np.float32(65504.0)


def f32(t: torch.Tensor) -> np.ndarray:
    return t.detach().float().cpu().numpy()


def to_type(x: np.ndarray, dtype: torch.dtype) -> torch.Tensor:
    """fp32 -> the 16-bit type, rounded to nearest even."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(dtype)


def axis_map(sections, interleaved):
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while sum(left):
        for a in range(len(left)):
            if left[a] > 0:
                left[a] -= 1
                out.append(a)
    return out


def rotate(x, positions, cos, sin, sections, interleaved, rotary_dim):
    """[T, H, D] fp32 holding 16-bit values; products are exact in fp32."""
    half = rotary_dim // 2
    y = x.copy()
    for i, a in enumerate(axis_map(sections, interleaved)):
        c = cos[positions[a], i][:, None]
        s = sin[positions[a], i][:, None]
        y[..., i] = x[..., i] * c - x[..., i + half] * s
        y[..., i + half] = x[..., i + half] * c + x[..., i] * s
    return y


def quantise(x):
    """[.., D] fp32 -> (signed nibbles int8, fp16 scales)."""
    y = x.reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(all="ignore"):
        amax = np.abs(y).max(-1)  # NaN propagates
        scale = np.where(np.isfinite(amax), np.minimum(np.maximum(amax / np.float32(7), TINY), TOP), amax)
        scale = scale.astype(np.float16)
        q = np.clip(np.rint(y / scale.astype(np.float32)[..., None]), -7, 7)
    q = np.where(np.isfinite(scale)[..., None], q, 0).astype(np.int8)
    return q.reshape(x.shape), scale


def pack(q):
    return ((q[..., 0::2] & 15) | ((q[..., 1::2] & 15) << 4)).astype(np.uint8)


def unpack(data):
    q = np.empty((*data.shape[:-1], data.shape[-1] * 2), np.int8)
    q[..., 0::2] = ((data & 15) ^ 8).astype(np.int8) - 8
    q[..., 1::2] = ((data >> 4) ^ 8).astype(np.int8) - 8
    return q


def dequant(data, scale, dtype=np.float32):
    with np.errstate(all="ignore"):
        return unpack(data).astype(dtype) * np.repeat(scale.astype(dtype), GROUP, axis=-1)


def bounds_ref(k_data, k_scale, block_table, lens, first, bounds, step):
    """Updates numpy bounds / step in place."""
    for b, n in enumerate(lens):
        f = 0 if first is None else max(0, int(first[b]))
        for col in range(f // PAGE, -(-int(n) // PAGE)):
            page = block_table[b, col]
            tok = min(PAGE, int(n) - col * PAGE)
            key = dequant(k_data[page, :tok], k_scale[page, :tok])  # [tok, H, D]
            for h in range(key.shape[1]):
                if not np.isfinite(k_scale[page, :tok, h].astype(np.float32)).all():
                    step[page, h] = np.inf
                    bounds[page, h, 0], bounds[page, h, 1] = -127, 127
                    continue
                lo, hi = key[:, h].min(0), key[:, h].max(0)
                u = np.maximum(np.abs(lo), np.abs(hi)).max() / np.float32(127)
                step[page, h] = u
                if u == 0:
                    bounds[page, h] = 0
                else:
                    bounds[page, h, 0] = np.clip(np.floor(lo / u), -127, 127)
                    bounds[page, h, 1] = np.clip(np.ceil(hi / u), -127, 127)


def scores_ref(query, bounds, step, block_table, hkv):
    """[B, Hkv, width] fp32 scores."""
    B, hq, _ = query.shape
    G = hq // hkv
    out = np.empty((B, hkv, block_table.shape[1]), np.float32)
    with np.errstate(all="ignore"):
        for b in range(B):
            page = block_table[b]
            for h in range(hkv):
                q = query[b, h * G:(h + 1) * G]
                amax = np.abs(q).max(-1)
                unit = np.where(np.isfinite(amax), amax / np.float32(127), np.float32(0)).astype(np.float32)
                code = np.where(unit[:, None] > 0, np.clip(np.rint(q / unit[:, None]), -127, 127), 0).astype(np.int64)
                lo, hi = bounds[page, h, 0].astype(np.int64), bounds[page, h, 1].astype(np.int64)
                s = np.minimum(code, 0) @ lo.T + np.maximum(code, 0) @ hi.T  # [G, width]
                u = step[page, h]
                v = (s.astype(np.float32) * u[None]) * unit[:, None]
                out[b, h] = np.where(np.isfinite(u), v.max(0), np.float32(np.inf))
    return out


def select_ref(scores, lens, max_pages, sink, recent):
    B, hkv, width = scores.shape
    lists = np.full((B, hkv, max_pages), -1, np.int32)
    counts = np.zeros((B, hkv), np.int32)
    for b in range(B):
        n = min(width, max(0, -(-int(lens[b]) // PAGE)))
        for h in range(hkv):
            if n <= max_pages:
                keep = list(range(n))
            else:
                forced = list(range(sink)) + list(range(n - recent, n))
                rest = [i for i in range(sink, n - recent)]
                rest.sort(key=lambda i: (-scores[b, h, i], i))
                keep = sorted(forced + rest[:max_pages - len(forced)])
            lists[b, h, :len(keep)] = keep
            counts[b, h] = len(keep)
    return lists, counts


def attend_ref(query, k_data, v_data, k_scale, v_scale, block_table, lens, lists, counts, scale=None):
    """float64 (output [B, Hq, D], lse [B, Hq])."""
    B, hq, D = query.shape
    hkv = k_data.shape[2]
    G = hq // hkv
    scale = D ** -0.5 if scale is None else scale
    out = np.zeros((B, hq, D), np.float64)
    lse = np.full((B, hq), -np.inf)
    for b in range(B):
        for h in range(hkv):
            ks, vs = [], []
            for col in lists[b, h, :max(0, min(int(counts[b, h]), lists.shape[2]))]:
                if col < 0 or col * PAGE >= lens[b]:
                    continue
                page, tok = block_table[b, col], min(PAGE, int(lens[b]) - col * PAGE)
                ks.append(dequant(k_data[page, :tok, h], k_scale[page, :tok, h], np.float64))
                vs.append(dequant(v_data[page, :tok, h], v_scale[page, :tok, h], np.float64))
            if not ks:
                continue
            k, v = np.concatenate(ks), np.concatenate(vs)
            x = query[b, h * G:(h + 1) * G].astype(np.float64) @ k.T * scale
            m = x.max(-1, keepdims=True)
            p = np.exp(x - m)
            total = p.sum(-1, keepdims=True)
            out[b, h * G:(h + 1) * G] = p @ v / total
            lse[b, h * G:(h + 1) * G] = ((m + np.log(total)) / math.log(2.0))[:, 0]
    return out, lse


def random_cache(rng, pages, hkv, dim):
    """Nibbles and scales as quantised normal keys and values have them."""
    data = [pack(np.clip(np.rint(rng.standard_normal((pages, PAGE, hkv, dim)) * 3), -7, 7).astype(np.int8))
            for _ in range(2)]
    scale = [np.clip(0.28 + 0.06 * rng.standard_normal((pages, PAGE, hkv, dim // GROUP)), 0.1, 0.6).astype(np.float16)
             for _ in range(2)]
    return data[0], data[1], scale[0], scale[1]
