"""Plain numpy statement of the 4-bit paged cache, beside oracle.kv8's rotary
embedding and attention: what the GPU operators are checked against.

`put` follows the operator's own 32-bit arithmetic operation by operation
(numpy's float32 operations are the IEEE ones), so that codes and scales can be
compared exactly; `values` is in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np

from . import kv8

GROUP = 64


def half_below(x) -> np.ndarray:
    """The largest fp16 number not above float32 x (NaN stays)."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        h = x.astype(np.float16)
        down = np.nextafter(h, np.float16(-np.inf), dtype=np.float16)
        # past the range the nearest is an infinity: 65504 lies below a finite x
        down = np.where(np.isposinf(h) & np.isfinite(x), np.float16(65504), down)
        return np.where(h.astype(np.float32) > x, down, h).astype(np.float16)


def half_above(x) -> np.ndarray:
    return -half_below(-np.asarray(x, np.float32))


def unpack(raw: np.ndarray) -> np.ndarray:
    """Bytes [..., n] to codes [..., 2 n]."""
    return np.stack([raw & 15, raw >> 4], -1).reshape(*raw.shape[:-1], -1)


def pack(codes: np.ndarray) -> np.ndarray:
    c = codes.astype(np.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def encode(x):
    """float32 rows [..., D]: bytes [..., D / 2] and (scale, bias) [..., D / 64, 2] fp16."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(all="ignore"):
        bias = half_below(g.min(-1) + np.float32(0))
        b = bias.astype(np.float32)
        scale = half_above((g.max(-1) - b) / np.float32(15))
        s = scale.astype(np.float32)
        good = np.isfinite(b) & np.isfinite(s)
        n = np.rint((g - b[..., None]) / s[..., None])
    n = np.where((good & (s > 0))[..., None], n, 0)
    pairs = np.where(good[..., None], np.stack([scale, bias], -1), np.float16(np.nan))
    return pack(n.reshape(x.shape)), pairs.astype(np.float16)


def put(rows, codes, scales, which, slots):
    """Codes rows [T, Hkv, D] (float32) into codes [P, Hkv, ps, D / 2] and scales
    [P, Hkv, ps, 2, D / 64, 2] at `slots`, in place."""
    ps = codes.shape[2]
    raw, pairs = encode(np.asarray(rows, np.float32))
    for t, s in enumerate(slots):
        if 0 <= s < codes.shape[0] * ps:
            codes[s // ps, :, s % ps] = raw[t]
            scales[s // ps, :, s % ps, which] = pairs[t]


def values(codes, scales, which):
    """[P, Hkv, ps, D] in 64 bits: code * scale + bias."""
    s = np.repeat(scales[:, :, :, which].astype(np.float64), GROUP, -2)
    return unpack(codes) * s[..., 0] + s[..., 1]


def turned(q, k, v, biases, cos, sin, positions, freq_axis):
    """q, k (turned) and v with their biases in float32, before any rounding to fp16."""
    rows = [kv8._rows(x, b) for x, b in zip((q, k, v), biases)]
    c, s = kv8._turn_at(positions, freq_axis, kv8._f32(cos), kv8._f32(sin))
    return [kv8.rotate(rows[0], c, s), kv8.rotate(rows[1], c, s), rows[2]]


def masses(q, codes_k, codes_v, scales, table, lens, p_of=None):
    """What the rounding errors of the decode kernel scale with, per sequence and
    head: sum_t p_t |n - 8| a' (weights' rounding), sum_t p_t ((n + 8) a' + |mid|)
    (sums), both [B, H, D], and max_t of the terms of a score's sum [B, H, 1]."""
    B, H, D = q.shape
    P, Hkv, ps, _ = codes_k.shape
    k, v = values(codes_k, scales, 0), values(codes_v, scales, 1)
    near, all_, big = np.zeros((B, H, D)), np.zeros((B, H, D)), np.zeros((B, H, 1))
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        ids = np.asarray(table[b][:-(-n // ps)], np.int64)
        real = (ids >= 0) & (ids < P)
        at = np.where(real, ids, 0)

        def rows(x):
            x = np.where(real.reshape(-1, *[1] * (x.ndim - 1)), x[at], 0)
            return np.moveaxis(x, 1, 0).reshape(Hkv, -1, *x.shape[3:])[:, :n]

        kk, nk, nv = rows(k), rows(unpack(codes_k)), rows(unpack(codes_v))
        pairs = rows(scales.astype(np.float64))                     # [Hkv, n, 2, NG, 2]
        ka, kb, va, vb = (np.repeat(pairs[:, :, w, :, i], GROUP, -1) for w in (0, 1) for i in (0, 1))
        for h in range(H):
            j = h // (H // Hkv)
            qh = q[b, h].astype(np.float64)
            s = kk[j] @ qh / math.sqrt(D)
            p = np.exp(s - s.max())
            p /= p.sum()
            near[b, h] = p @ (np.abs(nv[j] - 8.0) * va[j])
            all_[b, h] = p @ ((nv[j] + 8.0) * va[j] + np.abs(vb[j] + 8 * va[j]))
            big[b, h] = ((nk[j] * ka[j] + np.abs(kb[j])) @ np.abs(qh)).max() / math.sqrt(D)
    return near, all_, big
