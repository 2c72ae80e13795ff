"""Plain numpy statement of the 8-bit paged cache and of a serving step's
block tables: what the GPU operators are checked against.

Codes are held as raw bytes (uint8).  `attention` works in 64 bits; `append`
follows the operator's own 32-bit arithmetic operation by operation (numpy's
float32 operations are the IEEE ones), so that codes and scales can be compared
exactly, and `rotate64` gives the same rows in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np

BLOCK = 16
KMAX = {"int8": 127.0, "e4m3": 448.0}


def _e4m3_values() -> np.ndarray:
    """Value of each of the 256 codes: sign, 4 exponent bits (bias 7), 3
    mantissa bits; no infinities, 0x7f and 0xff are NaN."""
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        if c & 127 == 127:
            x = math.nan
        v[c] = -x if c & 128 else x
    return v


E4M3 = _e4m3_values()


def decode(codes: np.ndarray, code: str) -> np.ndarray:
    return codes.view(np.int8).astype(np.float64) if code == "int8" else E4M3[codes]


def encode(y: np.ndarray, code: str) -> np.ndarray:
    """float32 to the nearest code, ties to even, saturating; NaN to 0 (int8) or 0x7f."""
    y = np.asarray(y, np.float32)
    nan = np.isnan(y)
    if code == "int8":
        r = np.rint(np.clip(np.where(nan, 0, y), -127, 127)).astype(np.int8).view(np.uint8)
        return np.where(nan, 0, r).astype(np.uint8)
    pos = E4M3[:127]                                  # 0 .. 448, ascending
    a = np.minimum(np.abs(np.where(nan, 0, y)).astype(np.float64), 448.0)
    hi = np.clip(np.searchsorted(pos, a), 0, 126)     # first value >= a
    lo = np.maximum(hi - 1, 0)
    dlo, dhi = a - pos[lo], pos[hi] - a
    pick = np.where(dlo < dhi, lo, np.where(dhi < dlo, hi, np.where(lo % 2 == 0, lo, hi)))
    out = pick.astype(np.uint8) | np.where(np.signbit(y), 128, 0).astype(np.uint8)
    return np.where(nan, 0x7f, out).astype(np.uint8)


def _f32(x):
    return np.asarray(x, np.float32)


def _rows(x, bias):
    x = _f32(x)
    return x if bias is None else x + _f32(bias).reshape(1, x.shape[1], x.shape[2])


def _turn_at(positions, freq_axis, cos, sin):
    half = cos.shape[1]
    at = np.asarray(positions)[np.asarray(freq_axis)[:half]].T              # [T, D/2]
    f = np.arange(half)
    return cos[at, f][:, None], sin[at, f][:, None]


def rotate(x, c, s):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


def rotate64(x, bias, positions, freq_axis, cos, sin):
    x = np.asarray(x, np.float64)
    if bias is not None:
        x = x + np.asarray(bias, np.float64).reshape(1, x.shape[1], x.shape[2])
    c, s = _turn_at(positions, freq_axis, cos.astype(np.float64), sin.astype(np.float64))
    return rotate(x, c, s)


def put(rows, codes, scales, which, slots, code):
    """Codes rows [T, Hkv, D] (float32) into codes [P, Hkv, ps, D] (bytes) and
    scales [P, Hkv, ps / 16, 2] at `slots`, in place."""
    ps = codes.shape[2]
    kmax = np.float32(KMAX[code])
    t = 0
    while t < len(slots):
        if slots[t] < 0 or slots[t] >= codes.shape[0] * ps:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] % BLOCK:
            n += 1
        page, r0 = slots[t] // ps, slots[t] % ps
        first = r0 % BLOCK
        for h in range(rows.shape[1]):
            x = rows[t:t + n, h]
            at = scales[page, h, r0 // BLOCK]
            old = at[which]
            with np.errstate(all="ignore"):
                top = np.float32(np.nan) if np.isnan(x).any() else np.abs(x).max()
                scale = np.float32(top / kmax)
                if first:
                    scale = np.float32(np.nan) if np.isnan(scale) or np.isnan(old) else max(scale, np.abs(old))
                if 0 < scale < np.float32(2.0 ** -100):
                    scale = np.float32(2.0 ** -100)
                grew = first and not np.isnan(old) and (np.isnan(scale) or scale > abs(old))
                if grew:
                    held = codes[page, h, r0 - first:r0]
                    z = _f32(decode(held, code)) * old
                    codes[page, h, r0 - first:r0] = encode(z / scale, code)
                y = np.zeros_like(x) if scale == 0 else x / scale
                codes[page, h, r0:r0 + n] = encode(y, code)
            at[which] = scale
        t += n


def append(q, k, v, biases, cos, sin, positions, freq_axis, slots, codes_k, codes_v, scales, code):
    """(q_out, k_out, v_out) in float32 before their rounding to fp16; the cache in place."""
    rows = [_rows(x, b) for x, b in zip((q, k, v), biases)]
    c, s = _turn_at(positions, freq_axis, _f32(cos), _f32(sin))
    rows[0], rows[1] = rotate(rows[0], c, s), rotate(rows[1], c, s)
    put(rows[1], codes_k, scales, 0, slots, code)
    put(rows[2], codes_v, scales, 1, slots, code)
    return rows


def values(codes, scales, which, code):
    """[P, Hkv, ps, D] in 64 bits: code * scale."""
    return decode(codes, code) * np.repeat(scales[..., which].astype(np.float64), BLOCK, 2)[..., None]


def attention(q, k, v, table, lens):
    """q [B, H, D]; k, v [P, Hkv, ps, D] in 64 bits.  Returns the outputs, and
    beside them sum_t p_t |v_t| and max_t sum_i |q_i k_ti| / sqrt(D) (for error
    bounds)."""
    B, H, D = q.shape
    P, Hkv, ps, _ = k.shape
    out, mass, big = np.zeros((B, H, D)), np.zeros((B, H, D)), np.zeros((B, H, 1))
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        ids = np.asarray(table[b][:-(-n // ps)], np.int64)
        real = (ids >= 0) & (ids < P)
        at = np.where(real, ids, 0)
        kk, vv = (np.where(real[:, None, None, None], x[at], 0.0).transpose(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :n]
                  for x in (k, v))
        for h in range(H):
            j = h // (H // Hkv)
            qh = q[b, h].astype(np.float64)
            s = kk[j] @ qh / math.sqrt(D)
            with np.errstate(all="ignore"):
                p = np.exp(s - s.max())
                p /= p.sum()
            out[b, h] = p @ vv[j]
            mass[b, h] = p @ np.abs(vv[j])
            big[b, h] = (np.abs(kk[j]) @ np.abs(qh)).max() / math.sqrt(D)
    return out, mass, big


def step(kv_lens, new_lens, table, stack, count, page_size, max_tokens):
    """One serving step on Python lists; returns (status, kv_lens, table, stack,
    count, offsets, positions, slots)."""
    B, width, P = len(kv_lens), len(table[0]), len(stack)
    nothing = [0] * (B + 1), [0] * max_tokens, [-1] * max_tokens
    cap = width * page_size
    if any(h < 0 or h > cap or h + max(n, 0) > cap for h, n in zip(kv_lens, new_lens)):
        return 2, kv_lens, table, stack, count, *nothing
    pages = lambda n: -(-n // page_size)  # noqa: E731
    give = sum(pages(h) for h, n in zip(kv_lens, new_lens) if n < 0)
    if not 0 <= count <= P or count + give > P:
        return 4, kv_lens, table, stack, count, *nothing
    if sum(max(n, 0) for n in new_lens) > max_tokens:
        return 3, kv_lens, table, stack, count, *nothing
    take = sum(pages(h + n) - pages(h) for h, n in zip(kv_lens, new_lens) if n > 0)
    if take > count + give:
        return 1, kv_lens, table, stack, count, *nothing
    table, stack = [list(r) for r in table], list(stack)
    for b in range(B):
        if new_lens[b] < 0:
            for j in range(pages(kv_lens[b])):
                stack[count] = table[b][j]
                count += 1
    after, offsets, positions, slots = [], [0], [], []
    for b in range(B):
        h, n = kv_lens[b], new_lens[b]
        after.append(0 if n < 0 else h + n)
        for j in range(pages(h), pages(h + n) if n > 0 else 0):
            count -= 1
            table[b][j] = stack[count]
        for pos in range(h, h + max(n, 0)):
            positions.append(pos)
            slots.append(table[b][pos // page_size] * page_size + pos % page_size)
        offsets.append(len(positions))
    pad = max_tokens - len(positions)
    return 0, after, table, stack, count, offsets, positions + [0] * pad, slots + [-1] * pad
