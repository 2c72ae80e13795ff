"""Decode attention over the 4-bit cache with scores of any size that fp16 queries
and keys can give (up to 2^36 in base 2), where a step of fp32 is worth many nats.

Rows of equal K have equal scores in fp32 as well, so the outputs are means of the
V of the rows at the top, however large the scores: exact but for the outputs'
rounding (2^-11) and fp32 sums (2^-12 of the terms' sizes covers them, as in
test_kv4_decode_gpu).
"""
from __future__ import annotations

import numpy as np
import pytest

from oracle import kv4 as O
from test_kv4_decode_gpu import half, make_pool, make_table, run, run_long, to_cache

pytestmark = pytest.mark.gpu
LENS = [700, 40, 333]
SHAPES = [(14, 2, 64), (28, 4, 128), (24, 2, 64), (16, 1, 128)]


def means(scales, vc, table, at, H, ps=32):
    """Per sequence the mean of V over the positions at[b], and of its terms' sizes."""
    v = O.values(vc, scales, 1)
    mid = np.abs(scales[:, :, :, 1, :, 1].astype(np.float64)) + 15 * scales[:, :, :, 1, :, 0].astype(np.float64)
    mid = np.repeat(mid, 64, -1)
    out, size = [], []
    for b, where in enumerate(at):
        for x, to in ((v, out), (mid, size)):
            rows = np.stack([x[table[b, t // ps], :, t % ps] for t in where])           # [n, Hkv, D]
            to.append(np.repeat(rows.mean(0), H // rows.shape[1], 0))
    return np.stack(out), np.stack(size)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("size", [30, 3000, 9000, 20000, 60000])
@pytest.mark.parametrize("tiny", [0, 4, 12, 20])
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
def test_equal_scores(H, Hkv, D, tiny, size, long):
    """All rows of one K; V's scales 2^-tiny as large."""
    rng = np.random.default_rng(size + tiny)
    q = np.full((3, H, D), size, np.float16)
    q[:, 1::2] *= np.float16(0.37)                         # scores that are no power of two
    q[1] *= np.float16(-1)
    table, pages = make_table(rng, LENS, 32)
    kc, vc, scales = make_pool(rng, pages, Hkv, 32, D)
    kc[:] = rng.integers(0, 256, D // 2)
    scales[:, :, :, 0] = [0.0006 * size, 0.3 * size]
    scales[:, :, :, 1] *= np.float16(2.0 ** -tiny)
    cache = to_cache(kc, vc, scales)
    got = run_long(q, cache, table, LENS, 32) if long else run(q, cache, table, LENS)
    want, terms = means(scales, vc, table, [range(n) for n in LENS], H)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -12 * terms + 2.0 ** -24).all()


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("size", [30, 3000, 9000, 20000, 60000])
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
def test_steps_of_huge_scores(H, Hkv, D, size, long):
    """Scores that climb and fall by a hundredth of their size: the rows at the top
    share the output."""
    rng = np.random.default_rng(size)
    q = np.full((3, H, D), size, np.float16)
    table, pages = make_table(rng, LENS, 32)
    kc, vc, scales = make_pool(rng, pages, Hkv, 32, D)
    kc[:] = 0x33
    scales[:, :, :, 0] = [0.01, 0.3 * size]
    at = []
    for b, n in enumerate(LENS):
        level = rng.permutation(n) % 8
        for t in range(n):
            scales[table[b, t // 32], :, t % 32, 0, :, 1] += np.float16(0.02 * size * level[t])
        at.append(np.flatnonzero(level == level.max()))
    if size > 30:
        scales[:, :, ::3, 1, -1] *= np.float16(2.0 ** -9)
    cache = to_cache(kc, vc, scales)
    got = run_long(q, cache, table, LENS, 32) if long else run(q, cache, table, LENS)
    want, terms = means(scales, vc, table, at, H)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -12 * terms + 2.0 ** -24).all()
