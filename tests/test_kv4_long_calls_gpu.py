"""Decode attention over the 4-bit cache in calls whose bound max_kv_len allows
long sequences: what the outputs are off by is their rounding to fp16 and hardly
more, as in short calls, whatever the bound and the lengths.

Beside that rounding the kernel's own errors are those of weights in two fp16
parts (2^-22), of the exponentials (about 2^-22) and of fp32 sums of D products
(some 2^-21 of a score): all below a hundredth of the outputs' 2^-11.  So the
2-norm of the error stays within 1.1 times that of the exact result rounded to
fp16, where one fp16 rounding of each weight makes it 1.4 to 1.5 times.
"""
from __future__ import annotations

import numpy as np
import pytest

from oracle import kv4 as O
from oracle import kv8
from test_kv4_decode_gpu import SHAPES, check, half, make_pool, make_table, run, run_long, to_cache

pytestmark = pytest.mark.gpu


def case(lens, H, Hkv, D, ps):
    rng = np.random.default_rng(H + D + len(lens) + max(lens))
    q = half(rng, (len(lens), H, D))
    table, pages = make_table(rng, lens, ps)
    return (q, *make_pool(rng, pages, Hkv, ps, D), table)


def close(got, q, kc, vc, scales, table, lens):
    r, _, _ = kv8.attention(q, O.values(kc, scales, 0), O.values(vc, scales, 1), table, lens)
    rounded = np.linalg.norm(r.astype(np.float16).astype(np.float64) - r)
    e = np.linalg.norm(got.astype(np.float64) - r)
    assert e <= 1.1 * rounded, e / rounded


@pytest.mark.parametrize("H,Hkv,D", SHAPES)
@pytest.mark.parametrize("lens", [[512], [100, 700, 33, 0, 1500], [3000, 2047, 4111]])
def test_error_is_the_outputs_rounding(lens, H, Hkv, D):
    q, kc, vc, scales, table = case(lens, H, Hkv, D, 16)
    cache = to_cache(kc, vc, scales)
    got = run_long(q, cache, table, lens, 16)
    check(got, q, kc, vc, scales, table, lens)
    close(got, q, kc, vc, scales, table, lens)
    close(run(q, cache, table, lens), q, kc, vc, scales, table, lens)


@pytest.mark.parametrize("lens", [[20000], [65536], [9000, 1, 5003, 0, 7777, 12288]])
@pytest.mark.parametrize("H,Hkv,D", [(14, 2, 64), (24, 2, 64), (28, 4, 128), (16, 1, 128)])
def test_long_sequences(H, Hkv, D, lens):
    """Units of many pieces, whose merge goes in two levels, and rings that turn
    many times, in every shape for long calls; the bits do not depend on who
    merges."""
    q, kc, vc, scales, table = case(lens, H, Hkv, D, 64)
    cache = to_cache(kc, vc, scales)
    got = run_long(q, cache, table, lens, 64)
    check(got, q, kc, vc, scales, table, lens)
    close(got, q, kc, vc, scales, table, lens)
    for _ in range(5):
        assert np.array_equal(run_long(q, cache, table, lens, 64), got)
