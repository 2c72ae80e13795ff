"""Decode attention over the 8-bit cache for queries with a few channels far
larger than the others, as biases make them: the others have to keep their
bits, in short calls and in those whose bound allows long ones.

The bound is that of products of the fp16 queries as they are, summed in fp32
(see test_kv8_decode_gpu): |x - r| <= 2^-11 |r| + (2^-11 + 2^-13 +
2 D 2^-23 S) M + 1e-7.  S, the largest sum_i |q_i k_ti| / sqrt(D), does not
see a large channel over codes of zero.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_kv8_decode_gpu import check, half, make_pool, make_table, run, run_long, to_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("size", [1, 30, 300, 1000, 30000])
@pytest.mark.parametrize("H,Hkv,D", [(28, 4, 128), (14, 2, 64), (16, 1, 128)])
@pytest.mark.parametrize("long", [False, True])
def test_other_channels_keep_their_bits(long, H, Hkv, D, size, code):
    rng = np.random.default_rng(size)
    lens = [4096, 333, 1]
    q = half(rng, (len(lens), H, D))
    q[:, :, 5] = size
    q[1, :, D - 3] = -size
    table, pages = make_table(rng, lens, 32)
    kc, vc, scales = make_pool(rng, pages, Hkv, 32, D, code)
    kc[..., 5] = kc[..., D - 3] = 0
    cache = to_cache(kc, vc, scales, code)
    got = run_long(q, cache, table, lens, 32) if long else run(q, cache, table, lens)
    check(got, q, kc, vc, scales, code, table, lens)
