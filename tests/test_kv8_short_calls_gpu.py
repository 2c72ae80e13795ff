"""Short calls of decode attention over the 8-bit cache: what the outputs are off
by is their rounding to fp16 and hardly more.

Beside that rounding the kernel's own errors are those of weights in two fp16
parts (2^-22), of the exponentials (about 2^-22) and of fp32 sums of D products
(some 2^-21 of a score): all below a hundredth of the outputs' 2^-11.  So the
2-norm of the error stays within 1.1 times that of the exact result rounded to
fp16, where one fp16 rounding of each weight makes it 1.2 to 1.5 times.
"""
from __future__ import annotations

import numpy as np
import pytest

from oracle import kv8 as O
from test_kv8_decode_gpu import SHAPES, half, make_pool, make_table, run, to_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
@pytest.mark.parametrize("lens", [[512], [100, 700, 33, 0, 1500]])
def test_error_is_the_outputs_rounding(lens, H, Hkv, D, code):
    rng = np.random.default_rng(H + D + len(lens))
    q = half(rng, (len(lens), H, D))
    table, pages = make_table(rng, lens, 16)
    kc, vc, scales = make_pool(rng, pages, Hkv, 16, D, code)
    got = run(q, to_cache(kc, vc, scales, code), table, lens).astype(np.float64)
    r, _, _ = O.attention(q, O.values(kc, scales, 0, code), O.values(vc, scales, 1, code), table, lens)
    rounded = np.linalg.norm(r.astype(np.float16).astype(np.float64) - r)
    assert np.linalg.norm(got - r) <= 1.1 * rounded
