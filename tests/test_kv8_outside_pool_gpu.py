"""fr_qkv_rope_append_kv8 with slots past the pool: such a token is recorded
and not cached, and all of its outputs are written; its neighbours and the
cache are as if it were not there."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from forgert_b200 import attention as A
from oracle import kv8 as O
from test_kv8_append_gpu import ROWS, Pool, dev, half, runs_of, tables

pytestmark = pytest.mark.gpu


# 148 SMs: up to 592, 4736 and more tokens of two kv heads look through windows
# of 1, 4 and 16 tokens
@pytest.mark.parametrize("T", [5, 700, 5000])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("D,code,bias", [(64, "int8", True), (128, "e4m3", False)])
def test_outputs_of_tokens_past_the_pool(T, in_place, D, code, bias):
    rng = np.random.default_rng(T)
    H, Hkv, ps = 4, 2, 16
    pages = -(-T // ps) + 3
    pool = Pool(rng, pages, Hkv, ps, D, code)
    slots, pos = runs_of(rng, [(7, T // 2), (0, T - T // 2)], pages, ps)
    past = rng.random(T) < 0.2
    past[[0, T - 1]] = True
    slots[past] = pages * ps + rng.integers(0, 10 ** 12, past.sum())
    slots[rng.random(T) < 0.05] = -1
    x = [half(rng, (T, n, D)) for n in (H, Hkv, Hkv)]
    biases = [half(rng, (n, D)) if bias else None for n in (H, Hkv, Hkv)]
    cos, sin = tables(D)
    want = O.append(*x, biases, cos, sin, pos[None], [0] * (D // 2), slots, pool.k, pool.v, pool.scales, code)
    ins = [dev(a) for a in x]
    outs = ins if in_place else [torch.full_like(a, 9.0) for a in ins]
    A.qkv_rope_append_kv8(*ins, *outs, dev(cos), dev(sin), dev(pos.astype(np.int32)), dev(slots), pool.cache, T, H, ROWS,
                          *[dev(b) for b in biases])
    torch.cuda.synchronize()
    assert A.device_error() == (4 if (slots >= pages * ps).any() else 0)
    out = slots < 0
    for got, r, a in zip(outs, want, x):
        got = got.cpu().numpy()
        assert np.array_equal(got[~out], r[~out].astype(np.float16))
        assert np.array_equal(got[out], a[out] if in_place else np.full_like(a[out], 9.0))
    pool.same()
