"""Append and attention of the 4-bit cache together, on K with a few channels far
larger than the others, as real layers and their biases have them: scores of many
sizes, from the rows that the append coded.

The attention is held to the 64-bit oracle over what the cache holds, by
test_kv4_decode_gpu's bound; the cache to the oracle's codes, exactly.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from forgert_b200 import attention as A
from oracle import kv4 as O
from test_kv4_decode_gpu import check, half, make_table, run, run_long

pytestmark = pytest.mark.gpu
ROWS = 4096


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("loud", [8, 30, 200])
@pytest.mark.parametrize("H,Hkv,D", [(14, 2, 64), (28, 4, 128), (24, 2, 64), (16, 1, 128)])
def test_append_then_attend(H, Hkv, D, loud, long):
    rng = np.random.default_rng(loud + H + D)
    ps, lens = 32, [2500, 1, 333, 0, 1024]
    table, pages = make_table(rng, lens, ps)
    T = sum(lens)
    pos = np.concatenate([np.arange(n) for n in lens]).astype(np.int32)
    slots = np.concatenate([table[b, np.arange(n) // ps].astype(np.int64) * ps + np.arange(n) % ps for b, n in enumerate(lens)])
    q, k, v = (half(rng, (T, n, D)) for n in (H, Hkv, Hkv))
    size = np.where(rng.random((Hkv, D)) < 0.05, loud, 1)
    size[:, 3] = loud
    k = (k * size).astype(np.float16)
    biases = [half(rng, (n, D)) for n in (H, Hkv, Hkv)]
    biases[1] = (biases[1] * size).astype(np.float16)
    a = np.arange(ROWS)[:, None] * 1e6 ** (-2.0 * np.arange(D // 2) / D)
    cos, sin = np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)
    order = rng.permutation(T)                             # rows stand by themselves
    q, k, v, pos, slots = q[order], k[order], v[order], pos[order], slots[order]

    cache = A.KV4Cache.empty(pages, ps, Hkv, D)
    for x in (cache.k, cache.v):
        x.fill_(255)
    cache.scales.fill_(float("nan"))                       # rows that nothing is written to
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    qd = dev(q)
    A.qkv_rope_append_kv4(qd, dev(k), dev(v), qd, None, None, dev(cos), dev(sin), dev(pos[None]), dev(slots), cache, T, H,
                          ROWS, *[dev(b) for b in biases])
    rows = O.turned(q, k, v, biases, cos, sin, pos[None], [0] * (D // 2))
    codes = [np.full((pages, Hkv, ps, D // 2), 255, np.uint8) for _ in range(2)]
    scales = np.full((pages, Hkv, ps, 2, D // 64, 2), np.nan, np.float16)
    for which in range(2):
        O.put(rows[1 + which], codes[which], scales, which, slots)
    torch.cuda.synchronize()
    for got, want in ((cache.k, codes[0]), (cache.v, codes[1]), (cache.scales, scales)):
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=got.dtype == torch.float16)

    # the last token's turned q of each sequence attends over it
    at = np.array([int(np.flatnonzero(order == sum(lens[:b + 1]) - 1)[0]) if n else 0 for b, n in enumerate(lens)])
    ask = qd.cpu().numpy()[at]
    got = run_long(ask, cache, table, lens, ps) if long else run(ask, cache, table, lens)
    assert (got[3] == 0).all()
    clean = np.where(np.isnan(scales), 0, scales).astype(np.float16)
    check(got, ask, *codes, clean, table, lens)
