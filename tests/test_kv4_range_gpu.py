"""The 4-bit cache at the end of fp16's range: a group's scale is rounded up, so
its largest code may stand for a number above 65504.  Read-back and attention
give 65504 there, not an infinity.

Tolerances: the read-back is the oracle's value, cut, rounded once.  An output is
the exact one within test_kv4_decode_gpu's bound, and cutting takes it no further
from it than the exact one, cut.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from forgert_b200 import attention as A
from oracle import kv4 as O
from oracle import kv8
from test_kv4_decode_gpu import half, run, run_long, to_cache

pytestmark = pytest.mark.gpu
TOP = 65504.0


def wide_rows(D, n=64):
    """fp16 rows whose groups reach up to 65504 from minima of all sizes."""
    rng = np.random.default_rng(D)
    low = np.concatenate([[-TOP, -TOP, 0, TOP, 65472, 60000], np.exp2(rng.uniform(-24, 15.9, n - 6)) * rng.choice([-1, 1], n - 6)])
    x = low[:, None] + (TOP - low[:, None]) * rng.random((n, D))
    x[:, ::5], x[:, 1::5] = TOP, low[:, None]
    return x.astype(np.float16)


def cache_of(rows, bias=None):
    """Rows [n, D] as K and V of n tokens of one kv head, by the append (K unturned)."""
    n, D = rows.shape
    ps = 16
    cache = A.KV4Cache.empty(-(-n // ps), ps, 1, D)
    x = torch.from_numpy(rows[:, None].copy()).cuda()
    q = torch.zeros((n, 1, D), dtype=torch.float16, device="cuda")
    cos, sin = (torch.full((1, D // 2), c, dtype=torch.float32, device="cuda") for c in (1, 0))
    A.qkv_rope_append_kv4(q, x, x, q, None, None, cos, sin, torch.zeros((1, n), dtype=torch.int32, device="cuda"),
                          torch.arange(n, device="cuda"), cache, n, 1, 1, k_bias=bias, v_bias=bias)
    return cache, (cache.k.cpu().numpy(), cache.v.cpu().numpy(), cache.scales.cpu().numpy())


def back(cache, n, D):
    out = torch.empty((2, n, 1, D), dtype=torch.float16, device="cuda")
    A.kv4_gather(cache, torch.arange(n, device="cuda"), out[0], out[1], n)
    return out.cpu().numpy()[:, :, 0].astype(np.float64)


@pytest.mark.parametrize("D", [64, 128])
def test_read_back_is_within_half_a_scale(D):
    rows = wide_rows(D)
    cache, (kc, vc, scales) = cache_of(rows)
    got = back(cache, len(rows), D)
    assert (O.values(vc, scales, 1) >= 65520).any()            # would round to infinity
    for which, codes in enumerate((kc, vc)):
        want = O.values(codes, scales, which).transpose(0, 2, 1, 3).reshape(-1, D)[:len(rows)]
        assert np.array_equal(got[which], np.minimum(want, TOP).astype(np.float16).astype(np.float64))
        s = np.repeat(scales[:, 0, :, which, :, 0].reshape(-1, D // 64)[:len(rows)].astype(np.float64), 64, 1)
        # half a scale, the fp32 roundings of x - bias and of the quotient (15 scales at
        # most, 2^-24 of that each), and the rounding to fp16
        assert (np.abs(got[which] - rows) <= s * (0.5 + 2.0 ** -19) + 2.0 ** -11 * (np.abs(rows) + s) + 2.0 ** -25).all()


@pytest.mark.parametrize("D", [64, 128])
def test_values_past_the_range_are_cut(D):
    """A bias takes rows above 65504; NaN groups stay NaN."""
    rows = wide_rows(D, 20)
    rows[7, 3] = np.nan
    bias = torch.full((D,), 30000.0, dtype=torch.float16, device="cuda")
    cache, (kc, vc, scales) = cache_of(rows, bias)
    want = np.minimum(O.values(vc, scales, 1).transpose(0, 2, 1, 3).reshape(-1, D)[:20], TOP)
    got = back(cache, 20, D)[1]
    assert np.array_equal(got, want.astype(np.float16).astype(np.float64), equal_nan=True)
    assert np.isnan(got[7, :64]).all() and np.isfinite(got[np.arange(20) != 7]).all() and (got[3] == TOP).all()


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("n", [1, 17, 5000])
@pytest.mark.parametrize("H,D", [(1, 64), (7, 128), (16, 128), (12, 64)])
def test_attention_is_finite(H, D, n, long):
    """Every V row at the top of the range: outputs whole and merged from pieces."""
    rng = np.random.default_rng(n)
    _, (kc, vc, scales) = cache_of(wide_rows(D, 16))
    top = vc[:1, :, :1].copy()                                 # the widest group's codes
    pages = -(-n // 16)
    vc, pair = np.repeat(np.repeat(top, 16, 2), pages, 0), scales[:1, :, :1, 1:].copy()
    kc = rng.integers(0, 256, vc.shape, dtype=np.uint8)
    sc = np.tile(np.repeat(pair, 16, 2), (pages, 1, 1, 2, 1, 1))
    sc[:, :, :, 0] = [0.1, -0.75]
    q = half(rng, (1, H, D))
    table = np.arange(pages, dtype=np.int32)[None]
    cache = to_cache(kc, vc, sc)
    got = run_long(q, cache, table, [n], 16) if long else run(q, cache, table, [n])
    r, _, _ = kv8.attention(q, O.values(kc, sc, 0), O.values(vc, sc, 1), table, [n])
    assert r.max() >= 65520
    assert np.isfinite(got).all()
    whole = np.abs(O.values(vc, sc, 1)).max() + 15 * 8736      # the sums' terms
    assert (np.abs(got - np.minimum(r, TOP)) <= 2.0 ** -11 * np.abs(r) + 2.0 ** -12 * whole).all()
