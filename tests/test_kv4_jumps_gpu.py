"""Decode attention over the 4-bit cache where a row's score lies hundreds of
nats above all before it, so far that its probability against the running
reference is infinite in 32 bits: at rows whose V scale is 0 (all their values
the bias, as the append writes constant groups), beside a NaN scale, and at a
page outside the pool (a row of zeros).

Tolerances are test_kv4_decode_gpu's: its bound holds whatever the scores.
"""
from __future__ import annotations

import numpy as np
import pytest

from oracle import kv4 as O
from oracle import kv8
from test_kv4_decode_gpu import check, half, make_pool, make_table, run, run_long, to_cache

pytestmark = pytest.mark.gpu

SHAPES = [(14, 2, 64), (28, 4, 128), (24, 2, 64), (16, 1, 128)]
LENS = [700, 40, 333, 1500]
# within a block, in a warp's next block, in its next step (of 128 or 256 positions),
# in another warp's rows; the last ones where four-block steps end
AT = [3, 21, 130, 259, 300, 517, 1290]


def lift(scales, table, lens, q, ps, at, nats, alone=False):
    """Raises K's biases from each position in `at` on (alone: at these positions
    only, each above the one before), so that every head's scores grow by at least
    `nats` there."""
    D = q.shape[2]
    for b, n in enumerate(lens):
        delta = nats * np.sqrt(D) / q[b].astype(np.float64).sum(-1).min()
        for t in range(n):
            if t in at or not alone:
                scales[table[b, t // ps], :, t % ps, 0, :, 1] += np.float16(delta * sum(t >= x for x in at))


def jumps(H, Hkv, D, nats, ps=32, seed=0, alone=False):
    rng = np.random.default_rng(seed + H + D)
    q = np.abs(half(rng, (len(LENS), H, D))) + np.float16(1)
    table, pages = make_table(rng, LENS, ps)
    kc, vc, scales = make_pool(rng, pages, Hkv, ps, D)
    lift(scales, table, LENS, q, ps, AT, nats, alone)
    assert np.isfinite(scales).all()
    return q, table, kc, vc, scales


def rows(table, ps, at=AT):
    """(page, row) of the positions `at`, of every sequence that holds them."""
    return [(table[b, t // ps], t % ps) for b, n in enumerate(LENS) for t in at if t < n]


def call(long, q, kc, vc, scales, table, lens, ps=32):
    cache = to_cache(kc, vc, scales)
    return run_long(q, cache, table, lens, ps) if long else run(q, cache, table, lens)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("alone", [False, True])
@pytest.mark.parametrize("nats", [80, 100, 300])
@pytest.mark.parametrize("groups", ["first", "last", "all"])
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
def test_jump_at_rows_of_scale_zero(H, Hkv, D, groups, nats, alone, long):
    q, table, kc, vc, scales = jumps(H, Hkv, D, nats, alone=alone)
    for page, r in rows(table, 32):
        x = {"first": slice(0, 1), "last": slice(-1, None), "all": slice(None)}[groups]
        scales[page, :, r, 1, x, 0] = 0
    got = call(long, q, kc, vc, scales, table, LENS)
    check(got, q, kc, vc, scales, table, LENS, long, norm=False)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
def test_constant_rows_above_ordinary_ones(H, Hkv, D, long):
    """Every V row from the jump on is constant: no weight at all beside the
    probabilities tells that the reference has to move."""
    q, table, kc, vc, scales = jumps(H, Hkv, D, 0)
    lift(scales, table, LENS, q, 32, [37, 170], 120)
    for b, n in enumerate(LENS):
        for t in range(37, n):
            scales[table[b, t // 32], :, t % 32, 1, :, 0] = 0
    got = call(long, q, kc, vc, scales, table, LENS)
    check(got, q, kc, vc, scales, table, LENS, long, norm=False)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("alone", [False, True])
@pytest.mark.parametrize("what", ["scale", "bias", "both"])
@pytest.mark.parametrize("x", [0, 1])
@pytest.mark.parametrize("H,Hkv", [(28, 4), (16, 1)])
def test_nan_group_beside_a_jump(H, Hkv, x, what, alone, long):
    """A NaN in one group of V at rows that raise the reference: the other
    group's dims are what they would be without."""
    D = 128
    q, table, kc, vc, scales = jumps(H, Hkv, D, 100, alone=alone)
    clean = scales.copy()
    for page, r in rows(table, 32, [21, 300]):
        scales[page, :, r, 1, x, {"scale": slice(0, 1), "bias": slice(1, 2), "both": slice(0, 2)}[what]] = np.nan
    got = call(long, q, kc, vc, scales, table, LENS)
    bad = np.zeros((len(LENS), H, D), bool)
    bad[[b for b, n in enumerate(LENS) if n > 21], :, 64 * x:64 * x + 64] = True
    assert np.isnan(got[bad]).all()
    got[bad] = call(long, q, kc, vc, clean, table, LENS)[bad]
    check(got, q, kc, vc, clean, table, LENS, long, norm=False)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("nats", [100, 400])
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
def test_page_outside_the_pool_above_low_scores(H, Hkv, D, nats, long):
    """All scores far below 0, that of the zero rows of a page outside the pool."""
    q, table, kc, vc, scales = jumps(H, Hkv, D, 0)
    lift(scales, table, LENS, q, 32, [0], -nats)
    table[0, 9], table[2, 3], table[3, 40] = -1, 2**31 - 1, -5
    got = call(long, q, kc, vc, scales, table, LENS)
    check(got, q, kc, vc, scales, table, LENS, long, norm=False)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
def test_a_head_that_jumps_leaves_the_others_bits(H, Hkv, D, long):
    """One head's references move, its neighbours' outputs keep their bits."""
    q, table, kc, vc, scales = jumps(H, Hkv, D, 0)
    for page, r in rows(table, 32):
        scales[page, :, r, 1, -1, 0] = 0
        scales[page, :, r, 0, :, 1] += np.float16(8)
    q /= np.float16(4)
    clean = call(long, q, kc, vc, scales, table, LENS)
    q2 = q.copy()
    q2[:, 2] *= np.float16(64)
    got = call(long, q2, kc, vc, scales, table, LENS)
    check(got, q2, kc, vc, scales, table, LENS, long, norm=False)
    keep = np.arange(H) != 2
    assert np.array_equal(got[:, keep], clean[:, keep])


def test_oracle_takes_the_jump():
    """What the bound is held against: a jump of 300 nats leaves the last rows alone."""
    q, table, kc, vc, scales = jumps(12, 2, 64, 300)
    r, _, _ = kv8.attention(q, O.values(kc, scales, 0), O.values(vc, scales, 1), table, LENS)
    assert np.isfinite(r).all()
