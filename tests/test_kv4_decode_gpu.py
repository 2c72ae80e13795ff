"""GPU tests of decode attention over the 4-bit paged cache
(fr_decode_attn_paged_kv4) against the 64-bit oracle (oracle.kv4, oracle.kv8).

Error bound, from the kernel's arithmetic.  A value is (n - 8) a + mid, mid the
group's middle.  The output is rounded to fp16 once (2^-11 of itself).  In long
calls each weight p a enters its product as one fp16: 2^-11 of
near = sum_t p_t |n - 8| a.  A score carries the roundings of a sum of D + 4
terms (2^-23 each, relative to the sum of the terms' sizes, big), which moves a
probability by that relative amount, in the numerator and in the sum; 2^-13
stands for the exponentials, the middles and the fp32 sums of codes 0 .. 15 and
of 8 (all = sum_t p_t ((n + 8) a + |mid|)):
  |x - r| <= 2^-11 |r| + 2^-11 near (long) + (2^-13 + 2 (D + 4) 2^-23 big) all + 1e-7.
On normal data the errors of many outputs average: their 2-norm is at most
1.1 * 2^-11 of the results' in short calls (the outputs' rounding alone is below
2^-11) and 2^-10 in long ones (the weights' rounding adds as much at most).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from forgert_b200 import attention as A
from forgert_b200._lib import ForgeRTError
from oracle import kv4 as O
from oracle import kv8

pytestmark = pytest.mark.gpu

SHAPES = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (8, 8, 64), (16, 1, 128), (24, 2, 64)]


def make_pool(rng, pages, Hkv, ps, D, spread=0.4):
    """Raw codes; scales and biases about those of normal data, of many sizes."""
    kc, vc = (rng.integers(0, 256, (pages, Hkv, ps, D // 2), dtype=np.uint8) for _ in range(2))
    a = 0.3 * np.exp(spread * rng.standard_normal((pages, Hkv, ps, 2, D // 64)))
    b = -7.5 * a * (1 + 0.2 * rng.standard_normal(a.shape))
    return kc, vc, np.stack([a, b], -1).astype(np.float16)


def make_table(rng, lens, ps, spare=3, width=None):
    need = [-(-max(0, n) // ps) for n in lens]
    pages = sum(need) + spare
    ids = rng.permutation(pages)
    width = width or max(1, max(need)) + 2
    table = rng.choice([-1, -2**31, pages, 2**31 - 1], (len(lens), width)).astype(np.int32)   # never read
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, pages


def poison(table, lens, ps, scales):
    """What nobody owns must not matter: NaN scales behind each end and in spare pages."""
    owned = np.zeros((scales.shape[0], ps), bool)
    for b, n in enumerate(lens):
        for j in range(-(-max(0, n) // ps)):
            owned[table[b, j], :max(0, min(ps, n - j * ps))] = True
    scales[np.broadcast_to(~owned[:, None, :, None, None, None], scales.shape)] = np.nan


def to_cache(kc, vc, scales, layout="head"):
    def lay(c):
        x = torch.from_numpy(c).cuda()
        if layout == "token":                          # [P, ps, Hkv, D / 2] pages
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "heads":                          # [Hkv, P, ps, D / 2]
            x = x.transpose(0, 1).contiguous().transpose(0, 1)
        if layout == "padded":                         # rows 16 bytes apart
            x = torch.cat([x, torch.full_like(x[..., :16], 255)], -1)[..., :x.shape[-1]]
        return x
    if layout == "mixed":                              # K and V pages side by side in one allocation
        both = torch.stack([torch.from_numpy(kc), torch.from_numpy(vc)], 1).cuda()
        k, v = both[:, 0], both[:, 1]
    else:
        k, v = lay(kc), lay(vc)
    return A.KV4Cache(k, v, torch.from_numpy(scales).cuda())


def run(q, cache, table, lens, max_kv_len=None, stream=None, q_stride=0, qd=None):
    B, H, D = q.shape
    qd = torch.from_numpy(q).cuda() if qd is None else qd
    out = torch.full((B, H, D), float("nan"), dtype=torch.float16, device="cuda")
    td, ld = torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    mk = max(0, max(lens)) if max_kv_len is None else max_kv_len
    A.decode_attn_paged_kv4(qd, cache, td, ld, out, B, H, table.shape[1], mk, q_stride=q_stride, stream=stream)
    torch.cuda.synchronize()
    assert A.device_error() == 0
    return out.cpu().numpy()


def run_long(q, cache, table, lens, page_size):
    """The shape for long calls: its bound max_kv_len allows many tiles."""
    bound = (1 << 19) // page_size * page_size
    wide = np.full((len(lens), bound // page_size), -1, np.int32)
    wide[:, :table.shape[1]] = table
    return run(q, cache, wide, lens, max_kv_len=bound)


def check(got, q, kc, vc, scales, table, lens, long=False, norm=True):
    r, _, _ = kv8.attention(q, O.values(kc, scales, 0), O.values(vc, scales, 1), table, lens)
    near, whole, big = O.masses(q, kc, vc, scales, table, lens)
    D = q.shape[2]
    tol = 2.0 ** -11 * np.abs(r) + (2.0 ** -11 if long else 0.0) * near + (2.0 ** -13 + 2 * (D + 4) * 2.0 ** -23 * big) * whole + 1e-7
    err = np.abs(got.astype(np.float64) - r)
    assert np.isfinite(got).all()
    assert (err <= tol).all(), f"max err / tol {(err / tol).max():.3f}"
    if norm:
        e = np.linalg.norm(err) / np.linalg.norm(r)
        assert e <= (2.0 ** -10 if long else 1.1 * 2.0 ** -11), f"2-norm of the error {e:.2e}"


def half(rng, shape):
    return rng.standard_normal(shape).astype(np.float16)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("page_size", [16, 48, 64, 256])
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
def test_matches_oracle(H, Hkv, D, page_size, long):
    rng = np.random.default_rng(page_size * 1000 + H * 10 + D)
    lens = [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, page_size, page_size + 1, 700, 0, 2049, 3 * page_size - 1]
    q = half(rng, (len(lens), H, D))
    table, pages = make_table(rng, lens, page_size)
    kc, vc, scales = make_pool(rng, pages, Hkv, page_size, D)
    clean = scales.copy()
    poison(table, lens, page_size, scales)
    cache = to_cache(kc, vc, scales)
    got = run_long(q, cache, table, lens, page_size) if long else run(q, cache, table, lens)
    assert (got[[0, 14]] == 0).all()
    check(got, q, kc, vc, clean, table, lens, long)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (3, 3), (5, 1), (8, 1), (9, 1), (10, 2), (24, 1), (33, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_group_sizes(D, H, Hkv, long):
    rng = np.random.default_rng(H * 7 + D)
    lens = [1, 40, 333]
    q = half(rng, (3, H, D))
    table, pages = make_table(rng, lens, 32)
    kc, vc, scales = make_pool(rng, pages, Hkv, 32, D)
    cache = to_cache(kc, vc, scales)
    got = run_long(q, cache, table, lens, 32) if long else run(q, cache, table, lens)
    check(got, q, kc, vc, scales, table, lens, long)


@pytest.mark.parametrize("n", [1, 2, 16, 129, 512, 1000, 4096, 20000, 65536])
@pytest.mark.parametrize("H,Hkv,D", [(14, 2, 64), (28, 4, 128), (16, 1, 128)])
def test_one_sequence(n, H, Hkv, D):
    """From one token to long ranges that many CTAs share; the bits do not
    depend on who merges."""
    rng = np.random.default_rng(n)
    q = half(rng, (1, H, D))
    table, pages = make_table(rng, [n], 64)
    kc, vc, scales = make_pool(rng, pages, Hkv, 64, D)
    cache = to_cache(kc, vc, scales)
    got = run(q, cache, table, [n])
    check(got, q, kc, vc, scales, table, [n])
    for _ in range(5):
        assert np.array_equal(run(q, cache, table, [n]), got)


@pytest.mark.parametrize("layout", ["token", "mixed"])
@pytest.mark.parametrize("H,Hkv,D", [(14, 2, 64), (28, 4, 128)])
def test_strides(layout, H, Hkv, D):
    rng = np.random.default_rng(5)
    lens = [77, 0, 640, 33]
    q = half(rng, (4, H, D))
    table, pages = make_table(rng, lens, 48)
    kc, vc, scales = make_pool(rng, pages, Hkv, 48, D)
    wide = torch.full((4, H * D + 2 * Hkv * D), 7.0, dtype=torch.float16, device="cuda")
    wide[:, :H * D] = torch.from_numpy(q.reshape(4, -1)).cuda()
    got = run(q, to_cache(kc, vc, scales, layout), table, lens, q_stride=wide.stride(0), qd=wide)
    check(got, q, kc, vc, scales, table, lens)
    assert np.array_equal(got, run(q, to_cache(kc, vc, scales), table, lens))


@pytest.mark.parametrize("layout", ["token", "mixed", "heads", "padded"])
@pytest.mark.parametrize("H,Hkv,D", [(14, 2, 64), (24, 2, 64), (28, 4, 128), (16, 1, 128)])
def test_strides_long(layout, H, Hkv, D):
    """The shapes for long calls on every layout: the bits are those of the plain one."""
    rng = np.random.default_rng(16)
    lens = [77, 0, 1640, 33]
    q = half(rng, (4, H, D))
    table, pages = make_table(rng, lens, 48)
    kc, vc, scales = make_pool(rng, pages, Hkv, 48, D)
    got = run_long(q, to_cache(kc, vc, scales, layout), table, lens, 48)
    check(got, q, kc, vc, scales, table, lens, long=True)
    assert np.array_equal(got, run_long(q, to_cache(kc, vc, scales), table, lens, 48))
    short = run(q, to_cache(kc, vc, scales, layout), table, lens)
    check(short, q, kc, vc, scales, table, lens)


def test_one_page_pool_and_one_head():
    """Dimensions of one element, whose strides mean nothing."""
    rng = np.random.default_rng(6)
    q = half(rng, (1, 4, 64))
    kc, vc, scales = make_pool(rng, 1, 1, 16, 64)
    table = np.zeros((1, 1), np.int32)
    check(run(q, to_cache(kc, vc, scales), table, [9]), q, kc, vc, scales, table, [9])


def test_pages_outside_the_pool_read_as_zero_rows():
    rng = np.random.default_rng(7)
    lens = [200, 130]
    q = half(rng, (2, 12, 128))
    table, pages = make_table(rng, lens, 32)
    kc, vc, scales = make_pool(rng, pages, 2, 32, 128)
    table[0, 2], table[1, 0], table[1, 4] = -1, pages, 2**31 - 1
    check(run(q, to_cache(kc, vc, scales), table, lens), q, kc, vc, scales, table, lens)


def test_lengths_are_cut_to_the_bound_and_negative_ones_are_empty():
    rng = np.random.default_rng(8)
    lens = [500, -3, 64]
    q = half(rng, (3, 12, 128))
    table, pages = make_table(rng, [512, 0, 64], 64, width=8)
    kc, vc, scales = make_pool(rng, pages, 2, 64, 128)
    got = run(q, to_cache(kc, vc, scales), table, lens, max_kv_len=100)
    check(got, q, kc, vc, scales, table, [100, 0, 64])
    assert (got[1] == 0).all()
    assert (run(q, to_cache(kc, vc, scales), table, lens, max_kv_len=0) == 0).all()


def test_batches_beyond_one_launch():
    rng = np.random.default_rng(9)
    lens = [int(x) for x in rng.integers(0, 90, 1201)]
    q = half(rng, (len(lens), 8, 64))
    table, pages = make_table(rng, lens, 16)
    kc, vc, scales = make_pool(rng, pages, 8, 16, 64)
    clean = scales.copy()
    poison(table, lens, 16, scales)
    check(run(q, to_cache(kc, vc, scales), table, lens), q, kc, vc, clean, table, lens, long=True)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_wide_range_of_scales(D, long):
    """V rows whose scales differ by many powers of two, rows of zero scale (all
    their values the bias), the two groups of D = 128 far apart: the large scores
    and values are neither lost nor blown up, small groups keep their bits."""
    rng = np.random.default_rng(10)
    lens = [900, 31, 64]
    q = half(rng, (3, 28, D))
    table, pages = make_table(rng, lens, 32)
    kc, vc, scales = make_pool(rng, pages, 4, 32, D)
    up = np.exp2(rng.integers(-12, 8, scales.shape[:3])).astype(np.float16)
    scales[:, :, :, 1] *= up[..., None, None]
    if D == 128:
        scales[:, :, :, 1, 1] *= np.float16(2.0 ** -8)
    scales[:, :, :, 0] *= np.exp2(rng.integers(-3, 3, scales.shape[:3])).astype(np.float16)[..., None, None]
    scales[table[0, 3], :, 5:20, :, :, 0] = 0
    scales[table[2, :2], 1, :, 1, :, 0] = 0            # a whole sequence's V of one kv head: biases only
    cache = to_cache(kc, vc, scales)
    got = run_long(q, cache, table, lens, 32) if long else run(q, cache, table, lens)
    check(got, q, kc, vc, scales, table, lens, long, norm=False)


def test_many_small_probabilities_count():
    """One position 2^17 times as likely as each of 60000 others, whose mass
    together is half of it: as fp16 fractions of the largest they would lose
    bits, shifted they do not."""
    n, D = 60001, 64
    kc = np.zeros((938, 1, 64, D // 2), np.uint8)
    vc = np.full((938, 1, 64, D // 2), 0xaa, np.uint8)
    kc[0, 0, 0] = 0xff
    vc[0, 0, 0] = 0x22
    scales = np.zeros((938, 1, 64, 2, 1, 2), np.float16)
    scales[..., 0] = 1
    q = np.zeros((1, 1, D), np.float16)
    q[0, 0, :] = 17 * np.log(2) / (15 * 8)
    table = np.arange(938, dtype=np.int32)[None]
    got = run(q, to_cache(kc, vc, scales), table, [n])
    check(got, q, kc, vc, scales, table, [n])


@pytest.mark.parametrize("long", [False, True])
def test_references_move(long):
    """Scores that climb by hundreds along the sequence: every step outgrows the
    references of the one before."""
    rng = np.random.default_rng(15)
    lens = [600, 333]
    q = np.abs(half(rng, (2, 12, 128))) + np.float16(1)
    table, pages = make_table(rng, lens, 32)
    kc, vc, scales = make_pool(rng, pages, 2, 32, 128)
    for b in range(2):
        for j in range(-(-lens[b] // 32)):
            scales[table[b, j], :, :, 0, :, 1] += (np.arange(32) * 0.25 + 8 * j)[:, None].astype(np.float16)
    cache = to_cache(kc, vc, scales)
    got = run_long(q, cache, table, lens, 32) if long else run(q, cache, table, lens)
    check(got, q, kc, vc, scales, table, lens, long, norm=False)


def test_nan_stays_where_it_belongs():
    """A row with a NaN scale or bias spoils the query heads of its own kv head
    and sequence (a V group its own dims), no other."""
    rng = np.random.default_rng(11)
    lens = [300, 300, 90]
    q = half(rng, (3, 12, 128))
    table, pages = make_table(rng, lens, 32)
    kc, vc, scales = make_pool(rng, pages, 2, 32, 128)
    clean = run(q, to_cache(kc, vc, scales), table, lens)
    s2 = scales.copy()
    s2[table[0, 4], 1, 7, 0, 1, 0] = np.nan    # sequence 0, kv head 1: K, a scale
    s2[table[1, 0], 0, 31, 1, 0, 1] = np.nan   # sequence 1, kv head 0: V, a bias of the first group
    got = run(q, to_cache(kc, vc, s2), table, lens)
    assert np.isnan(got[0, 6:]).all() and np.isnan(got[1, :6, :64]).all()
    assert np.array_equal(got[0, :6], clean[0, :6]) and np.array_equal(got[1, 6:], clean[1, 6:])
    assert np.array_equal(got[2], clean[2])


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_query_extremes(D, long):
    """Heads of zeros, of the smallest and of large halves, of one large
    element; NaN and infinity spoil their own head only."""
    rng = np.random.default_rng(D)
    lens = [333, 40]
    q = half(rng, (2, 7, D))
    q[0, 0] = 0
    q[0, 1] = np.float16(6e-8)
    q[0, 2] *= np.float16(300)
    q[0, 3, 1:] = 0
    q[1, 4] = np.float16(-2.0)
    table, pages = make_table(rng, lens, 32)
    kc, vc, scales = make_pool(rng, pages, 1, 32, D)
    cache = to_cache(kc, vc, scales)

    def call(x):
        return run_long(x, cache, table, lens, 32) if long else run(x, cache, table, lens)

    clean = call(q)
    check(clean, q, kc, vc, scales, table, lens, long, norm=False)
    bad = q.copy()
    bad[0, 5, 3], bad[1, 6, 0] = np.nan, np.inf
    got = call(bad)
    assert np.isnan(got[0, 5]).all() and np.isnan(got[1, 6]).all()
    keep = np.ones((2, 7), bool)
    keep[0, 5] = keep[1, 6] = False
    assert np.array_equal(got[keep], clean[keep])


def test_offsets_past_32_bits():
    """A pool of 5 GB of codes of K and of V: the last pages lie past 2^32 bytes."""
    rng = np.random.default_rng(12)
    Hkv, D, ps, pages = 4, 128, 128, 160000
    lens = [700, 100]
    q = half(rng, (2, 28, D))
    small, _ = make_table(rng, lens, ps, spare=0)
    kc, vc, scales = make_pool(rng, 7, Hkv, ps, D)
    ids = np.array([159999, 3, 65537, 159998, 140000, 70001, 0])
    k, v = (torch.empty((pages, Hkv, ps, D // 2), dtype=torch.uint8, device="cuda") for _ in range(2))
    sc = torch.full((pages, Hkv, ps, 2, 2, 2), float("nan"), dtype=torch.float16, device="cuda")
    at = torch.from_numpy(ids).cuda()
    k[at], v[at], sc[at] = (torch.from_numpy(x).cuda() for x in (kc, vc, scales))
    table = np.where(small >= 0, ids[np.clip(small, 0, 6)], 0).astype(np.int32)
    got = run(q, A.KV4Cache(k, v, sc), table, lens)
    check(got, q, kc, vc, scales, np.clip(small, 0, 6), lens)


def test_side_stream_and_graph():
    """On a stream of its own, captured and replayed with new lengths and q."""
    rng = np.random.default_rng(13)
    lens = [300, 17, 0, 1000]
    q = half(rng, (4, 28, 128))
    table, pages = make_table(rng, lens, 64)
    kc, vc, scales = make_pool(rng, pages, 4, 64, 128)
    cache = to_cache(kc, vc, scales)
    qd, td = torch.from_numpy(q).cuda(), torch.from_numpy(table).cuda()
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(qd)
    A.reserve_workspace(A.kv4_workspace_size(4, 28, 4, 128, 1000))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    call = lambda: A.decode_attn_paged_kv4(qd, cache, td, ld, out, 4, 28, table.shape[1], 1000, stream=s)  # noqa: E731
    with torch.cuda.stream(s):
        for _ in range(3):
            call()
        s.synchronize()
        check(out.cpu().numpy(), q, kc, vc, scales, table, lens)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call()
    q2, lens2 = half(rng, q.shape), [299, 1, 5, 640]
    qd.copy_(torch.from_numpy(q2))
    ld.copy_(torch.tensor(lens2, dtype=torch.int32))
    table[2, 0] = table[0, 0]
    td.copy_(torch.from_numpy(table))
    torch.cuda.synchronize()
    for _ in range(2):
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check(out.cpu().numpy(), q2, kc, vc, scales, table, lens2)
    assert A.device_error() == 0


def test_refusals():
    rng = np.random.default_rng(14)
    kc, vc, scales = make_pool(rng, 4, 2, 32, 64)
    cache = to_cache(kc, vc, scales)
    q = torch.zeros((2, 8, 64), dtype=torch.float16, device="cuda")
    t = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    n = torch.ones(2, dtype=torch.int32, device="cuda")
    for B, H, mb, mk, qs in ((0, 8, 2, 64, 0), (2, 7, 2, 64, 0), (2, 8, 2, 65, 0), (2, 8, 0, 0, 0), (2, 8, 2, 64, 100)):
        with pytest.raises(ForgeRTError, match="invalid argument"):
            A.decode_attn_paged_kv4(q, cache, t, n, q, B, H, mb, mk, q_stride=qs)
    with pytest.raises(ForgeRTError, match="misaligned"):
        A.decode_attn_paged_kv4(q.data_ptr() + 8, cache, t, n, q, 2, 8, 2, 64)
    with pytest.raises(ValueError):
        A.decode_attn_paged_kv4(q.cpu(), cache, t, n, q, 2, 8, 2, 64)
