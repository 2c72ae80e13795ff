"""GPU tests of decode attention over the 8-bit paged cache
(fr_decode_attn_paged_kv8) against the 64-bit oracle (oracle.kv8).

Error bound, from the kernel's arithmetic: the output is rounded to fp16 once
(2^-11 of itself), each probability enters the P.V product as one fp16
(2^-11), and a score carries the rounding of a D-term fp32 sum (at most
D 2^-23 of sum |q_i k_i| / sqrt(D)), which moves a probability by that
relative amount, in the numerator and in the sum; 2^-13 stands for the
exponentials and the fp32 merges.  With M = sum_t p_t |v_t|:
  |x - r| <= 2^-11 |r| + (2^-11 + 2^-13 + 2 D 2^-23 S) M + 1e-7.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from forgert_b200 import attention as A
from forgert_b200._lib import ForgeRTError
from oracle import kv8 as O

pytestmark = pytest.mark.gpu

TORCH = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
SHAPES = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (8, 8, 64), (16, 1, 128)]


def make_pool(rng, pages, Hkv, ps, D, code):
    """Raw codes and scales; e4m3 codes are finite."""
    codes = [rng.integers(0, 256, (pages, Hkv, ps, D), dtype=np.uint8) for _ in range(2)]
    for c in codes:
        if code == "e4m3":
            c[(c & 127) == 127] = 0x3c
        else:
            c[c == 128] = 0
    scales = np.exp(0.4 * rng.standard_normal((pages, Hkv, ps // 16, 2))).astype(np.float32)
    return codes[0], codes[1], scales * np.float32((2.5 if code == "int8" else 1.5) / O.KMAX[code])


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


def poison(table, lens, ps, codes, scales, code):
    """What nobody owns must not matter: NaN codes (or the largest) behind each
    end and in spare pages, NaN scales in blocks without rows."""
    owned = np.zeros((codes[0].shape[0], ps), bool)
    for b, n in enumerate(lens):
        for j in range(-(-max(0, n) // ps)):
            owned[table[b, j], :max(0, min(ps, n - j * ps))] = True
    for c in codes:
        c[np.broadcast_to(~owned[:, None, :, None], c.shape)] = 0x7f
    blocks = owned.reshape(len(owned), ps // 16, 16).any(2)
    scales[np.broadcast_to(~blocks[:, None, :, None], scales.shape)] = np.nan


def to_cache(kc, vc, scales, code, layout="head"):
    def lay(c):
        x = torch.from_numpy(c).cuda()
        if layout == "token":                          # [P, ps, Hkv, D] pages
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        return x
    if layout == "mixed":                              # K and V pages side by side in one allocation
        both = torch.stack([torch.from_numpy(kc), torch.from_numpy(vc)], 1).cuda()
        k, v = both[:, 0], both[:, 1]
    else:
        k, v = lay(kc), lay(vc)
    return A.KV8Cache(k.view(TORCH[code]), v.view(TORCH[code]), torch.from_numpy(scales).cuda())


def run(q, cache, table, lens, max_kv_len=None, stream=None, q_stride=0, qd=None):
    B, H, D = q.shape
    qd = torch.from_numpy(q).cuda() if qd is None else qd
    out = torch.full((B, H, D), float("nan"), dtype=torch.float16, device="cuda")
    td, ld = torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    mk = max(0, max(lens)) if max_kv_len is None else max_kv_len
    A.decode_attn_paged_kv8(qd, cache, td, ld, out, B, H, table.shape[1], mk, q_stride=q_stride, stream=stream)
    torch.cuda.synchronize()
    assert A.device_error() == 0
    return out.cpu().numpy()


def check(got, q, kc, vc, scales, code, table, lens):
    r, mass, big = O.attention(q, O.values(kc, scales, 0, code), O.values(vc, scales, 1, code), table, lens)
    D = q.shape[2]
    tol = 2.0 ** -11 * np.abs(r) + (2.0 ** -11 + 2.0 ** -13 + 2 * D * 2.0 ** -23 * big) * mass + 1e-7
    err = np.abs(got.astype(np.float64) - r)
    assert np.isfinite(got).all()
    assert (err <= tol).all(), f"max err / tol {(err / tol).max():.3f}"


def half(rng, shape):
    return rng.standard_normal(shape).astype(np.float16)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("page_size", [16, 48, 64, 128, 256])
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
def test_matches_oracle(H, Hkv, D, page_size, code):
    rng = np.random.default_rng(page_size * 1000 + H * 10 + D)
    lens = [0, 1, 15, 16, 17, 127, 128, 129, page_size, page_size + 1, 700, 0, 2049, 3 * page_size - 1]
    q = half(rng, (len(lens), H, D))
    table, pages = make_table(rng, lens, page_size)
    kc, vc, scales = make_pool(rng, pages, Hkv, page_size, D, code)
    poison(table, lens, page_size, (kc, vc), scales, code)
    got = run(q, to_cache(kc, vc, scales, code), table, lens)
    assert (got[[0, 11]] == 0).all()
    check(got, q, kc, vc, scales, code, table, lens)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (3, 3), (5, 1), (8, 1), (9, 1), (10, 2), (24, 1), (33, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_group_sizes(D, H, Hkv, code):
    rng = np.random.default_rng(H * 7 + D)
    lens = [1, 40, 333]
    q = half(rng, (3, H, D))
    table, pages = make_table(rng, lens, 32)
    kc, vc, scales = make_pool(rng, pages, Hkv, 32, D, code)
    check(run(q, to_cache(kc, vc, scales, code), table, lens), q, kc, vc, scales, code, table, lens)


@pytest.mark.parametrize("n", [1, 2, 16, 129, 512, 1000, 4096, 20000, 65536])
@pytest.mark.parametrize("H,Hkv,D,code", [(14, 2, 64, "int8"), (28, 4, 128, "e4m3")])
def test_one_sequence(n, H, Hkv, D, code):
    """From one token to long ranges that many CTAs share; the bits do not
    depend on who merges."""
    rng = np.random.default_rng(n)
    q = half(rng, (1, H, D))
    table, pages = make_table(rng, [n], 64)
    kc, vc, scales = make_pool(rng, pages, Hkv, 64, D, code)
    cache = to_cache(kc, vc, scales, code)
    got = run(q, cache, table, [n])
    check(got, q, kc, vc, scales, code, table, [n])
    for _ in range(5):
        assert np.array_equal(run(q, cache, table, [n]), got)


@pytest.mark.parametrize("layout", ["token", "mixed"])
@pytest.mark.parametrize("H,Hkv,D,code", [(14, 2, 64, "e4m3"), (28, 4, 128, "int8")])
def test_strides(layout, H, Hkv, D, code):
    rng = np.random.default_rng(5)
    lens = [77, 0, 640, 33]
    q = half(rng, (4, H, D))
    table, pages = make_table(rng, lens, 48)
    kc, vc, scales = make_pool(rng, pages, Hkv, 48, D, code)
    poison(table, lens, 48, (kc, vc), scales, code)
    wide = torch.full((4, H * D + 2 * Hkv * D), 7.0, dtype=torch.float16, device="cuda")
    wide[:, :H * D] = torch.from_numpy(q.reshape(4, -1)).cuda()
    cache = to_cache(kc, vc, scales, code, layout)
    got = run(q, cache, table, lens, q_stride=wide.stride(0), qd=wide)
    check(got, q, kc, vc, scales, code, table, lens)
    assert np.array_equal(got, run(q, to_cache(kc, vc, scales, code), table, lens))


def test_one_page_pool_and_one_head():
    """Dimensions of one element, whose strides mean nothing."""
    rng = np.random.default_rng(6)
    q = half(rng, (1, 4, 64))
    kc, vc, scales = make_pool(rng, 1, 1, 16, 64, "int8")
    table = np.zeros((1, 1), np.int32)
    check(run(q, to_cache(kc, vc, scales, "int8"), table, [9]), q, kc, vc, scales, "int8", table, [9])


def test_pages_outside_the_pool_read_as_zero_rows():
    rng = np.random.default_rng(7)
    lens = [200, 130]
    q = half(rng, (2, 12, 128))
    table, pages = make_table(rng, lens, 32)
    kc, vc, scales = make_pool(rng, pages, 2, 32, 128, "e4m3")
    table[0, 2], table[1, 0], table[1, 4] = -1, pages, 2**31 - 1
    check(run(q, to_cache(kc, vc, scales, "e4m3"), table, lens), q, kc, vc, scales, "e4m3", table, lens)


def test_lengths_are_cut_to_the_bound_and_negative_ones_are_empty():
    rng = np.random.default_rng(8)
    lens = [500, -3, 64]
    q = half(rng, (3, 12, 128))
    table, pages = make_table(rng, [512, 0, 64], 64, width=8)
    kc, vc, scales = make_pool(rng, pages, 2, 64, 128, "int8")
    got = run(q, to_cache(kc, vc, scales, "int8"), table, lens, max_kv_len=100)
    check(got, q, kc, vc, scales, "int8", table, [100, 0, 64])
    assert (got[1] == 0).all()
    assert (run(q, to_cache(kc, vc, scales, "int8"), table, lens, max_kv_len=0) == 0).all()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_batches_beyond_one_launch(code):
    rng = np.random.default_rng(9)
    lens = [int(x) for x in rng.integers(0, 90, 1201)]
    q = half(rng, (len(lens), 8, 64))
    table, pages = make_table(rng, lens, 16)
    kc, vc, scales = make_pool(rng, pages, 8, 16, 64, code)
    poison(table, lens, 16, (kc, vc), scales, code)
    check(run(q, to_cache(kc, vc, scales, code), table, lens), q, kc, vc, scales, code, table, lens)


def test_wide_range_of_scales():
    """Blocks whose scales differ by many powers of two: the large scores and
    the large values are neither lost nor blown up."""
    rng = np.random.default_rng(10)
    lens = [900, 31]
    q = half(rng, (2, 28, 128))
    table, pages = make_table(rng, lens, 32)
    kc, vc, scales = make_pool(rng, pages, 4, 32, 128, "int8")
    scales[..., 1] *= np.exp2(rng.integers(-30, 6, scales.shape[:3])).astype(np.float32)
    scales[..., 0] *= np.exp2(rng.integers(-6, 2, scales.shape[:3])).astype(np.float32)
    scales[0, :, 0] = 0.0
    r, mass, big = O.attention(q, O.values(kc, scales, 0, "int8"), O.values(vc, scales, 1, "int8"), table, lens)
    got = run(q, to_cache(kc, vc, scales, "int8"), table, lens).astype(np.float64)
    tol = 2.0 ** -11 * np.abs(r) + (2.0 ** -11 + 2.0 ** -13 + 256 * 2.0 ** -23 * big) * mass + 1e-7
    assert (np.abs(got - r) <= tol).all()


def test_many_small_probabilities_count():
    """One position 2^17 times as likely as each of 60000 others, whose mass
    together is half of it: as fp16 fractions of the largest they would lose
    bits, shifted they do not."""
    n, D = 60001, 64
    kc = np.zeros((938, 1, 64, D), np.uint8)
    vc = np.full((938, 1, 64, D), 32, np.uint8)
    kc[0, 0, 0] = 127
    vc[0, 0, 0] = (-96) & 255
    scales = np.ones((938, 1, 4, 2), np.float32)
    q = np.zeros((1, 1, D), np.float16)
    q[0, 0, :] = 17 * np.log(2) / (127 * 8)
    table = np.arange(938, dtype=np.int32)[None]
    got = run(q, to_cache(kc, vc, scales, "int8"), table, [n])
    check(got, q, kc, vc, scales, "int8", table, [n])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_nan_and_infinity_stay_where_they_belong(code):
    """A block with a NaN or infinite scale (or a NaN code) spoils the query
    heads of its own kv head and sequence, no other."""
    rng = np.random.default_rng(11)
    lens = [300, 300, 90]
    q = half(rng, (3, 12, 128))
    table, pages = make_table(rng, lens, 32)
    kc, vc, scales = make_pool(rng, pages, 2, 32, 128, code)
    clean = run(q, to_cache(kc, vc, scales, code), table, lens)
    s2, k2 = scales.copy(), kc.copy()
    s2[table[0, 4], 1, 0, 0] = np.nan          # sequence 0, kv head 1: K
    s2[table[1, 0], 0, 1, 1] = np.inf          # sequence 1, kv head 0: V
    vc[table[1, 0], 0, 16, 3] = 0              # ... with a zero among its codes
    k2[table[2, 0], 1, 3, 5] = 0x7f if code == "e4m3" else k2[table[2, 0], 1, 3, 5]
    got = run(q, to_cache(k2, vc, s2, code), table, lens)
    assert np.isnan(got[0, 6:]).all() and not np.isfinite(got[1, :6]).any()
    assert np.isnan(got[1, :6, 3]).all()
    assert np.array_equal(got[0, :6], clean[0, :6]) and np.array_equal(got[1, 6:], clean[1, 6:])
    assert np.array_equal(got[2, :6], clean[2, :6])
    if code == "e4m3":
        assert np.isnan(got[2, 6:]).all()


def test_offsets_past_32_bits():
    """A pool of 5 GB of K and of V: the last pages lie past 2^32 bytes."""
    rng = np.random.default_rng(12)
    Hkv, D, ps, pages = 4, 128, 128, 80000
    size = (pages, Hkv, ps, D)
    lens = [700, 100]
    q = half(rng, (2, 28, D))
    small, _ = make_table(rng, lens, ps, spare=0)
    kc, vc, scales = make_pool(rng, 7, Hkv, ps, D, "e4m3")
    ids = np.array([79999, 3, 65537, 79998, 40000, 70001, 0])
    k, v = (torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2))
    sc = torch.full((pages, Hkv, ps // 16, 2), float("nan"), device="cuda")
    at = torch.from_numpy(ids).cuda()
    k[at], v[at], sc[at] = (torch.from_numpy(x).cuda() for x in (kc, vc, scales))
    table = np.where(small >= 0, ids[np.clip(small, 0, 6)], 0).astype(np.int32)
    cache = A.KV8Cache(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), sc)
    got = run(q, cache, table, lens)
    check(got, q, kc, vc, scales, "e4m3", np.clip(small, 0, 6), lens)


def test_side_stream_and_graph():
    """On a stream of its own, captured and replayed with new lengths and q."""
    rng = np.random.default_rng(13)
    lens = [300, 17, 0, 1000]
    q = half(rng, (4, 28, 128))
    table, pages = make_table(rng, lens, 64)
    kc, vc, scales = make_pool(rng, pages, 4, 64, 128, "int8")
    cache = to_cache(kc, vc, scales, "int8")
    qd, td = torch.from_numpy(q).cuda(), torch.from_numpy(table).cuda()
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(qd)
    A.reserve_workspace(A.kv8_workspace_size(4, 28, 4, 128, 1000))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    call = lambda: A.decode_attn_paged_kv8(qd, cache, td, ld, out, 4, 28, table.shape[1], 1000, stream=s)  # noqa: E731
    with torch.cuda.stream(s):
        for _ in range(3):
            call()
        s.synchronize()
        check(out.cpu().numpy(), q, kc, vc, scales, "int8", table, lens)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call()
    q2, lens2 = half(rng, q.shape), [299, 1, 5, 640]
    table2, _ = make_table(np.random.default_rng(13), lens, 64)
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
        check(out.cpu().numpy(), q2, kc, vc, scales, "int8", table, lens2)
    assert A.device_error() == 0


def test_refusals():
    rng = np.random.default_rng(14)
    kc, vc, scales = make_pool(rng, 4, 2, 32, 64, "int8")
    cache = to_cache(kc, vc, scales, "int8")
    q = torch.zeros((2, 8, 64), dtype=torch.float16, device="cuda")
    t = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    n = torch.ones(2, dtype=torch.int32, device="cuda")
    for B, H, mb, mk, qs in ((0, 8, 2, 64, 0), (2, 7, 2, 64, 0), (2, 8, 2, 65, 0), (2, 8, 0, 0, 0), (2, 8, 2, 64, 100)):
        with pytest.raises(ForgeRTError, match="invalid argument"):
            A.decode_attn_paged_kv8(q, cache, t, n, q, B, H, mb, mk, q_stride=qs)
    with pytest.raises(ForgeRTError, match="misaligned"):
        A.decode_attn_paged_kv8(q.data_ptr() + 8, cache, t, n, q, 2, 8, 2, 64)
    with pytest.raises(ValueError):
        A.decode_attn_paged_kv8(q.cpu(), cache, t, n, q, 2, 8, 2, 64)


# ------------------------------------------------- the shape for long calls
# A call whose bound max_kv_len allows many tiles runs another shape of the
# kernel; the lengths themselves may be short.  With int8 codes and up to 8
# heads it takes q in 16-bit fixed point on the head's largest value: an
# element is off by 1 / 65278 of that, a score by at most
# max|q| sum |k_i| / (65278 sqrt(D)), which the bound doubles as it does the
# rounding of the scores' sums.

def run_long(q, cache, table, lens, page_size):
    bound = (1 << 19) // page_size * page_size
    wide = np.full((len(lens), bound // page_size), -1, np.int32)
    wide[:, :table.shape[1]] = table
    return run(q, cache, wide, lens, max_kv_len=bound)


def check_long(got, q, kc, vc, scales, code, table, lens):
    k = O.values(kc, scales, 0, code)
    r, mass, big = O.attention(q, k, O.values(vc, scales, 1, code), table, lens)
    B, H, D = q.shape
    fixed = np.zeros_like(big)
    for b, n in enumerate(lens):
        ids = np.asarray(table[b][:-(-max(0, n) // kc.shape[2])], np.int64)
        for j in range(kc.shape[1]):
            rows = np.abs(k[ids, j]).sum(-1).reshape(-1)[:max(0, n)]
            g = H // kc.shape[1]
            if len(rows):
                fixed[b, j * g:(j + 1) * g, 0] = rows.max() * np.abs(q[b, j * g:(j + 1) * g].astype(np.float64)).max(-1)
    fixed /= 65278 * np.sqrt(D)
    tol = 2.0 ** -11 * np.abs(r) + (2.0 ** -11 + 2.0 ** -13 + 2 * D * 2.0 ** -23 * big + 2 * fixed) * mass + 1e-7
    err = np.abs(got.astype(np.float64) - r)
    assert np.isfinite(got).all()
    assert (err <= tol).all(), f"max err / tol {(err / tol).max():.3f}"


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("H,Hkv,D", SHAPES + [(24, 2, 64), (9, 1, 64), (33, 1, 128)])
def test_long_shape(H, Hkv, D, code):
    rng = np.random.default_rng(H + D)
    lens = [0, 1, 15, 16, 17, 129, 700, 4097, 0, 2049, 20000]
    q = half(rng, (len(lens), H, D))
    table, pages = make_table(rng, lens, 48)
    kc, vc, scales = make_pool(rng, pages, Hkv, 48, D, code)
    poison(table, lens, 48, (kc, vc), scales, code)
    cache = to_cache(kc, vc, scales, code)
    got = run_long(q, cache, table, lens, 48)
    assert (got[[0, 8]] == 0).all()
    check_long(got, q, kc, vc, scales, code, table, lens)
    for _ in range(3):
        assert np.array_equal(run_long(q, cache, table, lens, 48), got)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_query_extremes(D, long, code):
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
    kc, vc, scales = make_pool(rng, pages, 1, 32, D, code)
    cache = to_cache(kc, vc, scales, code)

    def call(x):
        return run_long(x, cache, table, lens, 32) if long else run(x, cache, table, lens)

    clean = call(q)
    check_long(clean, q, kc, vc, scales, code, table, lens)
    bad = q.copy()
    bad[0, 5, 3], bad[1, 6, 0] = np.nan, np.inf
    got = call(bad)
    assert np.isnan(got[0, 5]).all() and np.isnan(got[1, 6]).all()
    keep = np.ones((2, 7), bool)
    keep[0, 5] = keep[1, 6] = False
    assert np.array_equal(got[keep], clean[keep])


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_long_shape_wide_scales_and_zero_blocks(code):
    """Blocks whose scales differ by many powers of two, blocks of zero scale."""
    rng = np.random.default_rng(21)
    lens = [900, 31, 64]
    q = half(rng, (3, 28, 128))
    table, pages = make_table(rng, lens, 32)
    kc, vc, scales = make_pool(rng, pages, 4, 32, 128, code)
    scales[..., 1] *= np.exp2(rng.integers(-30, 6, scales.shape[:3])).astype(np.float32)
    scales[..., 0] *= np.exp2(rng.integers(-6, 2, scales.shape[:3])).astype(np.float32)
    scales[table[0, 3], :, 0] = 0.0
    scales[table[2, :2], 1, :, 1] = 0.0           # a whole sequence's V of one kv head
    got = run_long(q, to_cache(kc, vc, scales, code), table, lens, 32)
    check_long(got, q, kc, vc, scales, code, table, lens)
    assert (got[2, 7:14] == 0).all()
