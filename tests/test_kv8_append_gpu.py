"""GPU tests of the 8-bit cache's prologue (fr_qkv_rope_append_kv8) and
read-back (fr_kv8_gather).

The oracle follows the operator's 32-bit operations one by one, so the cache
(codes and scales) is compared exactly, and so are the fp16 outputs; beside
that the outputs are held to the 64-bit rotation within half an fp16 ulp plus
the fp32 roundings of a three-operation sum:
  |x - r| <= 2^-11 |r| + 2^-22 (|a| + |b|) (+ 2^-25, fp16's smallest step).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from forgert_b200 import attention as A
from forgert_b200._lib import FR_ERR_INVALID_ARG, ForgeRTError, load
from oracle import kv8 as O

pytestmark = pytest.mark.gpu

TORCH = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
ROWS = 5000


def tables(D):
    a = np.arange(ROWS)[:, None] * 1e6 ** (-2.0 * np.arange(D // 2) / D)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def half(rng, shape, scale=1.0):
    return (rng.standard_normal(shape) * scale).astype(np.float16)


def dev(x):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()


class Pool:
    """A cache on the device and its copy for the oracle."""

    def __init__(self, rng, pages, Hkv, ps, D, code, layout="head"):
        self.code, self.ps = code, ps
        self.k, self.v = (rng.integers(0, 127, (pages, Hkv, ps, D), dtype=np.uint8) for _ in range(2))
        self.scales = np.exp(rng.standard_normal((pages, Hkv, ps // 16, 2))).astype(np.float32)
        self.scales *= np.float32(2.0 / O.KMAX[code])

        def lay(x):
            x = dev(x)
            return x.transpose(1, 2).contiguous().transpose(1, 2) if layout == "token" else x
        self.kd, self.vd, self.sd = lay(self.k), lay(self.v), dev(self.scales)
        self.cache = A.KV8Cache(self.kd.view(TORCH[code]), self.vd.view(TORCH[code]), self.sd)

    def same(self):
        assert np.array_equal(self.sd.cpu().numpy(), self.scales, equal_nan=True)
        for got, want in ((self.kd, self.k), (self.vd, self.v)):
            got = got.cpu().numpy()
            bad = np.argwhere(got != want)
            assert not len(bad), (len(bad), bad[:4].tolist())


def runs_of(rng, spans, pages, ps):
    """Slots of tokens [(held, new)] on shuffled pages, and their positions."""
    ids = list(rng.permutation(pages))
    slots, pos = [], []
    for held, new in spans:
        table = [ids.pop() for _ in range(-(-(held + new) // ps))]
        for t in range(held, held + new):
            slots.append(int(table[t // ps]) * ps + t % ps)
            pos.append(t)
    return np.array(slots, np.int64), np.array(pos, np.int32)


def do(rng, pool, H, Hkv, D, slots, positions, axis, bias=True, keep=True, in_place=False, strided=False, scale=1.0):
    T = len(slots)
    q, k, v = half(rng, (T, H, D), scale), half(rng, (T, Hkv, D), scale), half(rng, (T, Hkv, D), scale)
    biases = [half(rng, (n, D)) if bias else None for n in (H, Hkv, Hkv)]
    cos, sin = tables(D)
    positions = np.atleast_2d(positions)
    want = O.append(q, k, v, biases, cos, sin, positions, axis, slots, pool.k, pool.v, pool.scales, pool.code)
    strides = None
    if strided:                                          # q, k, v of a token in one row, outputs apart
        row = torch.full((T, (H + 2 * Hkv) * D + 12), 9.0, dtype=torch.float16, device="cuda")
        row[:, :(H + 2 * Hkv) * D] = torch.cat([dev(x).flatten(1) for x in (q, k, v)], 1)
        w = row.stride(0)
        at = [row.data_ptr(), row.data_ptr() + 2 * H * D, row.data_ptr() + 2 * (H + Hkv) * D]
        strides = [w, w, w, H * D + 4, Hkv * D, Hkv * D + 8]
    else:
        at = [dev(x) for x in (q, k, v)]
    if in_place:
        outs, views = list(at), list(at)
        if not keep:
            outs[1] = outs[2] = None
    else:
        widths = strides[3:] if strided else [H * D, Hkv * D, Hkv * D]
        raw = [torch.full((T, n), float("nan"), dtype=torch.float16, device="cuda") for n in widths]
        views = [x[:, :n * D].unflatten(1, (n, D)) for x, n in zip(raw, (H, Hkv, Hkv))]
        outs = raw if keep else [raw[0], None, None]
    A.qkv_rope_append_kv8(*at, *outs, dev(cos), dev(sin), dev(positions.astype(np.int32)), dev(slots), pool.cache, T, H,
                          ROWS, *[dev(b) for b in biases], num_axes=len(positions),
                          freq_axis=bytes(axis) if len(positions) > 1 else None, token_strides=strides)
    torch.cuda.synchronize()
    assert A.device_error() == 0
    real = slots >= 0
    used = views if keep else views[:1]
    for i, (got, r) in enumerate(zip(used, want)):
        g = got.cpu().numpy()[real]
        assert np.array_equal(g, r[real].astype(np.float16)), i
        x, b = (q, k, v)[i], biases[i]
        if i < 2:
            r64 = O.rotate64(x, b, positions, axis, cos, sin)[real]
            e = np.abs(x.astype(np.float64)) + (0 if b is None else np.abs(b.astype(np.float64)))
            e = (e + np.roll(e, D // 2, -1))[real]
            assert (np.abs(g - r64) <= 2.0 ** -11 * np.abs(r64) + 2.0 ** -22 * e + 2.0 ** -25).all()
    pool.same()
    return want


AXES3 = lambda D: [0] * (D // 8) + [1] * (D // 2 - 2 * (D // 8)) + [2] * (D // 8)  # noqa: E731
SPANS = [
    [(0, 1)], [(5, 1)], [(15, 1)], [(16, 1)], [(0, 16)], [(3, 13)], [(9, 8)], [(0, 100)], [(31, 2)],
    [(i * 7 % 33, 1) for i in range(40)],
    [(0, 37), (12, 1), (100, 3), (15, 50), (1, 15), (16, 16), (47, 1)],
]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("spans", SPANS)
@pytest.mark.parametrize("H,Hkv,D,ps", [(14, 2, 64, 16), (28, 4, 128, 48), (3, 3, 128, 32), (8, 8, 64, 64)])
def test_matches_oracle(H, Hkv, D, ps, spans, code):
    rng = np.random.default_rng(len(spans) * 100 + H + D)
    pool = Pool(rng, 60, Hkv, ps, D, code)
    slots, pos = runs_of(rng, spans, 60, ps)
    do(rng, pool, H, Hkv, D, slots, pos, [0] * (D // 2), bias=H != 3)


@pytest.mark.parametrize("T", [1, 3, 4, 5, 15, 16, 17, 63, 400, 3000])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_prompts_and_windows(T, code):
    """Every alignment of runs to the windows that warps look through; 3000
    tokens of 8 heads take the wide windows."""
    rng = np.random.default_rng(T)
    pool = Pool(rng, 250, 8, 16, 64, code)
    slots, pos = runs_of(rng, [(11, T // 2), (0, T - T // 2)], 250, 16)
    do(rng, pool, 16, 8, 64, slots, pos, [0] * 32)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("axes", [2, 3, 4])
def test_position_axes(D, axes, code):
    rng = np.random.default_rng(axes)
    pool = Pool(rng, 20, 2, 32, D, code)
    slots, pos = runs_of(rng, [(0, 70), (18, 1)], 20, 32)
    positions = np.stack([pos] + [rng.integers(0, ROWS, len(pos)) for _ in range(axes - 1)])
    axis = AXES3(D) if axes == 3 else [f % axes for f in range(D // 2)]
    do(rng, pool, 12, 2, D, slots, positions, axis)


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("in_place,strided,layout", [(True, False, "head"), (False, True, "token"), (False, False, "token")])
def test_outputs_and_strides(in_place, strided, layout, keep):
    rng = np.random.default_rng(3)
    pool = Pool(rng, 20, 4, 48, 128, "int8", layout)
    slots, pos = runs_of(rng, [(7, 30), (48, 1), (0, 20)], 20, 48)
    do(rng, pool, 28, 4, 128, slots, pos, [0] * 64, keep=keep, in_place=in_place, strided=strided)


def test_left_out_tokens():
    """Negative slots: none of the token's outputs is written, its neighbours are."""
    rng = np.random.default_rng(4)
    pool = Pool(rng, 20, 2, 16, 64, "e4m3")
    slots, pos = runs_of(rng, [(0, 40), (9, 1)], 20, 16)
    slots[[0, 7, 20, 40]] = -1
    do(rng, pool, 14, 2, 64, slots, pos, [0] * 32)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_token_by_token_growth(code):
    """One call per token, each louder than the last: every call codes the
    block's earlier rows anew."""
    rng = np.random.default_rng(5)
    pool = Pool(rng, 6, 4, 32, 128, code)
    for t in range(35):
        slots = np.array([2 * 32 + t if t < 32 else 5 * 32 + t - 32], np.int64)
        do(rng, pool, 28, 4, 128, slots, np.array([t]), [0] * 64, bias=False, keep=False, scale=1.0 + t % 16)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_zeros_extremes_nan_and_infinity(code):
    D, Hkv = 64, 2
    rng = np.random.default_rng(6)
    pool = Pool(rng, 10, Hkv, 16, D, code)
    T = 4 * 16
    slots = np.arange(T, dtype=np.int64)
    q = half(rng, (T, 4, D))
    k, v = half(rng, (T, Hkv, D)), half(rng, (T, Hkv, D))
    k[:16], v[:16] = 0, 0                                  # a block of zeros: scale 0
    k[16:32], v[16:32] = 6e-8, 65504                       # the smallest and the largest halves
    k[33, 0, 3], v[34, 1, 5] = np.nan, np.inf              # spoil block 2 of one head each
    k[48:], v[48:] = -65504, -6e-8
    cos, sin = tables(D)
    pos = np.zeros((1, T), np.int32)
    O.append(q, k, v, [None] * 3, cos, sin, pos, [0] * 32, slots, pool.k, pool.v, pool.scales, code)
    out = torch.empty((T, 4, D), dtype=torch.float16, device="cuda")
    A.qkv_rope_append_kv8(dev(q), dev(k), dev(v), out, None, None, dev(cos), dev(sin), dev(pos), dev(slots), pool.cache,
                          T, 4, ROWS)
    torch.cuda.synchronize()
    pool.same()
    ko, vo = (torch.empty((T, Hkv, D), dtype=torch.float16, device="cuda") for _ in range(2))
    A.kv8_gather(pool.cache, dev(slots), ko, vo, T)
    ko, vo = ko.cpu().numpy(), vo.cpu().numpy()
    assert (ko[:16] == 0).all() and (vo[:16] == 0).all()
    assert np.isnan(ko[32:48, 0]).all() and np.isfinite(ko[32:48, 1]).all()
    assert np.isnan(vo[32:48, 1]).all() and np.isfinite(vo[32:48, 0]).all()
    assert (ko[48:] == -65504).all() and (vo[16:32] == 65504).all()


def test_indices_out_of_range_are_reported():
    """A slot past the pool is not cached, a position past the table reads as
    position 0; both are recorded, and nothing else is touched."""
    rng = np.random.default_rng(7)
    for slots, pos in (([3, 10**12], [3, 4]), ([3, 64], [3, 4]), ([3, 4], [3, ROWS]), ([3, 4], [-1, 4])):
        pool = Pool(rng, 4, 2, 16, 64, "int8")
        q, k, v = half(rng, (2, 4, 64)), half(rng, (2, 2, 64)), half(rng, (2, 2, 64))
        cos, sin = tables(64)
        slots, pos = np.array(slots, np.int64), np.array([pos], np.int32)
        ok = np.where((pos < 0) | (pos >= ROWS), 0, pos)
        O.append(q, k, v, [None] * 3, cos, sin, ok, [0] * 32, slots, pool.k, pool.v, pool.scales, "int8")
        A.qkv_rope_append_kv8(dev(q), dev(k), dev(v), dev(q), None, None, dev(cos), dev(sin), dev(pos), dev(slots),
                              pool.cache, 2, 4, ROWS)
        torch.cuda.synchronize()
        pool.same()
        assert load().fr_get_device_error(0, None) == FR_ERR_INVALID_ARG
        assert A.device_error() == 4 and A.device_error() == 0


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("Hkv,D,ps,n", [(2, 64, 16, 1), (4, 128, 48, 333), (1, 64, 32, 1000), (8, 128, 64, 17)])
def test_gather(Hkv, D, ps, n, code):
    rng = np.random.default_rng(n)
    pool = Pool(rng, 30, Hkv, ps, D, code, "token" if n == 333 else "head")
    slots = rng.integers(0, 30 * ps, n)
    slots[rng.random(n) < 0.1] = -1
    slots[rng.random(n) < 0.1] = 30 * ps
    real = (slots >= 0) & (slots < 30 * ps)
    at = np.where(real, slots, 0)
    for want_k, want_v in ((True, True), (True, False), (False, True)):
        outs = [torch.full((n, Hkv, D), float("nan"), dtype=torch.float16, device="cuda") if w else None for w in (want_k, want_v)]
        A.kv8_gather(pool.cache, dev(slots.astype(np.int64)), *outs, n)
        for which, (codes, o) in enumerate(zip((pool.k, pool.v), outs)):
            if o is None:
                continue
            r = O.decode(codes, code).astype(np.float32) * np.repeat(pool.scales[..., which], 16, 2)[..., None]
            r = np.where(real[:, None, None], r[at // ps, :, at % ps], 0).astype(np.float16)
            assert np.array_equal(o.cpu().numpy(), r)


def test_offsets_past_32_bits():
    Hkv, D, ps, pages = 4, 128, 128, 80000
    k, v = (torch.zeros((pages, Hkv, ps, D), dtype=torch.int8, device="cuda") for _ in range(2))
    sc = torch.zeros((pages, Hkv, ps // 16, 2), device="cuda")
    cache = A.KV8Cache(k, v, sc)
    rng = np.random.default_rng(8)
    T = 20
    slots = np.arange(T, dtype=np.int64) + 79999 * ps + 96
    q, kk, vv = half(rng, (T, 28, D)), half(rng, (T, Hkv, D)), half(rng, (T, Hkv, D))
    cos, sin = tables(D)
    pos = np.zeros((1, T), np.int32)
    A.qkv_rope_append_kv8(dev(q), dev(kk), dev(vv), dev(q), None, None, dev(cos), dev(sin), dev(pos), dev(slots), cache, T,
                          28, ROWS)
    ko, vo = (torch.empty((T, Hkv, D), dtype=torch.float16, device="cuda") for _ in range(2))
    A.kv8_gather(cache, dev(slots), ko, vo, T)
    torch.cuda.synchronize()
    for got, want in ((ko, kk), (vo, vv)):
        step = np.abs(want).max() / 127
        assert np.abs(got.cpu().numpy().astype(np.float32) - want).max() <= 0.51 * step + 2e-3
    assert int((k != 0).any(3).any(1).sum()) == T


def test_graph_with_fewer_tokens():
    """A captured call replays with other tokens and with padded (-1) slots."""
    rng = np.random.default_rng(9)
    H, Hkv, D, ps, T = 12, 2, 128, 16, 24
    pool = Pool(rng, 12, Hkv, ps, D, "int8")
    cos, sin = tables(D)
    bufs = [torch.zeros((T, n, D), dtype=torch.float16, device="cuda") for n in (H, Hkv, Hkv)]
    out = torch.zeros_like(bufs[0])
    pd, sd = torch.zeros((1, T), dtype=torch.int32, device="cuda"), torch.full((T,), -1, dtype=torch.int64, device="cuda")
    cd, nd = dev(cos), dev(sin)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    call = lambda: A.qkv_rope_append_kv8(*bufs, out, None, None, cd, nd, pd, sd, pool.cache, T, H, ROWS, stream=s)  # noqa: E731
    with torch.cuda.stream(s):
        call()
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call()
    pool.same()
    for n in (24, 5, 1):
        x = [half(rng, tuple(b.shape)) for b in bufs]
        slots = np.full(T, -1, np.int64)
        slots[:n] = np.arange(n) + 3 * ps
        pos = np.arange(T, dtype=np.int32)[None]
        want = O.append(*x, [None] * 3, cos, sin, pos, [0] * 64, slots, pool.k, pool.v, pool.scales, "int8")
        for b, a in zip(bufs, x):
            b.copy_(torch.from_numpy(a))
        pd.copy_(torch.from_numpy(pos))
        sd.copy_(torch.from_numpy(slots))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy()[:n], want[0][:n].astype(np.float16))
        pool.same()


def test_refusals():
    rng = np.random.default_rng(10)
    pool = Pool(rng, 4, 2, 16, 64, "int8")
    q = torch.zeros((2, 4, 64), dtype=torch.float16, device="cuda")
    k = torch.zeros((2, 2, 64), dtype=torch.float16, device="cuda")
    c = torch.ones((8, 32), device="cuda")
    pos, slots = torch.zeros((1, 2), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    with pytest.raises(ForgeRTError, match="invalid argument"):
        A.qkv_rope_append_kv8(q, k, k, q, None, None, c, c, pos, slots, pool.cache, 2, 3, 8)
    with pytest.raises(ForgeRTError, match="invalid argument"):
        A.qkv_rope_append_kv8(q, k, k, q, None, None, c, c, pos, slots, pool.cache, 2, 4, 8, num_axes=2)
    with pytest.raises(ValueError):
        A.qkv_rope_append_kv8(q, k, k, q, None, None, c, c, pos, slots, pool.cache, 2, 4, 8, num_axes=2, freq_axis=bytes(31))
    with pytest.raises(ForgeRTError, match="misaligned"):
        A.qkv_rope_append_kv8(q.data_ptr() + 4, k, k, q, None, None, c, c, pos, slots, pool.cache, 1, 4, 8)
    with pytest.raises(ForgeRTError, match="invalid argument"):
        A.kv8_gather(pool.cache, slots, None, None, 2)
    pool.same()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_tiny_values(code):
    """Rotated values far below what fp16 holds: a scale stops at 2^-100, above
    it the codes are those of the division, remainders included."""
    rng = np.random.default_rng(11)
    for size in (1e-18, 1e-24, 1e-27, 1e-29, 1e-38):
        pool = Pool(rng, 4, 2, 16, 64, code)
        pool.scales[:] = 0
        pool.sd.zero_()
        T = 16
        slots, pos = np.arange(T, dtype=np.int64) + 16, np.arange(T, dtype=np.int32)[None]
        q, k, v = half(rng, (T, 4, 64)), half(rng, (T, 2, 64)), half(rng, (T, 2, 64))
        cos, sin = (x * np.float32(size) for x in tables(64))
        with np.errstate(under="ignore"):
            O.append(q, k, v, [None] * 3, cos, sin, pos, [0] * 32, slots, pool.k, pool.v, pool.scales, code)
        A.qkv_rope_append_kv8(dev(q), dev(k), dev(v), dev(q), None, None, dev(cos), dev(sin), dev(pos), dev(slots),
                              pool.cache, T, 4, ROWS)
        torch.cuda.synchronize()
        pool.same()
        assert pool.scales[1, 0, 0, 0] >= 2.0 ** -100
