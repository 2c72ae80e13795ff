"""GPU tests of the prologues of the 16-bit pages (fr_qkv_rope_append_paged) and
of the 4-bit cache (fr_qkv_rope_append_kv4), and of its read-back (fr_kv4_gather).

The oracle follows the operators' 32-bit operations one by one, so pages, codes
and scales are compared exactly, and so are the fp16 outputs; beside that the
outputs are held to the 64-bit rotation within half an fp16 step plus the fp32
roundings of a three-operation sum:
  |x - r| <= 2^-11 |r| + 2^-22 (|a| + |b|) + 2^-25 (fp16's smallest step).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from forgert_b200 import attention as A
from forgert_b200._lib import FR_ERR_INVALID_ARG, ForgeRTError, load
from oracle import kv4 as O
from oracle import kv8

pytestmark = pytest.mark.gpu
ROWS = 5000
KINDS = ["pages", "int4"]


def tables(D):
    a = np.arange(ROWS)[:, None] * 1e6 ** (-2.0 * np.arange(D // 2) / D)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def half(rng, shape, scale=1.0):
    return (rng.standard_normal(shape) * scale).astype(np.float16)


def dev(x):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()


class Pages:
    """16-bit pages on the device and their copy for the oracle."""

    def __init__(self, rng, pages, Hkv, ps, D, layout="head"):
        self.ps, self.n, self.shape = ps, pages, (Hkv, D)
        self.k, self.v = (half(rng, (pages, ps, Hkv, D)) for _ in range(2))
        self.kd, self.vd = dev(self.k), dev(self.v)

    def put(self, rows, slots):
        with np.errstate(over="ignore"):
            for pool, x in ((self.k, rows[1]), (self.v, rows[2])):
                flat = pool.reshape(-1, *self.shape)
                for t, s in enumerate(slots):
                    if 0 <= s < len(flat):
                        flat[s] = x[t].astype(np.float16)

    def call(self, *args, T, H, rows, biases, **kw):
        A.qkv_rope_append_paged(*args, self.kd, self.vd, self.ps, self.n, T, H, *self.shape, rows, *biases, **kw)

    def same(self):
        for got, want in ((self.kd, self.k), (self.vd, self.v)):
            assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)


class Codes:
    """A 4-bit cache on the device and its copy for the oracle."""

    def __init__(self, rng, pages, Hkv, ps, D, layout="head"):
        self.ps, self.n = ps, pages
        self.k, self.v = (rng.integers(0, 256, (pages, Hkv, ps, D // 2), dtype=np.uint8) for _ in range(2))
        self.scales = half(rng, (pages, Hkv, ps, 2, D // 64, 2))

        def lay(x):
            x = dev(x)
            return x.transpose(1, 2).contiguous().transpose(1, 2) if layout == "token" else x
        self.kd, self.vd, self.sd = lay(self.k), lay(self.v), dev(self.scales)
        self.cache = A.KV4Cache(self.kd, self.vd, self.sd)

    def put(self, rows, slots):
        O.put(rows[1], self.k, self.scales, 0, slots)
        O.put(rows[2], self.v, self.scales, 1, slots)

    def call(self, *args, T, H, rows, biases, **kw):
        A.qkv_rope_append_kv4(*args, self.cache, T, H, rows, *biases, **kw)

    def same(self):
        assert np.array_equal(self.sd.cpu().numpy(), self.scales, equal_nan=True)
        for got, want in ((self.kd, self.k), (self.vd, self.v)):
            got = got.cpu().numpy()
            bad = np.argwhere(got != want)
            assert not len(bad), (len(bad), bad[:4].tolist())


def pool_of(kind, *args, **kw):
    return (Pages if kind == "pages" else Codes)(*args, **kw)


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


def do(rng, pool, H, Hkv, D, slots, positions, axis=None, bias=True, keep=True, in_place=False, strided=False,
       qkv=None, stream=None, error=0):
    T = len(slots)
    q, k, v = qkv or (half(rng, (T, H, D)), half(rng, (T, Hkv, D)), half(rng, (T, Hkv, D)))
    biases = [half(rng, (n, D)) if bias else None for n in (H, Hkv, Hkv)]
    cos, sin = tables(D)
    positions = np.atleast_2d(positions)
    axis = axis or [0] * (D // 2)
    want = O.turned(q, k, v, biases, cos, sin, positions, axis)
    pool.put(want, slots)
    strides = None
    if strided:                                          # q, k, v of a token in one row, outputs apart
        row = torch.full((T, (H + 2 * Hkv) * D + 24), 9.0, dtype=torch.float16, device="cuda")
        row[:, :(H + 2 * Hkv) * D] = torch.cat([dev(x).flatten(1) for x in (q, k, v)], 1)
        w = row.stride(0)
        at = [row.data_ptr(), row.data_ptr() + 2 * H * D, row.data_ptr() + 2 * (H + Hkv) * D]
        strides = [w, w, w, H * D + 8, Hkv * D, Hkv * D + 16]
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
    args = [dev(cos), dev(sin), dev(positions.astype(np.int32)), dev(slots)]
    bd = [dev(b) for b in biases]
    torch.cuda.synchronize()
    pool.call(*at, *outs, *args, T=T, H=H, rows=ROWS, biases=bd, num_axes=len(positions),
              freq_axis=bytes(axis) if len(positions) > 1 else None, token_strides=strides, stream=stream)
    torch.cuda.synchronize()
    assert A.device_error() == error
    real = slots >= 0
    for i, (got, r) in enumerate(zip(views if keep else views[:1], want)):
        g = got.cpu().numpy()
        with np.errstate(over="ignore"):
            assert np.array_equal(g[real], r[real].astype(np.float16), equal_nan=True), i
        if not in_place:
            assert np.isnan(g[~real]).all()
        x, b = (q, k, v)[i], biases[i]
        if i < 2 and qkv is None:
            r64 = kv8.rotate64(x, b, positions, axis, cos, sin)[real]
            e = np.abs(x.astype(np.float64)) + (0 if b is None else np.abs(b.astype(np.float64)))
            e = (e + np.roll(e, D // 2, -1))[real]
            assert (np.abs(g[real] - r64) <= 2.0 ** -11 * np.abs(r64) + 2.0 ** -22 * e + 2.0 ** -25).all()
    pool.same()
    return want


AXES3 = lambda D: [0] * (D // 8) + [1] * (D // 2 - 2 * (D // 8)) + [2] * (D // 8)  # noqa: E731
SPANS = [
    [(0, 1)], [(5, 1)], [(15, 1)], [(16, 1)], [(0, 16)], [(3, 13)], [(0, 100)], [(31, 2)],
    [(i * 7 % 33, 1) for i in range(40)],
    [(0, 37), (12, 1), (100, 3), (15, 50), (1, 15), (16, 16), (47, 1)],
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("spans", SPANS)
@pytest.mark.parametrize("H,Hkv,D,ps", [(14, 2, 64, 16), (28, 4, 128, 48), (3, 3, 128, 32), (8, 8, 64, 64), (16, 1, 128, 16),
                                        (5, 1, 64, 16)])
def test_matches_oracle(H, Hkv, D, ps, spans, kind):
    rng = np.random.default_rng(len(spans) * 100 + H + D)
    pool = pool_of(kind, rng, 60, Hkv, ps, D)
    slots, pos = runs_of(rng, spans, 60, ps)
    do(rng, pool, H, Hkv, D, slots, pos, bias=H != 3)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 3, 17, 63, 400, 3001])
def test_prompts(T, kind):
    rng = np.random.default_rng(T)
    pool = pool_of(kind, rng, 250, 8, 16, 64)
    slots, pos = runs_of(rng, [(11, T // 2), (0, T - T // 2)], 250, 16)
    do(rng, pool, 16, 8, 64, slots, pos)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("axes", [2, 3, 4])
def test_position_axes(D, axes, kind):
    """Axes by groups of eight frequencies (three of them at D = 128) and one by one."""
    rng = np.random.default_rng(axes)
    pool = pool_of(kind, rng, 20, 2, 32, D)
    slots, pos = runs_of(rng, [(0, 70), (18, 1)], 20, 32)
    positions = np.stack([pos] + [rng.integers(0, ROWS, len(pos)) for _ in range(axes - 1)])
    axis = AXES3(D) if axes == 3 else [f % axes for f in range(D // 2)]
    do(rng, pool, 12, 2, D, slots, positions, axis)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("in_place,strided,layout", [(True, False, "head"), (False, True, "token"), (False, False, "token")])
def test_outputs_and_strides(in_place, strided, layout, keep, kind):
    rng = np.random.default_rng(3)
    pool = pool_of(kind, rng, 20, 4, 48, 128, layout=layout)
    slots, pos = runs_of(rng, [(7, 30), (48, 1), (0, 20)], 20, 48)
    do(rng, pool, 28, 4, 128, slots, pos, keep=keep, in_place=in_place, strided=strided)


@pytest.mark.parametrize("kind", KINDS)
def test_left_out_tokens(kind):
    """Negative slots: none of the token's outputs is written, its neighbours' are."""
    rng = np.random.default_rng(4)
    pool = pool_of(kind, rng, 20, 2, 16, 64)
    slots, pos = runs_of(rng, [(0, 40), (9, 1)], 20, 16)
    slots[[0, 7, 20, 40]] = [-1, -2 ** 62, -1, -5]
    do(rng, pool, 14, 2, 64, slots, pos)


@pytest.mark.parametrize("kind", KINDS)
def test_slots_and_positions_out_of_range(kind):
    """A slot past the pool: recorded and not cached, the token's outputs are
    written.  A position outside the table: recorded, position 0's row is taken."""
    rng = np.random.default_rng(5)
    pool = pool_of(kind, rng, 4, 2, 16, 128)
    slots = np.array([0, 64, 5, 2 ** 62, -1, 63], np.int64)
    do(rng, pool, 14, 2, 128, slots, np.arange(6), error=4)
    q, k, v = half(rng, (1, 14, 128)), half(rng, (1, 2, 128)), half(rng, (1, 2, 128))
    cos, sin = tables(128)
    want = O.turned(q, k, v, [None] * 3, cos, sin, np.zeros((1, 1), int), [0] * 64)
    pool.put(want, [9])
    out = torch.empty((1, 14, 128), dtype=torch.float16, device="cuda")
    for bad in (ROWS, -1):
        pool.call(dev(q), dev(k), dev(v), out, None, None, dev(cos), dev(sin), dev(np.full((1, 1), bad, np.int32)),
                  dev(np.array([9])), T=1, H=14, rows=ROWS, biases=[None] * 3)
        assert A.device_error() == 4 and A.device_error() == 0
        assert np.array_equal(out.cpu().numpy(), want[0].astype(np.float16))
        pool.same()


@pytest.mark.parametrize("kind", KINDS)
def test_zeros_extremes_nan_and_infinity(kind):
    D, Hkv, T = 128, 2, 24
    rng = np.random.default_rng(6)
    pool = pool_of(kind, rng, 10, Hkv, 16, D)
    q, k, v = half(rng, (T, 4, D)), half(rng, (T, Hkv, D)), half(rng, (T, Hkv, D))
    k[:4], v[:4] = 0, 0                                   # scale 0, bias 0
    v[4], k[5] = 3.25, -7                                 # scale 0 and a bias
    v[6], k[7] = 6e-8, 65504                              # the smallest and the largest halves
    v[8, :, ::2], v[8, :, 1::2] = 65504, -65504           # the widest group
    k[9, 0, 3], v[10, 1, 70], v[11, 0, 5] = np.nan, np.inf, -np.inf
    v[12] = 2048
    v[12, :, 7] = 2050                                    # neighbours of fp16
    v[13] = np.float16(-0.0)
    do(rng, pool, 4, Hkv, D, np.arange(T, dtype=np.int64) + 3, np.arange(T) * 10, bias=False, qkv=(q, k, v))
    if kind == "int4":
        got = O.values(pool.v, pool.scales, 1).transpose(0, 2, 1, 3).reshape(-1, Hkv, D)[3:3 + T]
        assert (got[4] == 3.25).all() and (got[:4] == 0).all() and (got[13] == 0).all()
        assert np.isnan(got[10, 1, 64:]).all() and np.isfinite(got[10, 1, :64]).all() and np.isfinite(got[10, 0]).all()
        assert np.isnan(got[11, 0, :64]).all()


def test_bounds_past_fp16():
    """A bias takes values past fp16's range: the group reads back as NaN where
    its minimum lies below -65504, and holds what lies above 65504."""
    D = 64
    rng = np.random.default_rng(7)
    for sign in (1, -1):
        pool = Codes(rng, 2, 1, 16, D)
        v = np.full((1, 1, D), sign * 60000, np.float16)
        b = np.full((1, D), sign * 60000, np.float16)
        z = np.zeros((1, 1, D), np.float16)
        cos, sin = tables(D)
        A.qkv_rope_append_kv4(dev(z), dev(z), dev(v), dev(z), None, None, dev(cos), dev(sin),
                              dev(np.zeros((1, 1), np.int32)), dev(np.array([3])), pool.cache, 1, 1, ROWS, v_bias=dev(b))
        torch.cuda.synchronize()
        rows = O.turned(z, z, v, [None, None, b], cos, sin, np.zeros((1, 1), int), [0] * 32)
        pool.put(rows, [3])
        pool.same()
        got = O.values(pool.v, pool.scales, 1)[0, 0, 3]
        assert np.isnan(got).all() if sign < 0 else (np.abs(got - 119968) <= pool.scales[0, 0, 3, 1, 0, 0] / 2 + 1).all()


@pytest.mark.parametrize("kind", KINDS)
def test_any_order_of_tokens(kind):
    """Rows stand by themselves: a step's tokens in any order, one by one or
    together, give the same pages."""
    rng = np.random.default_rng(8)
    H, Hkv, D, T = 6, 2, 128, 50
    slots = rng.permutation(64)[:T].astype(np.int64)
    pos = rng.integers(0, ROWS, T).astype(np.int32)
    q, k, v = half(rng, (T, H, D)), half(rng, (T, Hkv, D)), half(rng, (T, Hkv, D))
    a = pool_of(kind, np.random.default_rng(1), 4, Hkv, 16, D)
    b = pool_of(kind, np.random.default_rng(1), 4, Hkv, 16, D)
    do(rng, a, H, Hkv, D, slots, pos, bias=False, qkv=(q, k, v))
    for t in rng.permutation(T):
        do(rng, b, H, Hkv, D, slots[t:t + 1], pos[t:t + 1], bias=False, qkv=tuple(x[t:t + 1] for x in (q, k, v)))
    assert torch.equal(a.kd.view(torch.uint8), b.kd.view(torch.uint8))
    assert torch.equal(a.vd.view(torch.uint8), b.vd.view(torch.uint8))


@pytest.mark.parametrize("kind", KINDS)
def test_side_stream_and_graph(kind):
    """On a stream of its own, captured, and replayed on other tokens and slots."""
    rng = np.random.default_rng(9)
    H, Hkv, D, T = 14, 2, 64, 5
    pool = pool_of(kind, rng, 8, Hkv, 16, D)
    s = torch.cuda.Stream()
    slots, pos = runs_of(rng, [(0, 5)], 8, 16)
    do(rng, pool, H, Hkv, D, slots, pos, bias=False, stream=s)
    cos, sin = (dev(x) for x in tables(D))
    q, k, v = (torch.zeros((T, n, D), dtype=torch.float16, device="cuda") for n in (H, Hkv, Hkv))
    sd, pd = torch.zeros(T, dtype=torch.int64, device="cuda"), torch.zeros((1, T), dtype=torch.int32, device="cuda")
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        pool.call(q, k, v, out, None, None, cos, sin, pd, sd, T=T, H=H, rows=ROWS, biases=[None] * 3, stream=s)
    for slots in ([9, 10, 11, 12, 13], [80, -1, 33, 127, 2]):
        new = [half(rng, (T, n, D)) for n in (H, Hkv, Hkv)]
        pos = rng.integers(0, ROWS, (1, T))
        for x, y in zip((q, k, v), new):
            x.copy_(dev(y))
        sd.copy_(torch.tensor(slots))
        pd.copy_(torch.from_numpy(pos))
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = O.turned(*new, [None] * 3, *tables(D), pos, [0] * 32)
        pool.put(want, slots)
        pool.same()
        real = np.array(slots) >= 0
        assert np.array_equal(out.cpu().numpy()[real], want[0][real].astype(np.float16))
        assert np.isnan(out.cpu().numpy()[~real]).all()
    assert A.device_error() == 0


@pytest.mark.parametrize("D,Hkv,ps", [(64, 2, 16), (128, 4, 48)])
@pytest.mark.parametrize("layout", ["head", "token"])
def test_read_back(D, Hkv, ps, layout):
    """Exactly code * scale + bias rounded to fp16 once; slots outside the pool give zeros, the
    same slot twice the same row twice."""
    rng = np.random.default_rng(10)
    pool = Codes(rng, 9, Hkv, ps, D, layout)
    slots = np.concatenate([rng.permutation(9 * ps)[:77], [3, 3, -1, 9 * ps, 2 ** 62, 9 * ps - 1, 0]]).astype(np.int64)
    outs = [torch.full((len(slots), Hkv, D), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2)]
    A.kv4_gather(pool.cache, dev(slots), *outs, len(slots))
    torch.cuda.synchronize()
    real = (slots >= 0) & (slots < 9 * ps)
    for which, (codes, got) in enumerate(zip((pool.k, pool.v), outs)):
        x = O.values(codes, pool.scales, which).transpose(0, 2, 1, 3).reshape(-1, Hkv, D)
        want = np.where(real[:, None, None], x[np.where(real, slots, 0)].astype(np.float16), 0)
        assert np.array_equal(got.cpu().numpy(), want)
        one = [None, None]
        one[which] = torch.full_like(got, float("nan"))
        A.kv4_gather(pool.cache, dev(slots), *one, len(slots))
        assert torch.equal(one[which], got)
    outs[0].fill_(7.0)
    A.kv4_gather(pool.cache, dev(slots), outs[0], None, 0)
    assert (outs[0] == 7).all()


def test_offsets_past_32_bits():
    """16-bit pages of 6 GB and a 4-bit pool of 5 GB of codes: slots near their ends."""
    rng = np.random.default_rng(11)
    Hkv, D, ps = 8, 128, 128
    T, H = 3, 8
    q, k, v = half(rng, (T, H, D)), half(rng, (T, Hkv, D)), half(rng, (T, Hkv, D))
    cos, sin = tables(D)
    want = O.turned(q, k, v, [None] * 3, cos, sin, np.arange(T)[None], [0] * 64)
    args = [dev(x) for x in (q, k, v)] + [dev(q), None, None, dev(cos), dev(sin), dev(np.arange(T, dtype=np.int32)[None])]
    n = 23000
    slots = np.array([n * ps - 1, 5, n * ps - 700000], np.int64)
    kp, vp = (torch.zeros((n, ps, Hkv, D), dtype=torch.float16, device="cuda") for _ in range(2))
    A.qkv_rope_append_paged(*args, dev(slots), kp, vp, ps, n, T, H, Hkv, D, ROWS)
    at = dev(slots)
    for pool, r in ((kp, want[1]), (vp, want[2])):
        assert np.array_equal(pool.view(-1, Hkv, D)[at].cpu().numpy(), r.astype(np.float16))
        assert int((pool != 0).sum()) == int((r.astype(np.float16) != 0).sum())
    del kp, vp
    n = 76000
    slots = np.array([n * ps - 1, 5, n * ps - 7000000], np.int64)
    kc, vc = (torch.zeros((n, Hkv, ps, D // 2), dtype=torch.uint8, device="cuda") for _ in range(2))
    sc = torch.zeros((n, Hkv, ps, 2, 2, 2), dtype=torch.float16, device="cuda")
    cache = A.KV4Cache(kc, vc, sc)
    A.qkv_rope_append_kv4(*args, dev(slots), cache, T, H, ROWS)
    outs = [torch.zeros((T, Hkv, D), dtype=torch.float16, device="cuda") for _ in range(2)]
    A.kv4_gather(cache, dev(slots), *outs, T)
    for r, got in zip(want[1:], outs):
        raw, pairs = O.encode(r)
        s = np.repeat(pairs.astype(np.float64), 64, -2)
        x = O.unpack(raw) * s[..., 0] + s[..., 1]
        assert np.array_equal(got.cpu().numpy(), x.astype(np.float16))
    assert A.device_error() == 0


def test_refusals():
    rng = np.random.default_rng(12)
    pool = Codes(rng, 4, 2, 16, 64)
    x = torch.zeros((2, 8, 64), dtype=torch.float16, device="cuda")
    i = torch.zeros(2, dtype=torch.int64, device="cuda")
    c = torch.zeros((8, 32), device="cuda")
    with pytest.raises(ForgeRTError, match="invalid argument"):
        A.qkv_rope_append_kv4(x, x, x, x, None, None, c, c, i, i, pool.cache, 2, 7, 8)
    with pytest.raises(ForgeRTError, match="invalid argument"):
        A.qkv_rope_append_paged(x, x, x, x, None, None, c, c, i, i, x, x, 24, 1, 2, 8, 2, 64, 8)
    with pytest.raises(ForgeRTError, match="misaligned"):
        A.qkv_rope_append_kv4(x.data_ptr() + 8, x, x, x, None, None, c, c, i, i, pool.cache, 2, 8, 8)
    with pytest.raises(ForgeRTError, match="misaligned"):
        A.kv4_gather(pool.cache, i, x.data_ptr() + 8, None, 2)
    with pytest.raises(ValueError, match="freq_axis"):
        A.qkv_rope_append_kv4(x, x, x, x, None, None, c, c, i, i, pool.cache, 2, 8, 8, freq_axis=bytes(3), num_axes=2)
    with pytest.raises(ValueError):
        A.kv4_gather(pool.cache, i.cpu(), x, None, 2)
    assert load().fr_kv4_gather(None, 0, 0, 0, 1, None) == FR_ERR_INVALID_ARG
