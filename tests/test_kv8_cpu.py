"""The 8-bit paged cache without a GPU: the oracle's codes, the entry points'
refusals (all before any CUDA call), and the Python handle's checks."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from forgert_b200 import _lib
from forgert_b200 import attention as A
from oracle import kv8 as O

FAKE = 0x10000          # never dereferenced: validation rejects first


def cache(**over):
    f = dict(k=FAKE, v=FAKE, scales=FAKE, dtype=_lib.FR_KV8_INT8, num_pages=4, page_size=32,
             num_kv_heads=2, head_dim=64, page_stride=4096, head_stride=2048, row_stride=64)
    f.update(over)
    return _lib.Kv8CacheStruct(**f)


def test_e4m3_table_and_rounding_match_torch():
    codes = np.arange(256, dtype=np.uint8)
    t = torch.from_numpy(codes).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(np.isnan(t), np.isnan(O.E4M3)) and np.array_equal(t[~np.isnan(t)], O.E4M3[~np.isnan(t)])
    rng = np.random.default_rng(0)
    finite = np.sort(O.E4M3[:127])
    x = np.concatenate([rng.standard_normal(4000) * 2.0 ** rng.integers(-12, 9, 4000), finite,
                        (finite[1:] + finite[:-1]) / 2, [448.0, -448.0, 1e-9, 0.0]]).astype(np.float32)
    x = np.clip(x, -448, 448)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(O.encode(x, "e4m3"), want)
    assert O.encode(np.float32([1e6, -1e6]), "e4m3").tolist() == [126, 254]


def test_int8_rounding():
    x = np.float32([0.5, 1.5, -0.5, -2.5, 126.6, 400, -400, np.nan])
    assert O.encode(x, "int8").view(np.int8).tolist() == [0, 2, 0, -2, 127, 127, -127, 0]


def test_put_keeps_values_within_half_a_step():
    """One row after the other: every held value stays within its scale's
    rounding, which each growth of the scale adds to once."""
    rng = np.random.default_rng(1)
    rows = (rng.standard_normal((16, 1, 64)) * (1 + np.arange(16))[:, None, None]).astype(np.float32)
    for code in O.KMAX:
        codes = np.zeros((1, 1, 16, 64), np.uint8)
        scales = np.zeros((1, 1, 1, 2), np.float32)
        for t in range(16):
            O.put(rows[t:t + 1], codes, scales, 0, [t], code)
        got = O.values(codes, scales, 0, code)[0, 0]
        step = scales[0, 0, 0, 0] * (1.0 if code == "int8" else 32.0)       # largest gap between codes
        assert np.abs(got - rows[:, 0]).max() <= 16 * step / 2
        assert scales[0, 0, 0, 0] == np.float32(np.abs(rows).max() / np.float32(O.KMAX[code]))


def test_step_oracle_conserves_pages():
    rng = np.random.default_rng(2)
    B, ps, P, width = 7, 16, 40, 8
    lens, table, stack, count = [0] * B, [[-1] * width for _ in range(B)], list(range(P)), P
    for _ in range(200):
        new = [int(x) for x in rng.integers(-1, 20, B)]
        st, lens, table, stack, count, off, pos, slots = O.step(lens, new, table, stack, count, ps, 400)
        held = [table[b][j] for b in range(B) for j in range(-(-lens[b] // ps))]
        assert sorted(held + stack[:count]) == list(range(P))
        if st == 0:
            live = [s for s in slots if s >= 0]
            assert len(set(live)) == len(live) == off[-1]


def test_step_refusals(lib):
    def step(*arrays, B=4, ps=16, P=8, mb=4, mt=64):
        a = list(arrays) + [FAKE + 64 * i for i in range(len(arrays), 11)]
        return lib.fr_paged_step(*a, B, ps, P, mb, mt, None)

    assert step(None) == _lib.FR_ERR_INVALID_ARG
    for i in range(11):
        a = [FAKE + 64 * j for j in range(11)]
        a[i] = None
        assert step(*a) == _lib.FR_ERR_INVALID_ARG
        a[i] = FAKE + 64 * i + 2
        assert step(*a) == _lib.FR_ERR_MISALIGNED
    for over in (dict(B=0), dict(B=8193), dict(ps=0), dict(P=0), dict(mb=0), dict(mt=0), dict(mt=1 << 30),
                 dict(P=1 << 30), dict(mb=1 << 20, ps=1 << 10)):
        assert step(**over) == _lib.FR_ERR_INVALID_ARG, over
    shared = [FAKE + 64 * j for j in range(11)]
    shared[5] = shared[1]                       # kv_lens_out over new_lens
    assert step(*shared) == _lib.FR_ERR_INVALID_ARG


def append(lib, c, q=FAKE, k=FAKE, v=FAKE, qo=FAKE, ko=None, vo=None, strides=None, biases=(None,) * 3,
           cos=FAKE, sin=FAKE, rows=128, pos=FAKE, axes=1, axis=None, slots=FAKE, T=4, H=8):
    st = None if strides is None else (ctypes.c_longlong * 6)(*strides)
    return lib.fr_qkv_rope_append_kv8(q, k, v, qo, ko, vo, st, *biases, cos, sin, rows, pos, axes, axis, slots,
                                      None if c is None else ctypes.byref(c), T, H, None)


BAD_CACHES = [
    (dict(k=None), _lib.FR_ERR_INVALID_ARG), (dict(v=None), _lib.FR_ERR_INVALID_ARG),
    (dict(scales=None), _lib.FR_ERR_INVALID_ARG), (dict(dtype=2), _lib.FR_ERR_INVALID_ARG),
    (dict(dtype=-1), _lib.FR_ERR_INVALID_ARG), (dict(num_pages=0), _lib.FR_ERR_INVALID_ARG),
    (dict(page_size=24), _lib.FR_ERR_INVALID_ARG), (dict(page_size=0), _lib.FR_ERR_INVALID_ARG),
    (dict(num_kv_heads=0), _lib.FR_ERR_INVALID_ARG), (dict(head_dim=96), _lib.FR_ERR_UNSUPPORTED),
    (dict(row_stride=48), _lib.FR_ERR_INVALID_ARG), (dict(head_stride=0), _lib.FR_ERR_INVALID_ARG),
    (dict(page_stride=-4096), _lib.FR_ERR_INVALID_ARG), (dict(page_stride=1 << 40), _lib.FR_ERR_INVALID_ARG),
    (dict(row_stride=72), _lib.FR_ERR_MISALIGNED), (dict(k=FAKE + 8), _lib.FR_ERR_MISALIGNED),
    (dict(scales=FAKE + 4), _lib.FR_ERR_MISALIGNED),
]


@pytest.mark.parametrize("over,want", BAD_CACHES)
def test_every_entry_refuses_a_bad_cache(lib, over, want):
    c = cache(**over)
    assert append(lib, c) == want
    assert lib.fr_kv8_gather(ctypes.byref(c), FAKE, FAKE, FAKE, 4, None) == want
    assert lib.fr_decode_attn_paged_kv8(FAKE, 0, ctypes.byref(c), FAKE, FAKE, FAKE, 2, 8, 4, 64, None) == want


def test_append_refusals(lib):
    c = cache()
    inv, mis = _lib.FR_ERR_INVALID_ARG, _lib.FR_ERR_MISALIGNED
    assert append(lib, None) == inv
    for over in (dict(q=None), dict(k=None), dict(v=None), dict(qo=None), dict(cos=None), dict(sin=None),
                 dict(pos=None), dict(slots=None), dict(rows=0), dict(T=-1), dict(H=0), dict(H=7), dict(axes=0),
                 dict(axes=5, axis=bytes(32)), dict(axes=3), dict(axes=2, axis=bytes([2] * 32)),
                 dict(strides=[511, 128, 128, 512, 128, 128])):
        assert append(lib, c, **over) == inv, over
    for over in (dict(q=FAKE + 4), dict(ko=FAKE + 4), dict(vo=FAKE + 2), dict(cos=FAKE + 8), dict(pos=FAKE + 2),
                 dict(slots=FAKE + 4), dict(biases=(FAKE + 2, None, None)),
                 dict(strides=[514, 128, 128, 512, 128, 128])):
        assert append(lib, c, **over) == mis, over
    assert append(lib, c, T=0) == _lib.FR_OK


def test_gather_and_attention_refusals(lib):
    r = ctypes.byref(cache())
    inv, mis = _lib.FR_ERR_INVALID_ARG, _lib.FR_ERR_MISALIGNED
    g = lambda *a: lib.fr_kv8_gather(*a, None)  # noqa: E731
    assert g(None, FAKE, FAKE, FAKE, 4) == inv
    assert g(r, None, FAKE, FAKE, 4) == inv
    assert g(r, FAKE, None, None, 4) == inv
    assert g(r, FAKE, FAKE, FAKE, -1) == inv
    assert g(r, FAKE + 4, FAKE, FAKE, 4) == mis
    assert g(r, FAKE, FAKE + 8, None, 4) == mis
    assert g(r, FAKE, FAKE, None, 0) == _lib.FR_OK

    def attn(q=FAKE, qs=0, c=r, t=FAKE, n=FAKE, o=FAKE, B=2, H=8, mb=4, mk=64):
        return lib.fr_decode_attn_paged_kv8(q, qs, c, t, n, o, B, H, mb, mk, None)

    for over in (dict(q=None), dict(c=None), dict(t=None), dict(n=None), dict(o=None), dict(B=0), dict(H=0),
                 dict(H=7), dict(mb=0), dict(mk=-1), dict(mk=129), dict(qs=504), dict(qs=-512),
                 dict(mb=1 << 26, mk=1 << 30)):
        assert attn(**over) == inv, over
    for over in (dict(q=FAKE + 8), dict(o=FAKE + 8), dict(qs=516), dict(t=FAKE + 2), dict(n=FAKE + 2)):
        assert attn(**over) == mis, over


def test_handle_checks():
    k = torch.zeros((3, 2, 32, 64), dtype=torch.int8)
    s = torch.zeros((3, 2, 2, 2))
    bad = [(k.half(), k.half(), s), (k, k.view(torch.float8_e4m3fn), s), (k, k[:2], s), (k, k, s[..., :1]),
           (k, k, s.double()), (k, k, s.transpose(1, 2)), (k, k.transpose(1, 2).contiguous().transpose(1, 2), s),
           (k.transpose(2, 3), k.transpose(2, 3), s), (k[0], k[0], s)]
    for args in bad:
        with pytest.raises(ValueError):
            A.KV8Cache(*args)
    with pytest.raises(ValueError, match="CUDA"):
        A.KV8Cache(k, k, s)


def test_append_in_place_keeps_the_layout(lib):
    """An output over its input with another distance between tokens would be
    written where other tokens are still read."""
    c = cache()
    inv = _lib.FR_ERR_INVALID_ARG
    assert append(lib, c, strides=[512, 128, 128, 516, 128, 128], qo=FAKE) == inv
    assert append(lib, c, strides=[512, 128, 128, 512, 132, 128], ko=FAKE) == inv
    assert append(lib, c, strides=[512, 128, 128, 512, 128, 136], vo=FAKE) == inv
    assert append(lib, c, strides=[512, 128, 128, 516, 132, 136], qo=FAKE + 64, ko=FAKE + 64, vo=FAKE + 64, T=0) == _lib.FR_OK
