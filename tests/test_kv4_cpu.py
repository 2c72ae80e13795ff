"""The 4-bit paged cache and the 16-bit pages' append without a GPU: the
oracle's codes, the entry points' refusals (all before any CUDA call), and the
Python handle's checks."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from forgert_b200 import _lib
from forgert_b200 import attention as A
from oracle import kv4 as O

FAKE = 0x10000          # never dereferenced: validation rejects first
INV, MIS, UNS = _lib.FR_ERR_INVALID_ARG, _lib.FR_ERR_MISALIGNED, _lib.FR_ERR_UNSUPPORTED


def cache(**over):
    f = dict(k=FAKE, v=FAKE, scales=FAKE, num_pages=4, page_size=32, num_kv_heads=2, head_dim=64,
             page_stride=2048, head_stride=1024, row_stride=32)
    f.update(over)
    return _lib.Kv4CacheStruct(**f)


def test_half_below_and_above():
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(3000) * 2.0 ** rng.integers(-30, 15, 3000),
                        [0, 65504, -65504, 65519, 70000, 1e-9, -1e-9, 2.0 ** -24, 1 + 2.0 ** -11]]).astype(np.float32)
    below = O.half_below(x).astype(np.float64)
    after = np.nextafter(O.half_below(x), np.float16(np.inf)).astype(np.float64)
    assert (below <= x).all() and (after > x).all()
    fits = x <= 65504
    assert (O.half_above(x)[fits].astype(np.float64) >= x[fits]).all()
    assert np.isneginf(O.half_below(np.float32(-65520))) and np.isnan(O.half_below(np.float32(np.nan)))


def test_every_value_is_within_half_a_scale():
    """Quotients lie in 0 .. 15 whatever the group's place and width."""
    rng = np.random.default_rng(1)
    for spread in (1e-6, 1e-3, 1.0, 300.0):
        for centre in (0.0, 1.0, -3.3, 1000.0):
            x = (centre + spread * rng.standard_normal((200, 128))).astype(np.float32)
            raw, pairs = O.encode(x)
            s = np.repeat(pairs.astype(np.float64), 64, 1)
            err = np.abs(O.unpack(raw) * s[..., 0] + s[..., 1] - x)
            # beside half a scale: the roundings of x - bias and of the quotient to fp32
            assert (err <= s[..., 0] / 2 * (1 + 2.0 ** -20) + 2.0 ** -24 * np.abs(x - s[..., 1])).all()


def test_encode_extremes():
    x = np.zeros((6, 64), np.float32)
    x[1] = 3.0
    x[2, 5] = np.nan
    x[3, 0] = np.inf
    x[4, 9] = -70000.0
    x[5] = np.linspace(0, 1, 64)
    raw, pairs = O.encode(x)
    assert (raw[:5] == 0).all() and (pairs[0] == 0).all() and pairs[1].tolist() == [[0.0, 3.0]]
    assert np.isnan(pairs[2:5]).all()
    assert raw[5, 0] & 15 == 0 and raw[5, -1] >> 4 == 15


def append4(lib, c, q=FAKE, k=FAKE, v=FAKE, qo=FAKE, ko=None, vo=None, strides=None, biases=(None,) * 3,
            cos=FAKE, sin=FAKE, rows=128, pos=FAKE, axes=1, axis=None, slots=FAKE, T=4, H=8):
    st = None if strides is None else (ctypes.c_longlong * 6)(*strides)
    return lib.fr_qkv_rope_append_kv4(q, k, v, qo, ko, vo, st, *biases, cos, sin, rows, pos, axes, axis, slots,
                                      None if c is None else ctypes.byref(c), T, H, None)


def append16(lib, kp=FAKE, vp=FAKE, ps=32, np_=4, q=FAKE, k=FAKE, v=FAKE, qo=FAKE, ko=None, vo=None, strides=None,
             biases=(None,) * 3, cos=FAKE, sin=FAKE, rows=128, pos=FAKE, axes=1, axis=None, slots=FAKE, T=4, H=8,
             Hkv=2, D=64):
    st = None if strides is None else (ctypes.c_longlong * 6)(*strides)
    return lib.fr_qkv_rope_append_paged(q, k, v, qo, ko, vo, st, *biases, cos, sin, rows, pos, axes, axis, slots,
                                        kp, vp, ps, np_, T, H, Hkv, D, None)


BAD_CACHES = [
    (dict(k=None), INV), (dict(v=None), INV), (dict(scales=None), INV), (dict(num_pages=0), INV),
    (dict(page_size=24), INV), (dict(page_size=0), INV), (dict(num_kv_heads=0), INV), (dict(head_dim=96), UNS),
    (dict(row_stride=16), INV), (dict(head_stride=0), INV), (dict(page_stride=-2048), INV),
    (dict(page_stride=1 << 40), INV), (dict(row_stride=40), MIS), (dict(k=FAKE + 8), MIS), (dict(scales=FAKE + 8), MIS),
]


@pytest.mark.parametrize("over,want", BAD_CACHES)
def test_every_entry_refuses_a_bad_cache(lib, over, want):
    c = cache(**over)
    assert append4(lib, c) == want
    assert lib.fr_kv4_gather(ctypes.byref(c), FAKE, FAKE, FAKE, 4, None) == want
    assert lib.fr_decode_attn_paged_kv4(FAKE, 0, ctypes.byref(c), FAKE, FAKE, FAKE, 2, 8, 4, 64, None) == want


def test_append_refusals(lib):
    c = cache()
    assert append4(lib, None) == INV
    calls = (lambda **o: append4(lib, c, **o), lambda **o: append16(lib, **o))
    for call in calls:
        for over in (dict(q=None), dict(k=None), dict(v=None), dict(qo=None), dict(cos=None), dict(sin=None),
                     dict(pos=None), dict(slots=None), dict(rows=0), dict(T=-1), dict(H=0), dict(H=7), dict(axes=0),
                     dict(axes=5, axis=bytes(32)), dict(axes=3), dict(axes=2, axis=bytes([2] * 32)),
                     dict(strides=[504, 128, 128, 512, 128, 128]), dict(strides=[512, 128, 120, 512, 128, 128]),
                     dict(strides=[1 << 32, 128, 128, 512, 128, 128])):
            assert call(**over) == INV, over
        for over in (dict(q=FAKE + 8), dict(ko=FAKE + 8), dict(vo=FAKE + 2), dict(cos=FAKE + 8), dict(pos=FAKE + 2),
                     dict(slots=FAKE + 4), dict(biases=(FAKE + 8, None, None)),
                     dict(strides=[516, 128, 128, 512, 128, 128])):
            assert call(**over) == MIS, over
        assert call(T=0) == _lib.FR_OK
        # an output over its input, laid out otherwise, would be written where tokens are still read
        assert call(strides=[512, 128, 128, 520, 128, 128], qo=FAKE) == INV
        assert call(strides=[512, 128, 128, 512, 136, 128], ko=FAKE) == INV
        assert call(strides=[512, 128, 128, 512, 128, 136], vo=FAKE) == INV
        assert call(strides=[512, 128, 128, 520, 136, 144], qo=FAKE + 64, ko=FAKE + 64, vo=FAKE + 64, T=0) == _lib.FR_OK
    for over in (dict(kp=None), dict(vp=None), dict(ps=0), dict(ps=24), dict(np_=0), dict(Hkv=0), dict(Hkv=3)):
        assert append16(lib, **over) == INV, over
    assert append16(lib, D=96) == UNS
    assert append16(lib, kp=FAKE + 8) == MIS and append16(lib, vp=FAKE + 8) == MIS


def test_gather_and_attention_refusals(lib):
    r = ctypes.byref(cache())
    g = lambda *a: lib.fr_kv4_gather(*a, None)  # noqa: E731
    assert g(None, FAKE, FAKE, FAKE, 4) == INV
    assert g(r, None, FAKE, FAKE, 4) == INV
    assert g(r, FAKE, None, None, 4) == INV
    assert g(r, FAKE, FAKE, FAKE, -1) == INV
    assert g(r, FAKE + 4, FAKE, FAKE, 4) == MIS
    assert g(r, FAKE, FAKE + 8, None, 4) == MIS
    assert g(r, FAKE, FAKE, None, 0) == _lib.FR_OK

    def attn(q=FAKE, qs=0, c=r, t=FAKE, n=FAKE, o=FAKE, B=2, H=8, mb=4, mk=64):
        return lib.fr_decode_attn_paged_kv4(q, qs, c, t, n, o, B, H, mb, mk, None)

    for over in (dict(q=None), dict(c=None), dict(t=None), dict(n=None), dict(o=None), dict(B=0), dict(H=0),
                 dict(H=7), dict(mb=0), dict(mk=-1), dict(mk=129), dict(qs=504), dict(qs=-512),
                 dict(mb=1 << 26, mk=1 << 30)):
        assert attn(**over) == INV, over
    for over in (dict(q=FAKE + 8), dict(o=FAKE + 8), dict(qs=516), dict(t=FAKE + 2), dict(n=FAKE + 2)):
        assert attn(**over) == MIS, over
    assert lib.fr_kv4_workspace_size(0, 8, 2, 64, 64) == 0
    assert lib.fr_kv4_workspace_size(2, 8, 2, 96, 64) == 0


def test_handle_checks():
    k = torch.zeros((3, 2, 32, 32), dtype=torch.uint8)
    s = torch.zeros((3, 2, 32, 2, 1, 2), dtype=torch.float16)
    bad = [(k.to(torch.int8), k, s), (k, k.to(torch.int8), s), (k, k[:2], s), (k, k, s[..., :1]), (k, k, s.float()),
           (k, k, s.transpose(1, 2)), (k, k.transpose(1, 2).contiguous().transpose(1, 2), s),
           (k.transpose(2, 3), k.transpose(2, 3), s), (k[0], k[0], s)]
    for args in bad:
        with pytest.raises(ValueError):
            A.KV4Cache(*args)
    with pytest.raises(ValueError, match="CUDA"):
        A.KV4Cache(k, k, s)
