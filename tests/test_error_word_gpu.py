"""The device's error word when calls fail in two ways: a wait that ran out is
reported whatever was recorded before it."""
from __future__ import annotations

import pytest
import torch

from forgert_b200 import attention as A
from forgert_b200._lib import FR_ERR_INVALID_ARG, FR_ERR_TIMEOUT, load
from test_exchange_gpu import DEV_TIMEOUT_PEER, new_buffer

pytestmark = pytest.mark.gpu

BAD_INDEX = 4


def bad_position():
    z = lambda *shape, dtype=torch.float16: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
    cache = A.KV8Cache(z(2, 1, 16, 64, dtype=torch.int8), z(2, 1, 16, 64, dtype=torch.int8), z(2, 1, 1, 2, dtype=torch.float32))
    A.qkv_rope_append_kv8(z(1, 1, 64), z(1, 1, 64), z(1, 1, 64), z(1, 1, 64), None, None, z(4, 32, dtype=torch.float32),
                          z(4, 32, dtype=torch.float32), torch.full((1, 1), 4, dtype=torch.int32, device="cuda"),
                          z(1, dtype=torch.int64), cache, 1, 1, 4)


def missing_peer():
    """A call of two ranks of which one never comes: its bounded wait runs out."""
    H, Hkv, D, T = 12, 2, 128, 256
    q, k, v = (torch.zeros(s, dtype=torch.float16, device="cuda") for s in ((H, D), (T, Hkv, D), (T, Hkv, D)))
    bufs = [new_buffer(H, D, 2)[0] for _ in range(2)]
    A.decode_attn_exchange(q, k, v, T, torch.empty_like(q), H, Hkv, D, bufs, 0, 2)
    torch.cuda.synchronize()


@pytest.mark.parametrize("first,second", [(bad_position, missing_peer), (missing_peer, bad_position)])
def test_a_timeout_is_not_hidden(first, second):
    assert A.device_error() == 0
    first()
    second()
    torch.cuda.synchronize()
    assert load().fr_get_device_error(0, None) == FR_ERR_TIMEOUT
    assert A.device_error() == DEV_TIMEOUT_PEER
    assert A.device_error() == 0
    bad_position()
    assert load().fr_get_device_error(0, None) == FR_ERR_INVALID_ARG
    assert A.device_error() == BAD_INDEX
