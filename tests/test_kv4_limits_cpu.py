"""The sizes of a 4-bit cache that the entry points take and refuse, at their
borders (the header's limits; nothing is read)."""
from __future__ import annotations

import ctypes

import pytest

from forgert_b200 import _lib

FAKE = 0x10000          # never dereferenced: no slots
OK, INV = _lib.FR_OK, _lib.FR_ERR_INVALID_ARG
GB64 = 1 << 36


def gather(lib, **over):
    f = dict(k=FAKE, v=FAKE, scales=FAKE, num_pages=4, page_size=32, num_kv_heads=2, head_dim=64,
             page_stride=2048, head_stride=1024, row_stride=32)
    f.update(over)
    return lib.fr_kv4_gather(ctypes.byref(_lib.Kv4CacheStruct(**f)), FAKE, FAKE, FAKE, 0, None)


@pytest.mark.parametrize("over,want", [
    (dict(), OK),
    # a page's stride: below 2^32
    (dict(page_stride=(1 << 32) - 16), OK),
    (dict(page_stride=1 << 32), INV),
    # what the strides span together: below 2^36
    (dict(num_pages=1, page_stride=2048, head_stride=GB64 // 2 - 2048 - 1024, row_stride=32), OK),
    (dict(num_pages=1, page_stride=2048, head_stride=GB64 // 2 - 1024, row_stride=32), INV),
    (dict(num_pages=1, page_stride=2048, head_stride=GB64 // 2, row_stride=32), INV),
    (dict(num_pages=1, row_stride=GB64 // 32 - 256), OK),
    (dict(num_pages=1, row_stride=GB64 // 32), INV),
    (dict(num_pages=GB64 // 2048 - 2), OK),
    (dict(num_pages=GB64 // 2048 - 1), INV),
    # strides that a product would wrap
    (dict(num_pages=2**31 - 1, page_stride=(1 << 32) - 16), INV),
    (dict(head_stride=2**63 - 16), INV),
    (dict(row_stride=2**63 - 16), INV),
    (dict(num_pages=2**31 - 1, page_size=2**31 - 16, num_kv_heads=2**31 - 1), INV),
    # scales below 2^36: a row of 64 dims and one head has 8 bytes (K and V, scale and bias)
    (dict(num_pages=(1 << 29) - 1, page_size=16, num_kv_heads=1, page_stride=48, row_stride=32, head_stride=32), OK),
    (dict(num_pages=1 << 29, page_size=16, num_kv_heads=1, page_stride=48, row_stride=32, head_stride=32), INV),
])
def test_borders(lib, over, want):
    assert gather(lib, **over) == want


@pytest.mark.gpu
def test_workspace_size_of_lengths_that_no_call_takes(lib):
    assert lib.fr_kv4_workspace_size(2, 8, 2, 64, (1 << 30) - 1) > 0
    assert lib.fr_kv4_workspace_size(2, 8, 2, 64, 1 << 30) == 0
    assert lib.fr_kv4_workspace_size(2, 8, 2, 64, 2**31 - 1) == 0
