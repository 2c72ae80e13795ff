"""The serving loop of forgert_b200.kv8_serve: block tables, append, prefill,
read-back and attention over the 8-bit cache together, decode steps as a
replayed CUDA graph."""
from __future__ import annotations

import pytest

from forgert_b200 import kv8_serve

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,page_size", [((28, 4, 128), 64), ((14, 2, 64), 16)])
def test_serving_loop(heads, page_size, code):
    H, Hkv, D = heads
    r = kv8_serve.run(requests=7, layers=2, steps=20, code=code, num_heads=H, num_kv_heads=Hkv, head_dim=D,
                      page_size=page_size, longest=300, seed=3)
    assert r["status"] == 0
    assert r["pages_held"] + r["pages_free"] == r["pages"]
    # N(0, 1) values: the outputs (below 4) are rounded to fp16 and the
    # weights to 2^-12; the values compared with are read back as fp16, whose
    # half ulp of up to 2^-10 for |v| < 4 is averaged by the weights
    assert r["max_error"] <= 4 * (2.0 ** -11 + 2.0 ** -11) + 2.0 ** -10
