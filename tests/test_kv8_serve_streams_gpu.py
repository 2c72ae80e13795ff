"""kv8_serve.Server.step on the streams that the entry points take: none, a
torch stream, a raw handle; its row slots follow the step on the same stream."""
from __future__ import annotations

import pytest
import torch

from forgert_b200 import kv8_serve

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["none", "zero", "stream", "handle"])
def test_step_on_a_stream(kind):
    s = kv8_serve.Server(4, 4, 2, 64, 1, 16, 12, 48, 192, torch.int8, rope_rows=64)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    stream = {"none": None, "zero": 0, "stream": side, "handle": side.cuda_stream}[kind]
    torch.cuda.synchronize()
    with torch.cuda.stream(other):              # not the stream that the step is given
        s.new_lens.copy_(torch.tensor([3, 0, 17, 1], dtype=torch.int32))
        other.synchronize()
        s.step(21, stream)
    torch.cuda.synchronize()
    assert s.kv_lens.tolist() == [3, 0, 17, 1] and int(s.status) == 0
    assert s.offsets.tolist() == [0, 3, 3, 20, 21]
    assert s.row_positions.tolist() == [0, 0, 0, 0]
    slots = s.slots.tolist()
    assert s.row_slots.tolist() == [slots[0], -1, slots[3], slots[20]]
    s.new_lens.copy_(torch.tensor([0, 1, 1, -1], dtype=torch.int32))
    torch.cuda.synchronize()
    s.step(4, stream)
    torch.cuda.synchronize()
    assert s.row_positions.tolist() == [0, 0, 17, 0]
    slots = s.slots.tolist()
    assert s.row_slots.tolist() == [-1, slots[0], slots[1], -1]
