"""GPU tests of fr_paged_step against the plain statement (oracle.kv8.step).
Whole numbers: everything has to be equal."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from forgert_b200 import _lib
from forgert_b200 import attention as A
from forgert_b200._lib import ForgeRTError
from oracle import kv8 as O

pytestmark = pytest.mark.gpu


class Server:
    """The arrays of a server on the device, and their plain twin."""

    def __init__(self, B, ps, pages, width, max_tokens, seed=0):
        rng = np.random.default_rng(seed)
        self.B, self.ps, self.pages, self.width, self.max_tokens = B, ps, pages, width, max_tokens
        stack = rng.permutation(pages).tolist()
        self.plain = [[0] * B, [[-1] * width for _ in range(B)], stack, pages]
        i32 = dict(dtype=torch.int32, device="cuda")
        self.kv = torch.zeros(B, **i32)
        self.table = torch.full((B, width), -1, **i32)
        self.stack = torch.tensor(stack, **i32)
        self.count = torch.tensor([pages], **i32)
        self.out = dict(offsets=torch.empty(B + 1, **i32), positions=torch.empty(max_tokens, **i32),
                        slots=torch.empty(max_tokens, dtype=torch.int64, device="cuda"), status=torch.empty(1, **i32))

    def launch(self, new, kv_out=None, count_out=None, stream=None):
        o = self.out
        A.paged_step(self.kv, new, self.table, self.stack, self.count, self.kv if kv_out is None else kv_out,
                     self.count if count_out is None else count_out, o["offsets"], o["positions"], o["slots"], o["status"],
                     self.B, self.ps, self.pages, self.width, self.max_tokens, stream=stream)

    def step(self, new, in_place=True):
        for x in self.out.values():
            x.fill_(-77)
        kv_out = None if in_place else torch.full_like(self.kv, -5)
        count_out = None if in_place else torch.full_like(self.count, -5)
        self.launch(torch.tensor(new, dtype=torch.int32, device="cuda"), kv_out, count_out)
        st, *rest = O.step(self.plain[0], new, self.plain[1], self.plain[2], self.plain[3], self.ps, self.max_tokens)
        self.plain, (offsets, positions, slots) = rest[:4], rest[4:]
        if not in_place:
            self.kv, self.count = kv_out, count_out
        assert int(self.out["status"]) == st
        assert self.kv.tolist() == self.plain[0] and int(self.count) == self.plain[3]
        assert self.table.tolist() == self.plain[1]
        assert self.stack.tolist() == self.plain[2]
        assert self.out["offsets"].tolist() == offsets
        assert self.out["positions"].tolist() == positions
        assert self.out["slots"].tolist() == slots
        assert A.device_error() == 0
        return st


@pytest.mark.parametrize("B,ps,max_tokens", [(1, 16, 64), (5, 48, 300), (33, 16, 1000), (64, 64, 5000), (1025, 32, 20000)])
@pytest.mark.parametrize("in_place", [True, False])
def test_a_server_run(B, ps, max_tokens, in_place):
    """Requests start, decode, idle, end and start again; the pool is tight, so
    some steps are refused and change nothing."""
    rng = np.random.default_rng(B)
    width = 12
    s = Server(B, ps, max(4, B * width // 3), width, max_tokens, B)
    seen = set()
    for i in range(25):
        kind = rng.choice(["decode", "idle", "end", "long"], B, p=[0.6, 0.1, 0.15, 0.15])
        room = width * ps - np.array(s.plain[0])
        new = [{"decode": min(1, r), "idle": 0, "end": -int(rng.integers(1, 9)), "long": int(rng.integers(0, min(r, max_tokens // (B // 4 + 1)) + 1))}[k]
               for k, r in zip(kind, room)]
        seen.add(s.step([int(n) for n in new], in_place))
    assert 0 in seen


@pytest.mark.parametrize("B", [8192, 8191, 1024, 31])
def test_large_batches(B):
    rng = np.random.default_rng(B)
    s = Server(B, 16, 3 * B, 4, 40000, 1)
    assert s.step([int(x) for x in rng.integers(0, 4, B)]) == 0
    s.step([int(x) for x in rng.integers(-1, 5, B)])
    s.step([1] * B)


def test_long_prompts_in_many_ctas():
    s = Server(9, 64, 4000, 1200, 150000)
    assert s.step([60001, 0, 1, 64, 65, 30000, 0, 127, 17]) == 0
    assert s.step([1, 5, -1, 1, 1, -2, 0, 1, 48000]) == 0


def test_refused_steps():
    s = Server(4, 16, 10, 5, 64)
    assert s.step([16, 17, 1, 0]) == 0                    # 1 + 2 + 1 pages
    before = [list(s.plain[0]), s.plain[3]]
    assert s.step([64, 1, 1, 0]) == 3                     # too many tokens
    assert s.step([60, 0, 0, 0]) == 0
    assert s.step([0, 48, 0, 16]) == 1                    # 3 + 1 pages, 2 free
    assert s.step([-1, 48, 0, 16]) == 0                   # the ended request's pages are enough
    assert s.step([81, 0, 0, 0]) == 2                     # past the block-table row
    assert before
    s.kv[2] = -1
    s.plain[0][2] = -1
    assert s.step([1, 0, 0, 0]) == 2
    s.kv[2] = 1
    s.plain[0][2] = 1
    for count in (-1, 11, 10):                            # 10: the released pages would overflow the stack
        keep = int(s.count)
        s.count.fill_(count)
        s.plain[3] = count
        assert s.step([1, -1, 0, 0]) == 4
        s.count.fill_(keep)
        s.plain[3] = keep
    assert s.step([1, -1, 0, 0]) == 0


def test_sums_past_32_bits_are_refused():
    s = Server(8192, 1024, 64, 1 << 10, 1024)
    new = torch.full((8192,), 1 << 20, dtype=torch.int32, device="cuda")     # 2^33 tokens
    s.launch(new)
    assert int(s.out["status"]) == _lib.FR_STEP_TOO_MANY
    assert int(s.kv.abs().sum()) == 0 and int(s.count) == 64 and int(s.out["slots"].max()) == -1


def test_graph_replays_a_server():
    """Captured once with the arrays updated in place, replayed as a decode loop."""
    s = Server(40, 16, 400, 8, 3000)
    A.reserve_workspace(1 << 20)
    new = torch.zeros(40, dtype=torch.int32, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            s.launch(new, stream=st)
    rng = np.random.default_rng(3)
    for i in range(12):
        want = [int(x) for x in rng.integers(-1, 9, 40)]
        new.copy_(torch.tensor(want, dtype=torch.int32))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        status, *rest = O.step(s.plain[0], want, s.plain[1], s.plain[2], s.plain[3], 16, 3000)
        s.plain = rest[:4]
        assert int(s.out["status"]) == status == 0
        assert s.kv.tolist() == s.plain[0] and s.table.tolist() == s.plain[1] and s.out["slots"].tolist() == rest[6]


def test_refusals():
    s = Server(4, 16, 10, 5, 64)
    new = torch.zeros(4, dtype=torch.int32, device="cuda")
    for over in (dict(B=0), dict(ps=0), dict(pages=0), dict(width=0), dict(max_tokens=0)):
        keep = {k: getattr(s, k) for k in over}
        for k, v in over.items():
            setattr(s, k, v)
        with pytest.raises(ForgeRTError, match="invalid argument"):
            s.launch(new)
        for k, v in keep.items():
            setattr(s, k, v)
    with pytest.raises(ForgeRTError, match="invalid argument"):
        s.launch(new, kv_out=new)
    with pytest.raises(ValueError):
        s.launch(new.cpu())
