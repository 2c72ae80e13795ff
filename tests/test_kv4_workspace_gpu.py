"""The 4-bit decode attention and the library's workspace: captures that would
need more are refused, graphs captured before it grows go on, two graphs share it."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from forgert_b200 import attention as A
from oracle import kv4 as O
from oracle import kv8

pytestmark = pytest.mark.gpu


def case(rng, lens, H, Hkv, D, ps=32):
    need = [-(-n // ps) for n in lens]
    table = np.full((len(lens), max(need)), -1, np.int32)
    ids = rng.permutation(sum(need))
    for b, n in enumerate(need):
        table[b, :n] = ids[sum(need[:b]):sum(need[:b]) + n]
    kc, vc = (rng.integers(0, 256, (sum(need), Hkv, ps, D // 2), dtype=np.uint8) for _ in range(2))
    a = np.full((sum(need), Hkv, ps, 2, D // 64), 0.25)
    sc = np.stack([a, -7.5 * a], -1).astype(np.float16)
    q = rng.standard_normal((len(lens), H, D)).astype(np.float16)
    want, _, _ = kv8.attention(q, O.values(kc, sc, 0), O.values(vc, sc, 1), table, lens)
    dev = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    cache = A.KV4Cache(dev(kc), dev(vc), dev(sc))
    out = torch.zeros_like(dev(q))
    args = (dev(q), cache, dev(table), torch.tensor(lens, dtype=torch.int32, device="cuda"), out, len(lens), H, table.shape[1],
            max(lens))
    return args, out, want


def near(out, want):
    e = out.cpu().numpy().astype(np.float64) - want
    return np.linalg.norm(e) <= 1.1 * 2.0 ** -11 * np.linalg.norm(want)


def test_graphs_that_share_and_outlive_the_workspace():
    """Two graphs of different calls replayed in turn, then again after a larger
    call has outgrown the buffer that they were captured with."""
    rng = np.random.default_rng(0)
    cases = [case(rng, [700, 3, 512], 28, 4, 128), case(rng, [2000], 14, 2, 64)]
    A.reserve_workspace(max(A.kv4_workspace_size(3, 28, 4, 128, 700), A.kv4_workspace_size(1, 14, 2, 64, 2000)))
    s = torch.cuda.Stream()
    graphs = []
    for args, _, _ in cases:
        torch.cuda.synchronize()
        A.decode_attn_paged_kv4(*args, stream=s)            # first use sets the kernel up
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            A.decode_attn_paged_kv4(*args, stream=s)
        graphs.append(g)

    def replay():
        for _, out, _ in cases:
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(3):
            for g in graphs:
                g.replay()
        torch.cuda.synchronize()
        for _, out, want in cases:
            assert near(out, want)

    replay()
    A.reserve_workspace(64 << 20)
    replay()
    assert A.device_error() == 0


REFUSED = """
import sys
sys.path.insert(0, {root!r})
import torch
from forgert_b200 import attention as A
from forgert_b200._lib import ForgeRTError
from tests.test_kv4_workspace_gpu import case
import numpy as np
args, out, want = case(np.random.default_rng(1), [600], 28, 4, 128)
s = torch.cuda.Stream()
A.device_error()
A.kv4_workspace_size(1, 28, 4, 128, 600)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    try:
        A.decode_attn_paged_kv4(*args, stream=s)
        print("captured")
    except ForgeRTError as e:
        print("refused", e.status)
"""


def test_a_capture_without_workspace_is_refused():
    root = str(Path(__file__).resolve().parents[1])
    r = subprocess.run([sys.executable, "-c", REFUSED.format(root=root)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.split() == ["refused", "6"]


def test_two_calls_on_one_stream_and_the_same_request_twice():
    """Rows of a batch may name the same pages: the outputs are those of one."""
    rng = np.random.default_rng(2)
    args, out, want = case(rng, [300, 41], 12, 2, 128)
    q, cache, table, lens, _, _, H, width, longest = args
    both = torch.cat([q, q])
    res = torch.zeros_like(both)
    A.decode_attn_paged_kv4(both, cache, torch.cat([table, table]), torch.cat([lens, lens]), res, 4, H, width, longest)
    A.decode_attn_paged_kv4(*args)
    torch.cuda.synchronize()
    assert near(res[:2], want) and near(res[2:], want) and near(out, want)
    assert torch.equal(res[:2], res[2:])
