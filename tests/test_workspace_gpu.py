"""The library's workspace when it grows: graphs captured before go on with the
one they were captured with."""
from __future__ import annotations

import json
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from forgert_b200 import attention as A
from forgert_b200._lib import load

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]


def in_a_fresh_process(script: str) -> dict:
    res = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, cwd=ROOT, timeout=300,
                         env=dict(os.environ, PYTHONPATH=str(ROOT)))
    assert res.returncode == 0, res.stderr[-2000:]
    return json.loads(res.stdout.strip().splitlines()[-1])


def long_kv8_call():
    """One sequence whose units are cut into many pieces, merged in two levels."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    n, H, Hkv, D, ps = 40000, 28, 4, 128, 64
    pages = -(-n // ps)
    k, v = (torch.randint(-127, 128, (pages, Hkv, ps, D), generator=gen, device="cuda", dtype=torch.int8) for _ in range(2))
    scales = torch.full((pages, Hkv, ps // 16, 2), 0.02, device="cuda")
    q = torch.randn((1, H, D), generator=gen, device="cuda").half()
    out, table = torch.zeros_like(q), torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    cache, lens = A.KV8Cache(k, v, scales), torch.tensor([n], dtype=torch.int32, device="cuda")
    A.reserve_workspace(A.kv8_workspace_size(1, H, Hkv, D, n))
    return out, lambda s=None: A.decode_attn_paged_kv8(q, cache, table, lens, out, 1, H, pages, n, stream=s)


def long_fp16_call():
    gen = torch.Generator(device="cuda").manual_seed(2)
    B, H, Hkv, D, n = 3, 28, 4, 128, 9000
    k, v = (torch.randn((B * n, Hkv, D), generator=gen, device="cuda").half() for _ in range(2))
    q = torch.randn((B, H, D), generator=gen, device="cuda").half()
    out, at = torch.zeros_like(q), torch.arange(B, device="cuda") * n
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    A.reserve_workspace(A.decode_workspace_size(B, H, Hkv, D, n))
    return out, lambda s=None: A.decode_attn_batched(q, k, v, at, lens, out, B, H, Hkv, D, B * n, n, stream=s)


@pytest.mark.parametrize("make", [long_kv8_call, long_fp16_call])
def test_a_captured_graph_outlives_growth(make):
    out, call = make()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(s)
        s.synchronize()
        want = out.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(s)
    torch.cuda.synchronize()
    kept = []
    for _ in range(3):
        before = load().fr_allocated_bytes()
        A.reserve_workspace(before)                        # more than the newest: it grows by a quarter
        assert load().fr_allocated_bytes() >= 2 * before
        kept.append(torch.full((before // 4,), float("nan"), device="cuda"))   # memory that was freed would be reused
        for _ in range(2):
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            out.fill_(float("nan"))
            call()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
    assert A.device_error() == 0


SERVE = r"""
import json, torch
from forgert_b200 import attention as A, kv8_serve
from forgert_b200._lib import load
H, Hkv, D, max_len = 28, 4, 128, 1629
s = kv8_serve.Server(1, H, Hkv, D, 1, 64, 26, max_len, max_len, torch.int8)
reserved = load().fr_allocated_bytes()
sizes = []
for n in (45, 700, 1240, 1500, max_len):
    s.new_lens.fill_(n)
    s.step(n)
    x = [torch.randn((n, h, D), device="cuda").half() for h in (H, Hkv, Hkv)]
    s.prefill(0, *x, [n])
    s.new_lens.fill_(-1)
    s.step(1)
    torch.cuda.synchronize()
    sizes.append(load().fr_allocated_bytes())
need = max(A.prefill_workspace_size(n, H, D) for n in range(1, max_len + 1))
r = kv8_serve.run(requests=1, layers=1, steps=8, longest=1500)
print(json.dumps(dict(reserved=reserved, sizes=sizes, need=need, error=A.device_error(), **r)))
"""


def test_serving_reserves_for_every_prompt():
    """A server with one row starts with a short prompt, captures its decode
    step and admits a long one, whose prefill splits."""
    r = in_a_fresh_process(SERVE)
    assert r["need"] > 0 and r["reserved"] >= r["need"]
    assert set(r["sizes"]) == {r["reserved"]}
    assert r["error"] == 0 and r["status"] == 0
    assert r["max_error"] <= 4 * (2.0 ** -11 + 2.0 ** -11) + 2.0 ** -10


FIRST_CALL = r"""
import json, torch
from forgert_b200 import attention as A
from oracle import kv8 as O
B, ps, width, pages, max_tokens = 1025, 16, 8, 6000, 20000
i32 = dict(dtype=torch.int32, device="cuda")
new = [(b * 7) % 19 for b in range(B)]
kv, newd = torch.zeros(B, **i32), torch.tensor(new, **i32)
table, stack, count = torch.full((B, width), -1, **i32), torch.arange(pages, **i32), torch.tensor([pages], **i32)
offsets, positions = torch.full((B + 1,), -7, **i32), torch.full((max_tokens,), -7, **i32)
slots, status = torch.full((max_tokens,), -7, dtype=torch.int64, device="cuda"), torch.full((1,), -7, **i32)
dirty = [torch.full((1 << 19,), -1, **i32) for _ in range(64)]
torch.cuda.synchronize()
del dirty
torch.cuda.empty_cache()                    # what cudaMalloc gives next may hold ones
s = torch.cuda.Stream()                     # does not wait for the default stream
torch.cuda._sleep(400_000_000)              # a fifth of a second of work on the default stream
A.paged_step(kv, newd, table, stack, count, kv, count, offsets, positions, slots, status, B, ps, pages, width,
             max_tokens, stream=s)
torch.cuda.synchronize()
st, lens, tab, stk, n, off, pos, sl = O.step([0] * B, new, [[-1] * width for _ in range(B)], list(range(pages)), pages, ps, max_tokens)
print(json.dumps(dict(status=int(status), want=st, lens=kv.tolist() == lens, table=table.tolist() == tab, count=int(count) == n,
                      offsets=offsets.tolist() == off, positions=positions.tolist() == pos, slots=slots.tolist() == sl,
                      error=A.device_error())))
"""


def test_first_growth_on_a_non_blocking_stream():
    """The counters are zero before the first kernel reads them, whatever the
    default stream is busy with."""
    r = in_a_fresh_process(FIRST_CALL)
    assert r == dict(status=0, want=0, lens=True, table=True, count=True, offsets=True, positions=True, slots=True, error=0)
