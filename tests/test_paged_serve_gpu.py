"""Serving from 4-bit and 16-bit pages (forgert_b200.kv8_serve with those caches):
block tables, append, prefill, read-back and attention together, decode steps as
one replayed graph, requests that sit out, end and start.

The attention's bounds are those of its own tests (test_kv4_decode_gpu.py; at 16
bits |x - r| <= 2^-11 |r| + (2^-13 + 2 D 2^-23 S) M + 1e-7 with
M = sum_t p_t |v_t|, the weights in two fp16 parts).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from forgert_b200 import attention as A
from forgert_b200 import kv8_serve
from oracle import kv4 as O
from oracle import kv8

pytestmark = pytest.mark.gpu

TORCH = {"int4": torch.uint8, "fp16": torch.float16}


@pytest.mark.parametrize("code", ["int4", "fp16"])
@pytest.mark.parametrize("heads,page_size", [((28, 4, 128), 64), ((14, 2, 64), 16)])
def test_serving_loop(heads, page_size, code):
    H, Hkv, D = heads
    r = kv8_serve.run(requests=7, layers=2, steps=20, code=code, num_heads=H, num_kv_heads=Hkv, head_dim=D,
                      page_size=page_size, longest=300, seed=3)
    assert r["status"] == 0
    assert r["pages_held"] + r["pages_free"] == r["pages"]
    # N(0, 1) values: the outputs (below 4) are rounded to fp16 and the weights to
    # 2^-11; the values compared with are read back as fp16, whose half ulp of up
    # to 2^-10 for |v| < 4 is averaged by the weights
    assert r["max_error"] <= 4 * (2.0 ** -11 + 2.0 ** -11) + 2.0 ** -10


class Twin:
    """The server's state in plain Python and numpy."""

    def __init__(self, s, code, layers):
        self.s, self.code = s, code
        self.state = [[0] * s.rows, [[-1] * s.width for _ in range(s.rows)], s.free_pages.tolist(), s.num_pages]
        if code == "int4":
            shape = (s.num_pages, s.Hkv, s.page_size, s.D // 2)
            self.caches = [(np.zeros(shape, np.uint8), np.zeros(shape, np.uint8),
                            np.zeros((s.num_pages, s.Hkv, s.page_size, 2, s.D // 64, 2), np.float16)) for _ in range(layers)]
        else:
            shape = (s.num_pages, s.page_size, s.Hkv, s.D)
            self.caches = [(np.zeros(shape, np.float16), np.zeros(shape, np.float16)) for _ in range(layers)]
        self.cos, self.sin = s.cos.cpu().numpy(), s.sin.cpu().numpy()

    def step(self, new, max_tokens):
        st, *rest = kv8.step(self.state[0], new, self.state[1], self.state[2], self.state[3], self.s.page_size, max_tokens)
        self.state = rest[:4]
        self.offsets, self.positions, self.slots = rest[4:]
        return st

    def append(self, layer, q, k, v):
        """Packed tokens, in the step's order; their turned queries in fp16."""
        n, cache = len(q), self.caches[layer]
        pos, slots = np.array([self.positions[:n]], np.int64), np.array(self.slots[:n], np.int64)
        rows = O.turned(q, k, v, [None] * 3, self.cos, self.sin, pos, [0] * (self.s.D // 2))
        if self.code == "int4":
            O.put(rows[1], cache[0], cache[2], 0, slots)
            O.put(rows[2], cache[1], cache[2], 1, slots)
        else:
            for pool, x in zip(cache, rows[1:]):
                pool.reshape(-1, *x.shape[1:])[slots] = x.astype(np.float16)
        return rows[0].astype(np.float16)

    def same(self):
        s = self.s
        assert s.kv_lens.tolist() == self.state[0] and int(s.free_count) == self.state[3]
        assert s.table.tolist() == self.state[1]
        for cache, want in zip(s.caches, self.caches):
            have = (cache.k, cache.v, cache.scales) if self.code == "int4" else cache
            for x, y in zip(have, want):
                assert np.array_equal(x.cpu().numpy(), y)

    def attention(self, layer, q):
        """64-bit outputs and their bounds."""
        cache, (lens, table) = self.caches[layer], self.state[:2]
        D = self.s.D
        if self.code == "int4":
            kc, vc, sc = cache
            r, _, _ = kv8.attention(q, O.values(kc, sc, 0), O.values(vc, sc, 1), table, lens)
            _, whole, big = O.masses(q, kc, vc, sc, table, lens)
            return r, 2.0 ** -11 * np.abs(r) + (2.0 ** -13 + 2 * (D + 4) * 2.0 ** -23 * big) * whole + 1e-7
        k, v = (x.astype(np.float64).transpose(0, 2, 1, 3) for x in cache)
        r, mass, big = kv8.attention(q, k, v, table, lens)
        return r, 2.0 ** -11 * np.abs(r) + (2.0 ** -13 + 2 * D * 2.0 ** -23 * big) * mass + 1e-7


@pytest.mark.parametrize("code", ["int4", "fp16"])
@pytest.mark.parametrize("H,Hkv,D,ps", [(12, 2, 128, 16), (14, 2, 64, 48)])
def test_requests_sit_out_end_and_start(H, Hkv, D, ps, code):
    rng = np.random.default_rng(H)
    R, layers, max_len = 6, 2, 96
    s = kv8_serve.Server(R, H, Hkv, D, layers, ps, R * -(-max_len // ps), max_len, R * max_len, TORCH[code], rope_rows=256)
    for c in s.caches:
        for x in ((c.k, c.v, c.scales) if code == "int4" else c):
            x.zero_()
    twin = Twin(s, code, layers)

    def half(*shape):
        return rng.standard_normal(shape).astype(np.float16)

    prompts = [5, 40, 9, 31, 1, 16]
    s.new_lens.copy_(torch.tensor(prompts, dtype=torch.int32))
    s.step(sum(prompts))
    assert twin.step(prompts, sum(prompts)) == 0
    for layer in range(layers):
        x = [half(sum(prompts), n, D) for n in (H, Hkv, Hkv)]
        twin.append(layer, *x)
        s.prefill(layer, *[torch.from_numpy(a).cuda() for a in x], prompts)
    torch.cuda.synchronize()
    twin.same()

    q, k, v = (torch.zeros((layers, R, n, D), dtype=torch.float16, device="cuda") for n in (H, Hkv, Hkv))
    out = torch.zeros_like(q)
    s.new_lens.zero_()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            s.step(R, stream)
            for layer in range(layers):
                s.decode(layer, q[layer], k[layer], v[layer], out[layer], stream)
    torch.cuda.current_stream().wait_stream(stream)

    steps = [[0, 1, 1, 1, 1, 1], [1, 1, 1, 1, 1, 1], [0, 1, 0, 0, 1, 0], [1, -1, 1, 0, 1, 1], [0, 0, 0, 0, 0, 0], [0, 0, 0, 0, 0, 1],
             [1, 1, 0, 1, -2, 1], [-1, 1, 1, 0, 0, 1], [1, 1, 1, 1, 1, 1], [1, max_len, 1, 1, 0, 1], [0, 1, 1, 0, 1, 1]]
    for new in steps:
        x = [half(layers, R, n, D) for n in (H, Hkv, Hkv)]
        for buf, a in zip((q, k, v), x):
            buf.copy_(torch.from_numpy(a))
        s.new_lens.copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        status = twin.step(new, R)
        assert int(s.status) == status == (2 if max_len in new else 0)
        live = [b for b in range(R) if new[b] == 1] if status == 0 else []
        for layer in range(layers):
            if not live:
                continue
            want = twin.append(layer, *[a[layer][live] for a in x])
            got = q[layer].cpu().numpy()
            assert np.array_equal(got[live], want), new
            r, tol = twin.attention(layer, got)
            err = np.abs(out[layer].cpu().numpy().astype(np.float64) - r)
            assert (err[live] <= tol[live]).all(), new
        twin.same()
    assert A.device_error() == 0
