"""Decode steps of forgert_b200.kv8_serve.Server in which some requests sit
out, end or start: every live request and every layer's cache are held to the
plain statement (oracle.kv8), step by step, through one captured graph.

The attention's bound is that of its own tests: |x - r| <= 2^-11 |r| +
(2^-11 + 2^-13 + 2 D 2^-23 S) M + 1e-7, with M = sum_t p_t |v_t| and
S = max_t sum_i |q_i k_ti| / sqrt(D).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from forgert_b200 import attention as A
from forgert_b200 import kv8_serve
from oracle import kv8 as O

pytestmark = pytest.mark.gpu

TORCH = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class Twin:
    """The server's state in plain Python and numpy."""

    def __init__(self, s, code, layers):
        self.s, self.code = s, code
        self.state = [[0] * s.rows, [[-1] * s.width for _ in range(s.rows)], s.free_pages.tolist(), s.num_pages]
        shape = (s.num_pages, s.Hkv, s.page_size, s.D)
        self.caches = [(np.zeros(shape, np.uint8), np.zeros(shape, np.uint8),
                        np.zeros((s.num_pages, s.Hkv, s.page_size // 16, 2), np.float32)) for _ in range(layers)]
        self.cos, self.sin = s.cos.cpu().numpy(), s.sin.cpu().numpy()

    def step(self, new, max_tokens):
        st, *rest = O.step(self.state[0], new, self.state[1], self.state[2], self.state[3], self.s.page_size, max_tokens)
        self.state = rest[:4]
        self.offsets, self.positions, self.slots = rest[4:]
        return st

    def append(self, layer, q, k, v):
        """Packed tokens, in the step's order; their turned queries in fp16."""
        n, (kc, vc, sc) = len(q), self.caches[layer]
        pos, slots = np.array([self.positions[:n]], np.int64), np.array(self.slots[:n], np.int64)
        return O.append(q, k, v, [None] * 3, self.cos, self.sin, pos, [0] * (self.s.D // 2), slots, kc, vc, sc,
                        self.code)[0].astype(np.float16)

    def same(self):
        s = self.s
        assert s.kv_lens.tolist() == self.state[0] and int(s.free_count) == self.state[3]
        assert s.table.tolist() == self.state[1]
        for cache, (kc, vc, sc) in zip(s.caches, self.caches):
            assert np.array_equal(cache.scales.cpu().numpy(), sc)
            assert np.array_equal(cache.k.view(torch.uint8).cpu().numpy(), kc)
            assert np.array_equal(cache.v.view(torch.uint8).cpu().numpy(), vc)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("H,Hkv,D,ps", [(12, 2, 128, 16), (14, 2, 64, 48)])
def test_requests_sit_out_end_and_start(H, Hkv, D, ps, code):
    rng = np.random.default_rng(H)
    R, layers, max_len = 6, 2, 96
    s = kv8_serve.Server(R, H, Hkv, D, layers, ps, R * -(-max_len // ps), max_len, R * max_len, TORCH[code], rope_rows=256)
    for c in s.caches:
        for x in (c.k, c.v, c.scales):
            x.view(torch.uint8).zero_()
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
            want = twin.append(layer, *[a[layer][live] for a in x]) if live else None
            got = q[layer].cpu().numpy()
            kc, vc, sc = twin.caches[layer]
            if not live:
                continue
            assert np.array_equal(got[live], want), new
            r, mass, big = O.attention(got, O.values(kc, sc, 0, code), O.values(vc, sc, 1, code), twin.state[1], twin.state[0])
            tol = 2.0 ** -11 * np.abs(r) + (2.0 ** -11 + 2.0 ** -13 + 2 * D * 2.0 ** -23 * big) * mass + 1e-7
            err = np.abs(out[layer].cpu().numpy().astype(np.float64) - r)
            assert (err[live] <= tol[live]).all(), new
        twin.same()
    assert A.device_error() == 0
