"""A small serving loop over the 8-bit paged cache: the operators together, as a
server calls them.

Requests come with prompts of different lengths, are decoded token by token,
end, and others start in their rows:

  paged_step              pages, positions and slots of the step's tokens,
                          packed in request order
  per layer
    qkv_rope_append_kv8   bias + RoPE, K/V coded into the layer's cache
    prefill_attn_causal   prompts, on the 16-bit K/V that the append returns
    decode_attn_paged_kv8 one token per request, on the 8-bit cache

A decode step (block tables, every layer's append and attention) is one CUDA
graph, replayed while the lengths, tables and free pages move on the device.
There are no weights: each layer's q, k, v projections are synthetic N(0, 1).

Usage: python -m forgert_b200.kv8_serve [--code int8|e4m3] [--requests N]
       [--layers N] [--steps N]
Prints the time of a decode step and how far the last step's attention is from
softmax attention in 64 bits over the cache read back with kv8_gather.
"""
from __future__ import annotations

import argparse
import math


class Server:
    """`rows` request slots over one pool of pages (shared by all layers, each
    with a cache of its own).

    A step's tokens are packed: token t of the step is row t of prefill's q, k
    and v.  decode's have one row per request instead, whether it takes part
    or not.
    """

    def __init__(self, rows: int, num_heads: int, num_kv_heads: int, head_dim: int, layers: int,
                 page_size: int, num_pages: int, max_len: int, max_tokens: int, dtype,
                 rope_rows: int = 16384, theta: float = 1e6):
        import torch

        from . import attention as A

        self.rows, self.H, self.Hkv, self.D = rows, num_heads, num_kv_heads, head_dim
        self.page_size, self.num_pages = page_size, num_pages
        self.max_len, self.max_tokens, self.rope_rows = max_len, max_tokens, rope_rows
        self.width = -(-max_len // page_size)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.kv_lens = torch.zeros(rows, **i32)
        self.new_lens = torch.zeros(rows, **i32)
        self.table = torch.full((rows, self.width), -1, **i32)
        self.free_pages = torch.arange(num_pages, **i32)
        self.free_count = torch.full((1,), num_pages, **i32)
        self.offsets = torch.zeros(rows + 1, **i32)
        # one entry more than a step writes: of a request without a token
        self.positions = torch.zeros(max_tokens + 1, **i32)
        self.slots = torch.full((max_tokens + 1,), -1, dtype=torch.int64, device="cuda")
        self.status = torch.zeros(1, **i32)
        # of each request's first token of the step; slot -1 without one
        self.row_positions = torch.zeros(rows, **i32)
        self.row_slots = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
        self.cos, self.sin = A.rope_tables_device(rope_rows, head_dim, theta)
        self.caches = [A.KV8Cache.empty(num_pages, page_size, num_kv_heads, head_dim, dtype)
                       for _ in range(layers)]
        # before any capture, once for good: the attention's partial states, the
        # step's counter, and what a prompt of any length splits into
        A.reserve_workspace(max(
            A.kv8_workspace_size(rows, num_heads, num_kv_heads, head_dim, max_len),
            max(A.prefill_workspace_size(n, num_heads, head_dim) for n in range(1, max_len + 1))))

    def step(self, max_tokens: int, stream=None) -> None:
        """Pages, positions and slots for new_lens, lengths moved on in place."""
        import torch

        from . import attention as A

        A.paged_step(self.kv_lens, self.new_lens, self.table, self.free_pages, self.free_count,
                     self.kv_lens, self.free_count, self.offsets, self.positions, self.slots,
                     self.status, self.rows, self.page_size, self.num_pages, self.width,
                     max_tokens, stream=stream)
        if not stream:
            stream = torch.cuda.default_stream()
        elif isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream)
        with torch.cuda.stream(stream):
            first = self.offsets[:-1]
            at = torch.where(self.offsets[1:] > first, first, self.max_tokens)
            torch.index_select(self.positions, 0, at, out=self.row_positions)
            torch.index_select(self.slots, 0, at, out=self.row_slots)

    def append(self, layer: int, q, k, v, q_out, k_out, v_out, tokens: int, stream=None,
               positions=None, slots=None) -> None:
        """`tokens` rows at `positions` and `slots`, by default the packed tokens'."""
        from . import attention as A

        A.qkv_rope_append_kv8(q, k, v, q_out, k_out, v_out, self.cos, self.sin,
                              self.positions if positions is None else positions,
                              self.slots if slots is None else slots, self.caches[layer], tokens,
                              self.H, self.rope_rows, stream=stream)

    def decode(self, layer: int, q, k, v, out, stream=None) -> None:
        """One layer of a step in which every request gets one token or none:
        row b of q, k, v and out is request b's (a request that takes no part
        has no slot: nothing of it is turned or cached, and its output means
        nothing)."""
        from . import attention as A

        self.append(layer, q, k, v, q, None, None, self.rows, stream, self.row_positions, self.row_slots)
        A.decode_attn_paged_kv8(q, self.caches[layer], self.table, self.kv_lens, out, self.rows,
                                self.H, self.width, self.max_len, stream=stream)

    def prefill(self, layer: int, q, k, v, lens) -> list:
        """Prompts of the step, one after the other in q, k, v; their attention."""
        import torch

        from . import attention as A

        k16, v16 = torch.empty_like(k), torch.empty_like(v)
        self.append(layer, q, k, v, q, k16, v16, len(q))
        outs, at = [], 0
        for n in lens:
            out = torch.empty_like(q[at:at + n])
            A.prefill_attn_causal(q[at:at + n], k16[at:at + n], v16[at:at + n], out, n, self.H,
                                  self.Hkv, self.D)
            outs.append(out)
            at += n
        return outs


def attention64(server: Server, layer: int, row: int, q):
    """Softmax attention in 64 bits of q [H, D] over what the cache holds of
    request `row`."""
    import torch

    from . import attention as A

    n = int(server.kv_lens[row])
    pos = torch.arange(n, device="cuda")
    slots = server.table[row, pos // server.page_size].long() * server.page_size + pos % server.page_size
    k = torch.empty((n, server.Hkv, server.D), dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    A.kv8_gather(server.caches[layer], slots, k, v, n)
    group = server.H // server.Hkv
    k, v = (x.double().repeat_interleave(group, 1).transpose(0, 1) for x in (k, v))
    p = torch.softmax(k @ q.double()[:, :, None] / math.sqrt(server.D), 1)
    return (p * v).sum(1)


def run(requests: int = 16, layers: int = 4, steps: int = 64, code: str = "int8", num_heads: int = 28,
        num_kv_heads: int = 4, head_dim: int = 128, page_size: int = 64, longest: int = 1500,
        seed: int = 0) -> dict:
    import torch

    from . import attention as A

    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16)

    dtype = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}[code]
    max_len = longest + 2 * steps + 1
    s = Server(requests, num_heads, num_kv_heads, head_dim, layers, page_size,
               requests * -(-max_len // page_size), max_len, requests * longest, dtype)

    def admit(lens):
        """A step in which `lens` (row -> prompt tokens) start."""
        new = torch.zeros(requests, dtype=torch.int32)
        for row, n in lens.items():
            new[row] = n
        s.new_lens.copy_(new)
        tokens = sum(lens.values())
        s.step(tokens)
        assert int(s.status) == 0, f"step refused: {int(s.status)}"
        for layer in range(layers):
            s.prefill(layer, rand(tokens, num_heads, head_dim), rand(tokens, num_kv_heads, head_dim),
                      rand(tokens, num_kv_heads, head_dim), [lens[r] for r in sorted(lens)])

    lengths = torch.randint(1, longest + 1, (requests,), generator=host).tolist()
    admit(dict(enumerate(lengths)))

    # one decode step of every request as a graph
    q, k, v = (rand(layers, requests, n, head_dim) for n in (num_heads, num_kv_heads, num_kv_heads))
    out = torch.zeros_like(q)
    s.new_lens.fill_(1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            s.step(requests, stream)
            for layer in range(layers):
                s.decode(layer, q[layer], k[layer], v[layer], out[layer], stream)
    torch.cuda.current_stream().wait_stream(stream)

    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)

    def decode(count):
        ms = 0.0
        for _ in range(count):
            for x in (q, k, v):
                x.normal_(generator=gen)
            begin.record()
            graph.replay()
            end.record()
            end.synchronize()
            ms += begin.elapsed_time(end)
        return ms / max(1, count)

    decode(steps)
    # every third request ends, the next step starts others in their rows
    leaving = list(range(0, requests, 3))
    s.new_lens.zero_()
    s.new_lens[leaving] = -1
    s.step(requests)
    admit({row: int(torch.randint(1, longest + 1, (1,), generator=host)) for row in leaving})
    s.new_lens.fill_(1)
    ms = decode(steps)
    held = int((torch.div(s.kv_lens + page_size - 1, page_size, rounding_mode="floor")).sum())
    worst = 0.0
    for layer in range(layers):
        for row in range(requests):
            want = attention64(s, layer, row, q[layer, row])
            worst = max(worst, float((out[layer, row].double() - want).abs().max()))
    assert A.device_error() == 0
    return {"us_per_step": ms * 1e3, "max_error": worst, "status": int(s.status),
            "pages_held": held, "pages_free": int(s.free_count), "pages": s.num_pages,
            "tokens_held": int(s.kv_lens.sum())}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--code", choices=("int8", "e4m3"), default="int8")
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--steps", type=int, default=64)
    a = ap.parse_args()
    r = run(a.requests, a.layers, a.steps, a.code)
    print(f"{a.requests} requests, {r['tokens_held']} tokens held in {r['pages_held']} of {r['pages']} pages "
          f"({a.code}): {r['us_per_step']:.1f} us per decode step of {a.layers} layers; "
          f"attention is off by {r['max_error']:.1e} at most")


if __name__ == "__main__":
    main()
