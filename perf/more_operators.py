"""Cases for appending to paged caches and for a paged cache held in 4 bits:
bias + rotary embedding + append through a slot map (16-bit pages; 4-bit
pages), read-back, and decode attention over 4 bits.

Each case is run either through the framework's entry points (`own` true) or
in plain torch operations in 32 bits.  Shapes are those of the Qwen2-0.5B,
1.5B and 7B layers that the benchmark and the tests use (H14 Hkv2 D64,
H12 Hkv2 D128, H28 Hkv4 D128), with multi-head and wide-group layouts beside
them.

Layouts.  16 bits: pages [num_pages, page_size, Hkv, D] fp16, of K and of V.
4 bits: codes [num_pages, Hkv, page_size, D / 2] bytes, dim 2i in the low
half of byte i, dim 2i + 1 in the high half; scales [num_pages, Hkv,
page_size, 2 (K, V), D / 64, 2 (scale, bias)] fp16, a pair for each row, kv head
and group of 64 dims.  A value is code * scale + bias with codes 0 .. 15:

  bias  = the largest fp16 number that is not above the group's minimum
  scale = the smallest fp16 number that is not below (maximum - bias) / 15
  code  = (x - bias) / scale, rounded to the nearest whole number, ties to even

in 32 bits, so no value is cut off and each is off by half a scale at most.
"""
import math
import random

import torch

own = False

GROUP = 64
ROPE_ROWS = 16384
THETA = 1e6


# --------------------------------------------------------------------- cases
def listed():
    attn = dict(op="attention", empty=0)
    app = dict(bias=True, axes=1, fresh=False)
    p16, p4 = dict(app, op="append16"), dict(app, op="append4")
    return [
        # one decoded token of one request of the smallest model, 16-bit pages
        dict(p16, name="append 16-bit, 1 token", H=14, Hkv=2, D=64, page=16, batch=1, tokens=1),
        # prompts of ragged length with image patches: three position axes, K and V kept for prefill attention
        dict(p16, name="append 16-bit, prompts", H=28, Hkv=4, D=128, page=32, batch=9, tokens=913, axes=3, fresh=True),
        # the same two uses of the 4-bit cache, and a decode step's new tokens between them
        dict(p4, name="append 4-bit, 1 token", H=14, Hkv=2, D=64, page=16, batch=1, tokens=1),
        dict(p4, name="append 4-bit, 64 tokens", H=28, Hkv=4, D=128, page=64, batch=64, tokens=1),
        dict(p4, name="append 4-bit, prompts", H=28, Hkv=4, D=128, page=32, batch=9, tokens=913, axes=3, fresh=True),
        # a cached prefix read back as 16-bit K/V to go on with a prompt: a short one, and three long ones
        dict(name="read back, 512", op="gather", Hkv=2, D=64, page=16, batch=1, max_kv=512),
        dict(name="read back, long", op="gather", Hkv=4, D=128, page=64, batch=3, max_kv=30011),
        # one short request of the smallest model: latency
        dict(attn, name="attention, 1 x 512", H=14, Hkv=2, D=64, page=16, batch=1, lo=512, hi=512),
        # odd lengths and pages, requests that hold nothing yet
        dict(attn, name="attention, odd", H=12, Hkv=2, D=128, page=48, batch=17, lo=1, hi=2999, empty=3),
        # the benchmark's ragged batch
        dict(attn, name="attention, 64 ragged", H=28, Hkv=4, D=128, page=64, batch=64, lo=1024, hi=8192),
        # as many requests of four times the length: what 4 bits make room for
        dict(attn, name="attention, 64 long", H=28, Hkv=4, D=128, page=64, batch=64, lo=8192, hi=32768),
        # one long context
        dict(attn, name="attention, 1 x 131072", H=28, Hkv=4, D=128, page=128, batch=1, lo=131072, hi=131072),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (8, 8, 64), (8, 2, 128), (16, 1, 128), (24, 2, 64)]


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append4", "append4", "append16", "append16", "gather"])
    page = rng.choice([16, 32, 48, 64, 128])
    H, Hkv, D = rng.choice(HEADS)
    if op in ("append16", "append4"):
        batch = _log(rng, 1, 200)
        return dict(op=op, H=H, Hkv=Hkv, D=D, page=page, batch=batch, tokens=rng.choice([1, _log(rng, 1, max(1, 8192 // batch))]),
                    axes=rng.choice([1, 3]), bias=rng.random() < 0.5, fresh=rng.random() < 0.5)
    if op == "gather":
        batch = _log(rng, 1, 16)
        return dict(op=op, Hkv=Hkv, D=D, page=page, batch=batch, max_kv=_log(rng, 16, 90000 // batch))
    batch = _log(rng, 1, 256)
    hi = _log(rng, 1, min(131072, 400_000_000 // (batch * Hkv * D), 2_000_000_000 // (batch * H * D)))
    return dict(op=op, H=H, Hkv=Hkv, D=D, page=page, batch=batch, lo=rng.choice([1, hi]) if batch == 1 else rng.randint(1, hi), hi=hi,
                empty=rng.randint(0, batch // 4))


def _up(a, b):
    return -(-a // b)


def _lens(case):
    """The requests' lengths: of the case alone, so that work() knows them."""
    r = random.Random("lengths %r" % sorted((k, v) for k, v in case.items() if k != "name"))
    op, n = case["op"], case["batch"]
    if op == "attention":
        held = [r.randint(case["lo"], case["hi"]) for _ in range(n)]
        return [0] * case["empty"] + held[case["empty"]:]
    if op == "gather":
        return [case["max_kv"]] + [r.randint(1, case["max_kv"]) for _ in range(n - 1)]
    held = [0 if case["fresh"] else r.randint(0, 4000) for _ in range(n)]      # (tokens held before, new tokens)
    return [(h, case["tokens"] if i == 0 else r.randint(1, case["tokens"])) for i, h in enumerate(held)]


def _row4(D):
    """Bytes of a row's K and V of one kv head in 4 bits."""
    return D + 2 * (D // GROUP) * 4


def work(case):
    op, lens = case["op"], _lens(case)
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    if op == "gather":
        n = sum(lens)
        return {"bytes": n * (Hkv * (_row4(D) + 4 * D) + 8), "flops": 4 * n * Hkv * D}
    H = case["H"]
    if op in ("append16", "append4"):
        n, last = sum(new for _, new in lens), max(h + new for h, new in lens)
        cached = Hkv * (4 * D if op == "append16" else _row4(D))
        rows = 2 if case["fresh"] else 1            # K and V are written back for prefill attention, or only read
        moved = n * (2 * H * D * 2 + rows * 2 * Hkv * D * 2 + cached + 8 + 4 * case["axes"]) + min(n, last) * 4 * D
        back = 0 if op == "append16" else n * (Hkv * (_row4(D) + 4 * D) + 8)
        return {"bytes": moved + back, "flops": n * (6 * H + (8 if op == "append16" else 20) * Hkv) * D}
    n = sum(lens)
    return {"bytes": n * Hkv * _row4(D) + 4 * sum(_up(x, page) for x in lens) + case["batch"] * (4 + 2 * H * D * 2), "flops": 4 * n * H * D}


# -------------------------------------------------------------------- inputs
def _pages(gen, have, page, spare, dev):
    """Pages of `have` pages per request, handed out in a shuffled order: (table, number of pages)."""
    have = torch.tensor(have, device=dev)
    total = int(have.sum()) + spare
    ids = torch.randperm(total, generator=gen, device=dev).int()
    at = torch.arange(max(1, int(have.max())), device=dev)
    first = have.cumsum(0) - have
    return torch.where(at < have[:, None], ids[(first[:, None] + at).clamp(max=total - 1)], -1).int().contiguous(), total


def _half_below(x):
    """The largest fp16 number that is not above x (|x| < 65504), in x's type."""
    step = torch.exp2((torch.frexp(x).exponent - 11).clamp(min=-24).double()).to(x.dtype)
    return torch.floor(x / step) * step


def _code(x):
    """Codes, scales and biases of rows [..., D] in groups of 64 dims: whole numbers [..., D] and two [..., D / 64]."""
    g = x.unflatten(-1, (-1, GROUP))
    bias = _half_below(g.amin(-1))
    fifteen = torch.full_like(bias, 15.0)               # a number would be divided by as a product with its reciprocal
    scale = -_half_below(-((g.amax(-1) - bias) / fifteen))
    n = torch.where(scale[..., None] > 0, (g - bias[..., None]) / scale[..., None], 0.0).round()
    return n.flatten(-2), scale, bias


def _bytes(n):
    """Codes [..., D] as bytes [..., D / 2]."""
    n = n.to(torch.uint8)
    return n[..., 0::2] | n[..., 1::2] << 4


def _cache4(gen, case, pages, dev):
    """A pool of normal rows in 4 bits, K and V."""
    Hkv, page, D = case["Hkv"], case["page"], case["D"]
    codes = [torch.empty((pages, Hkv, page, D // 2), dtype=torch.uint8, device=dev) for _ in range(2)]
    scales = torch.empty((pages, Hkv, page, 2, D // GROUP, 2), dtype=torch.float16, device=dev)
    some = max(1, 2 ** 26 // (Hkv * page * D))
    for p in range(0, pages, some):
        for which in range(2):
            x = torch.randn((min(some, pages - p), Hkv, page, D), generator=gen, device=dev)
            n, scale, bias = _code(x)
            codes[which][p:p + some] = _bytes(n)
            scales[p:p + some, :, :, which] = torch.stack([scale, bias], -1).half()
    return dict(k=codes[0], v=codes[1], scales=scales)


def _slots(table, seq, pos, page):
    return table[seq, pos // page].long() * page + pos % page


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    op, lens, page = case["op"], _lens(case), case["page"]
    append = op in ("append16", "append4")
    held = [h + new for h, new in lens] if append else lens
    table, total = _pages(gen, [_up(x, page) for x in held], page, 3, dev)
    n, Hkv, D = len(lens), case["Hkv"], case["D"]
    seqs = torch.arange(n, device=dev)
    s = dict(case=case, table=table, pages=total)
    if op == "append16":
        pool = [torch.randn((total, page, Hkv, D), generator=gen, device=dev, dtype=torch.float16) for _ in range(2)]
        s.update(k=pool[0], v=pool[1])
    else:
        s.update(_cache4(gen, case, total, dev))
    if op == "attention":
        t = torch.tensor(held, device=dev)
        # what lies behind a request's end in its last page is nobody's: any codes, scales that are NaN
        ends = t % page
        last = table[seqs, ((t - 1) // page).clamp(min=0)].long()[ends > 0]
        behind = (torch.arange(page, device=dev) >= ends[ends > 0, None])[:, None, :, None, None, None]
        s["scales"][last] = s["scales"][last].masked_fill(behind, math.nan)
        q = torch.randn((n, case["H"], D), generator=gen, device=dev).half()
        return dict(s, q=q, kv_lens=t.int(), longest=max(held), out=torch.empty_like(q))
    if op == "gather":
        t = torch.tensor(lens, device=dev)
        seq = torch.repeat_interleave(seqs, t)
        slots = _slots(table, seq, torch.arange(len(seq), device=dev) - (t.cumsum(0) - t)[seq], page)
        out = torch.empty((len(seq), Hkv, D), dtype=torch.float16, device=dev)
        return dict(s, slots=slots, k_out=out, v_out=torch.empty_like(out))
    H = case["H"]
    before, new = torch.tensor([h for h, _ in lens], device=dev), torch.tensor([x for _, x in lens], device=dev)
    seq = torch.repeat_interleave(seqs, new)
    pos = torch.arange(len(seq), device=dev) - (new.cumsum(0) - new)[seq] + before[seq]
    T = len(seq)
    freq = torch.arange(D // 2, device=dev)
    if case["axes"] == 3:  # rows of a patch grid: time, height and width of each token, in sections of the frequencies
        positions = torch.stack([pos // 1024, pos % 1024 // 32, pos % 32])
        axis = torch.bucketize(freq * 64 // (D // 2), torch.tensor([16, 40], device=dev), right=True)
    else:
        positions, axis = pos[None], torch.zeros_like(freq)
    angle = torch.arange(ROPE_ROWS, device=dev, dtype=torch.float64)[:, None] * THETA ** (-2.0 * freq.double() / D)
    half = dict(generator=gen, device=dev)
    # K of real layers has a few channels far larger than the others
    loud = 1 + 7 * (torch.rand(Hkv * D, generator=gen, device=dev) < 0.03).float()
    s.update(q=torch.randn((T, H, D), **half).half(), positions=positions.int().contiguous(), axis=axis, slots=_slots(table, seq, pos, page),
             cos=angle.cos().float(), sin=angle.sin().float(), new_k=(torch.randn((T, Hkv, D), **half) * loud.view(Hkv, D)).half(),
             new_v=torch.randn((T, Hkv, D), **half).half(), axis_bytes=bytes(axis.tolist()))
    s["bias"] = [torch.randn(m * D, **half).half() for m in (H, Hkv, Hkv)] if case["bias"] else [None] * 3
    keep = case["fresh"]
    s["out"] = dict(q=torch.empty_like(s["q"]), k=torch.empty_like(s["new_k"]) if keep else None, v=torch.empty_like(s["new_v"]) if keep else None)
    if op == "append4":
        s["read"] = [torch.empty((T, Hkv, D), dtype=torch.float16, device=dev) for _ in range(2)]
    return s


# ----------------------------------------------------------------- operators
def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _own_cache(s):
    """The handle that a program keeps for the life of its cache."""
    from forgert_b200 import attention as A

    if "handle" not in s:
        s["handle"] = A.KV4Cache(s["k"], s["v"], s["scales"])
    return A, s["handle"]


def _own_append16(s):
    from forgert_b200 import attention as A

    o, c = s["out"], s["case"]
    A.qkv_rope_append_paged(s["q"], s["new_k"], s["new_v"], o["q"], o["k"], o["v"], s["cos"], s["sin"], s["positions"], s["slots"], s["k"], s["v"],
                            c["page"], s["pages"], len(s["q"]), c["H"], c["Hkv"], c["D"], ROPE_ROWS, *s["bias"], num_axes=c["axes"],
                            freq_axis=s["axis_bytes"])
    return dict(o, k_pages=s["k"], v_pages=s["v"])


def _own_append4(s):
    A, cache = _own_cache(s)
    o, c = s["out"], s["case"]
    A.qkv_rope_append_kv4(s["q"], s["new_k"], s["new_v"], o["q"], o["k"], o["v"], s["cos"], s["sin"], s["positions"], s["slots"], cache,
                          len(s["q"]), c["H"], ROPE_ROWS, *s["bias"], num_axes=c["axes"], freq_axis=s["axis_bytes"])
    A.kv4_gather(cache, s["slots"], *s["read"], len(s["slots"]))
    return dict(o, cached_k=s["read"][0], cached_v=s["read"][1])


def _own_gather(s):
    A, cache = _own_cache(s)
    A.kv4_gather(cache, s["slots"], s["k_out"], s["v_out"], len(s["slots"]))
    return s["k_out"], s["v_out"]


def _own_attention(s):
    A, cache = _own_cache(s)
    A.decode_attn_paged_kv4(s["q"], cache, s["table"], s["kv_lens"], s["out"], len(s["q"]), s["case"]["H"], s["table"].shape[1], s["longest"])
    return s["out"]


def _turned(s):
    """q, k and v in 32 bits, with their biases, q and k turned."""
    D = s["case"]["D"]
    at = s["positions"].long()[s["axis"]].t()                               # [T, D/2]
    f = torch.arange(D // 2, device=at.device)
    cos, sin = s["cos"][at, f][:, None], s["sin"][at, f][:, None]
    rows = [x.float() if b is None else x.float() + b.float().view(-1, D) for x, b in zip((s["q"], s["new_k"], s["new_v"]), s["bias"])]
    for i in range(2):
        a, b = rows[i].chunk(2, -1)
        rows[i] = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return rows


def _plain_append16(s):
    q, k, v = _turned(s)
    for pool, x in ((s["k"], k), (s["v"], v)):
        pool.flatten(0, 1)[s["slots"]] = x.half()
    keep = s["case"]["fresh"]
    return dict(q=q.half(), k=k.half() if keep else None, v=v.half() if keep else None, k_pages=s["k"], v_pages=s["v"])


def _values(codes, pairs):
    """Codes [..., D / 2] and their (scale, bias) [..., D / 64, 2] as numbers [..., D] in 32 bits."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    return (n * pairs[..., :1].float() + pairs[..., 1:].float()).flatten(-2)


def _plain_read(s, which, slots):
    page = s["case"]["page"]
    pg, row = slots // page, slots % page
    return _values((s["k"], s["v"])[which][pg, :, row], s["scales"][pg, :, row, which]).half()


def _plain_append4(s):
    q, k, v = _turned(s)
    page = s["case"]["page"]
    pg, row = s["slots"] // page, s["slots"] % page
    for which, (pool, x) in enumerate(((s["k"], k), (s["v"], v))):
        n, scale, bias = _code(x)
        pool[pg, :, row] = _bytes(n)
        s["scales"][pg, :, row, which] = torch.stack([scale, bias], -1).half()
    keep = s["case"]["fresh"]
    return dict(q=q.half(), k=k.half() if keep else None, v=v.half() if keep else None,
                cached_k=_plain_read(s, 0, s["slots"]), cached_v=_plain_read(s, 1, s["slots"]))


def _plain_gather(s):
    return _plain_read(s, 0, s["slots"]), _plain_read(s, 1, s["slots"])


def _plain_attention(s):
    c = s["case"]
    n, H, Hkv, D, page = len(s["q"]), c["H"], c["Hkv"], c["D"], c["page"]
    wide = s["table"].shape[1] * page
    some = max(1, 2 ** 28 // (wide * Hkv * D))          # sequences at a time
    found = []
    for b in range(0, n, some):
        table, lens = s["table"][b:b + some].long().clamp(min=0), s["kv_lens"][b:b + some]
        real = torch.arange(wide, device=table.device) < lens[:, None]                              # [n, L]

        def rows(pool, which):
            x = _values(pool[table], s["scales"][table][..., which, :, :])                          # [n, pages, Hkv, page, D]
            return x.transpose(1, 2).reshape(len(table), Hkv, wide, D).masked_fill_(~real[:, None, :, None], 0.0)

        q = s["q"][b:b + some].float().view(-1, Hkv, H // Hkv, D)
        score = (q @ rows(s["k"], 0).transpose(2, 3)) / math.sqrt(D)
        score = score.masked_fill(~real[:, None, None], -math.inf)
        top = score.amax(-1, keepdim=True)
        p = (score - torch.where(top == -math.inf, 0.0, top)).exp()
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total > 0, total, 1.0)                          # a request that holds nothing answers zeros
        found.append((p @ rows(s["v"], 1)).view(-1, H, D).half())
    return torch.cat(found)


_own = dict(append16=_own_append16, append4=_own_append4, gather=_own_gather, attention=_own_attention)
_plain = dict(append16=_plain_append16, append4=_plain_append4, gather=_plain_gather, attention=_plain_attention)


# ------------------------------------------------------------------ 64 bits
def _exact_values(raw, pairs):
    """The numbers that bytes [..., D / 2] stand for, by a table of the 256 bytes."""
    both = torch.tensor([[i % 16, i // 16] for i in range(256)], dtype=torch.float64, device=raw.device)
    n = both[raw.long()].reshape(*raw.shape[:-1], -1)
    pairs = pairs.double().repeat_interleave(GROUP, -2)
    return n * pairs[..., 0] + pairs[..., 1]


def exact(case, seed):
    s = prepare(case, seed)
    op, page, Hkv, D = case["op"], case["page"], case["Hkv"], case["D"]
    pools = (s["k"], s["v"])
    if op == "gather":
        pg, row = torch.div(s["slots"], page, rounding_mode="floor"), torch.remainder(s["slots"], page)
        return tuple(_exact_values(pool[pg, :, row], s["scales"][pg, :, row, which]) for which, pool in enumerate(pools))
    if op == "attention":
        out = torch.zeros((len(s["q"]), case["H"], D), dtype=torch.float64, device=s["q"].device)
        group = case["H"] // Hkv
        for b, n in enumerate(_lens(case)):
            if not n:
                continue
            pg = s["table"][b, :_up(n, page)].long()
            k, v = (_exact_values(pool[pg].transpose(0, 1).reshape(Hkv, -1, D // 2)[:, :n],
                                  s["scales"][pg][:, :, :, which].transpose(0, 1).reshape(Hkv, -1, D // GROUP, 2)[:, :n])
                    for which, pool in enumerate(pools))
            for j in range(Hkv):
                q = s["q"][b, j * group:(j + 1) * group].double()
                out[b, j * group:(j + 1) * group] = torch.softmax(q @ k[j].t() * D ** -0.5, -1) @ v[j]
        return out
    # appends: the rotation by complex numbers
    turn = torch.complex(s["cos"].double(), s["sin"].double())
    at = torch.stack([turn[s["positions"][a].long(), f] for f, a in enumerate(s["axis"].tolist())], 1)[:, None]
    rows = []
    for x, b in zip((s["q"], s["new_k"], s["new_v"]), s["bias"]):
        x = x.double()
        rows.append(x if b is None else x + b.double().view(1, -1, D))
    for i in range(2):
        z = torch.complex(rows[i][..., :D // 2], rows[i][..., D // 2:]) * at
        rows[i] = torch.cat([z.real, z.imag], -1)
    keep = case["fresh"]
    found = dict(q=rows[0], k=rows[1] if keep else None, v=rows[2] if keep else None)
    if op == "append16":
        for name, pool, x in (("k_pages", pools[0], rows[1]), ("v_pages", pools[1], rows[2])):
            pages = pool.double()
            pages.view(-1, Hkv, D).index_copy_(0, s["slots"], x)
            found[name] = pages
        return found
    for name, x in (("cached_k", rows[1]), ("cached_v", rows[2])):
        parts = []
        for g in range(0, D, GROUP):
            y = x[..., g:g + GROUP]
            low, high = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
            bias = low.half().double()                       # to the nearest, then down where that went up
            ulp = torch.exp2((torch.floor(torch.log2(low.abs().clamp(min=2.0 ** -14))) - 10))
            down = torch.where(low >= 0, torch.floor(low / ulp), -torch.ceil(-low / ulp)) * ulp
            bias = torch.where(bias > low, down, bias)
            want = (high - bias) / 15
            scale = want.half().double()
            ulp = torch.exp2((torch.floor(torch.log2(want.clamp(min=2.0 ** -14))) - 10))
            scale = torch.where(scale < want, torch.ceil(want / ulp) * ulp, scale)
            n = torch.where(scale > 0, torch.round((y - bias) / torch.where(scale > 0, scale, 1.0)), 0.0)
            parts.append(n * scale + bias)
        found[name] = torch.cat(parts, -1)
    return found
