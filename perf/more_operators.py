"""Rotary positions of several axes and a paged key-value cache of 8 and 4 bits, as cases that can be timed and compared.

One case is one pass as a decoder's step or its prompt makes it: queries and keys turned by their positions, new
tokens' keys and values quantised into the cache's pages and read back, a sequence's pages read back, and one new
token's attention over the packed pages.  Sizes are those of this repository's benchmark (32 heads of 128) and generic
ones around them.

  listed()           the named cases
  draw(rng)          one more case of the same ranges
  prepare(c, seed)   inputs on the GPU, made from the seed, and the views and events a program keeps
  run(state)         one pass; returns every output it writes, packed values as what they stand for
  work(c)            bytes and operations that the pass cannot do without
  exact(c, seed)     the same outputs in 64 bits, from the definitions

`own` selects what run() calls: the library's operators, or their plain form in torch.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

# bytes of a block of 32 values: an f16 scale d, and 32 signed bytes q (d q), or 16 bytes of two nibbles q (d (q - 8))
BLOCK = {"q8_0": 34, "q4_0": 18}
NIBBLES = [0, 2, 4, 6, 1, 3, 5, 7]  # which of eight values each nibble holds, lowest bits first


def listed():
    return [
        # One new token, a long way into a document: the smallest call, where latency counts.
        {"name": "rotate_one", "kind": "rotate", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "sections": "16 24 24", "base": 1e6, "far": 200000,
         "adjacent": False, "in_turn": False, "own_frequencies": False, "factors": False, "backward": False},
        # A long prompt of text and images, positions by time, height and width.
        {"name": "rotate_prompt", "kind": "rotate", "tokens": 8001, "heads": 32, "kv_heads": 8, "dim": 128, "sections": "24 20 20", "base": 5e6, "far": 4000,
         "adjacent": False, "in_turn": True, "own_frequencies": False, "factors": False, "backward": False},
        # An image encoder's patches, by height and width, each with the whole range of frequencies.
        {"name": "rotate_patches", "kind": "rotate", "tokens": 73 * 73, "heads": 16, "kv_heads": 16, "dim": 80, "sections": "20 20", "base": 1e4, "far": 0,
         "adjacent": False, "in_turn": False, "own_frequencies": True, "factors": False, "backward": False},
        # The gradient of a video's tokens, three quarters of each head turned, neighbours in pairs, stretched frequencies.
        {"name": "rotate_back", "kind": "rotate", "tokens": 4097, "heads": 16, "kv_heads": 2, "dim": 128, "sections": "16 16 16", "base": 1e4, "far": 60000,
         "adjacent": True, "in_turn": False, "own_frequencies": False, "factors": True, "backward": True},
        # The step's new keys and values of a batch, some slots of it idle.
        {"name": "write_step", "kind": "write", "k_type": "q4_0", "v_type": "q4_0", "tokens": 64, "kv_heads": 8, "dim": 128, "page": 16, "pages": 4096, "order": "token"},
        # A long prompt's, keys in more bits than values.
        {"name": "write_prompt", "kind": "write", "k_type": "q8_0", "v_type": "q4_0", "tokens": 8001, "kv_heads": 8, "dim": 128, "page": 64, "pages": 512, "order": "head"},
        # One conversation's cache, as it is taken over into another one.
        {"name": "read_chat", "kind": "read", "k_type": "q4_0", "v_type": "q4_0", "tokens": 500, "kv_heads": 2, "dim": 64, "page": 16, "pages": 4096, "order": "token"},
        # A long document's.
        {"name": "read_long", "kind": "read", "k_type": "q8_0", "v_type": "q8_0", "tokens": 40001, "kv_heads": 8, "dim": 128, "page": 64, "pages": 1024, "order": "head"},
        # One sequence, a few thousand tokens in: few rows, so the cache's length is what can be shared out.
        {"name": "attend_one", "kind": "attend", "k_type": "q4_0", "v_type": "q4_0", "heads": 32, "kv_heads": 8, "dim": 128, "seqs": 1, "low": 4001, "high": 4001,
         "page": 16, "order": "token", "window": 0, "cap": 0.0},
        # A batch of sequences of very different lengths.
        {"name": "attend_batch", "kind": "attend", "k_type": "q4_0", "v_type": "q4_0", "heads": 32, "kv_heads": 8, "dim": 128, "seqs": 64, "low": 90, "high": 9000,
         "page": 16, "order": "token", "window": 0, "cap": 0.0},
        # Two sequences over a long document, every head with keys of its own.
        {"name": "attend_long", "kind": "attend", "k_type": "q8_0", "v_type": "q8_0", "heads": 32, "kv_heads": 32, "dim": 128, "seqs": 2, "low": 40001, "high": 60001,
         "page": 64, "order": "head", "window": 0, "cap": 0.0},
        # Wide heads, a sliding window and capped scores, keys in more bits than values.
        {"name": "attend_window", "kind": "attend", "k_type": "q8_0", "v_type": "q4_0", "heads": 16, "kv_heads": 2, "dim": 256, "seqs": 17, "low": 500, "high": 20000,
         "page": 32, "order": "head", "window": 1024, "cap": 50.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotate", "write", "read", "attend", "attend"])
    types = {"k_type": rng.choice(["q8_0", "q4_0"]), "v_type": rng.choice(["q8_0", "q4_0"])}
    if kind == "rotate":
        dim, kv = rng.choice([64, 80, 96, 128, 192, 256]), rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 7])
        pairs = dim // 2 if rng.random() < 0.6 else rng.randint(8, dim // 2)
        axes = rng.choice([1, 2, 3, 3, 3, 4])
        cuts = sorted(rng.sample(range(1, pairs), axes - 1))
        return {"kind": kind, "tokens": min(_log(rng, 1, 16000), 40_000_000 // ((heads + kv) * dim)), "heads": heads, "kv_heads": kv, "dim": dim,
                "sections": " ".join(str(b - a) for a, b in zip([0] + cuts, cuts + [pairs])), "base": rng.choice([1e4, 5e5, 1e6]), "far": rng.choice([0, _log(rng, 1, 1000000)]),
                "adjacent": rng.random() < 0.4, "in_turn": rng.random() < 0.4, "own_frequencies": rng.random() < 0.3, "factors": rng.random() < 0.3,
                "backward": rng.random() < 0.3}
    if kind in ("write", "read"):
        return {"kind": kind, **types, "tokens": _log(rng, 1, 8000 if kind == "write" else 16000), "kv_heads": rng.choice([1, 2, 4, 8]), "dim": rng.choice([64, 96, 128, 256]),
                "page": rng.choice([8, 16, 24, 64]), "pages": rng.randint(2100, 2400), "order": rng.choice(["token", "head"])}
    kv = rng.choice([1, 2, 4, 8, 16])
    heads = kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    dim, seqs = rng.choice([64, 96, 128, 160, 192, 256]), _log(rng, 1, 128)
    high = min(_log(rng, 1, 60000), max(1, 180_000_000 // (kv * dim * seqs)), max(1, 60_000_000 // (heads * seqs)))
    return {"kind": kind, **types, "heads": heads, "kv_heads": kv, "dim": dim, "seqs": seqs, "low": min(high, _log(rng, 1, 4000)), "high": high,
            "page": rng.choice([1, 8, 16, 24, 64, 256]), "order": rng.choice(["token", "head"]), "window": rng.choice([0, 0, 0, _log(rng, 1, 8192)]),
            "cap": rng.choice([0.0, 0.0, 30.0])}


# ---- inputs -------------------------------------------------------------------------------


def _sections(c):
    """Pairs of each axis."""
    return [int(n) for n in c["sections"].split()]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, scale=1.0):
    return torch.empty(*shape, device="cuda").normal_(0.0, scale, generator=g)


def _grid(t, rows, cols):
    """The positions [3, rows * cols] of a grid of patches at time t: time, height, width."""
    y, x = torch.arange(rows).repeat_interleave(cols), torch.arange(cols).repeat(rows)
    return torch.stack([torch.full_like(x, t), t + y, t + x])


def _positions(c, g):
    """I32 [axes, tokens]: one axis counts tokens; two are an image's rows and columns; more mix runs of text, where all
    axes count alike, with images, which stand still in time."""
    axes, n = len(_sections(c)), c["tokens"]
    rest = torch.randint(0, 2**31 - 1, (64,), device="cuda", generator=g).tolist()
    at = rest[0] % (c["far"] + 1)
    if axes == 1:
        p = (at + torch.arange(n))[None]
    elif axes == 2:
        side = max(1, math.isqrt(n))
        p = _grid(0, -(-n // side), side)[1:] + at
    else:
        parts, have = [], 0
        for i in range(1, 64, 3):
            text, rows, cols = 1 + rest[i] % 700, 1 + rest[i + 1] % 40, 1 + rest[i + 2] % 40
            parts += [(at + torch.arange(text)).expand(3, -1), _grid(at + text, rows, cols)]
            at, have = at + text + max(rows, cols), have + text + rows * cols
        while have < n:
            parts.append((at + torch.arange(1024)).expand(3, -1))
            at, have = at + 1024, have + 1024
        p = torch.cat(parts, 1)
        p = torch.cat([p, p[:1]])[:axes]
    return p[:, :n].to(torch.int32).cuda().contiguous()


def _pool(c, kind, g=None):
    """A pool of packed pages, as bytes [pages, kv_heads, page, bytes of a token's head]; "token" order keeps a token's
    heads side by side in memory.  Quantised normal values where g is given."""
    row = c["dim"] // 32 * BLOCK[kind]
    shape = (c["pages"], c["kv_heads"], c["page"], row) if c["order"] == "head" else (c["pages"], c["page"], c["kv_heads"], row)
    t = torch.zeros(shape, dtype=torch.uint8, device="cuda")
    if g is not None:
        flat, step = t.view(-1, row), max(1, 50_000_000 // c["dim"])
        for i in range(0, flat.shape[0], step):
            part = flat[i:i + step]
            part.copy_(_encode(kind, _normal(g, part.shape[0], c["dim"])))
    return t if c["order"] == "head" else t.transpose(1, 2)


def _lengths(c):
    """Lengths spread evenly over the logarithm of the range."""
    n = c["seqs"]
    at = [0.5] if n == 1 else [i / (n - 1) for i in range(n)]
    return [int(round(c["low"] * (c["high"] / c["low"]) ** x)) for x in at]


def prepare(c, seed):
    g = _gen(seed)
    s = {"case": c}
    if c["kind"] == "rotate":
        s["q"], s["k"] = _normal(g, c["tokens"], c["heads"], c["dim"], scale=1.5), _normal(g, c["tokens"], c["kv_heads"], c["dim"])
        s["positions"] = _positions(c, g)
        if c["factors"]:  # high frequencies as they are, low ones up to 8 times slower
            pairs = sum(_sections(c))
            s["factors"] = 1.0 + 7.0 * (torch.arange(pairs, device="cuda") / pairs) ** 2 + 0.01 * torch.rand(pairs, device="cuda", generator=g)
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
    elif c["kind"] in ("write", "read"):
        fill = g if c["kind"] == "read" else None
        s["k_pages"], s["v_pages"] = _pool(c, c["k_type"], fill), _pool(c, c["v_type"], fill)
        shape = (c["tokens"], c["kv_heads"], c["dim"])
        s["k_out"], s["v_out"] = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
        if c["kind"] == "write":
            s["k"], s["v"] = _normal(g, *shape), _normal(g, *shape, scale=0.3)
            slots = torch.randperm(c["page"] * c["pages"], device="cuda", generator=g)[:c["tokens"]]
            s["slots"] = torch.where(torch.rand(c["tokens"], device="cuda", generator=g) < 0.05, -1, slots).to(torch.int32)
        else:  # a sequence's pages, in an order of their own
            at = torch.arange(c["tokens"], device="cuda")
            table = torch.randperm(c["pages"], device="cuda", generator=g)
            s["slots"] = (table[at // c["page"]] * c["page"] + at % c["page"]).to(torch.int32)
    else:
        lens = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")
        s["lengths"] = lens[torch.randperm(c["seqs"], device="cuda", generator=g)]
        per = -(-c["high"] // c["page"])
        sized = {**c, "pages": c["seqs"] * per}
        s["q"] = _normal(g, c["seqs"], c["heads"], c["dim"], scale=1.5)
        s["k_pages"], s["v_pages"] = _pool(sized, c["k_type"], g), _pool(sized, c["v_type"], g)
        s["table"] = torch.randperm(c["seqs"] * per, device="cuda", generator=g).to(torch.int32).view(c["seqs"], per)
        s["y"] = torch.empty(c["seqs"], c["heads"], c["dim"], device="cuda")
    return s


# ---- the library's operators -----------------------------------------------------------------


def _events(c, s):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "emel.rs_amd"))
    import emel_hip as eh

    def layout(t):
        kind = {torch.float32: eh.DType.F32, torch.int32: eh.DType.I32}[t.dtype]
        shape, strides = (1,) * (4 - t.dim()) + tuple(t.shape), [st * t.element_size() for st in t.stride()]
        strides = [strides[0] * t.shape[0]] * (4 - t.dim()) + strides
        return eh.Layout(kind, shape[::-1], strides[::-1])

    def view(t):
        return eh.TensorView(t, layout(t))

    def out(t):
        return eh.TensorViewMut(t, layout(t))

    def pages(t, kind, make):
        code = eh.DType.Q8_0 if kind == "q8_0" else eh.DType.Q4_0
        return make(t, eh.Layout(code, [c["dim"], t.shape[2], t.shape[1], t.shape[0]], [1, t.stride(2), t.stride(1), t.stride(0)]))

    kernel = eh.Kernel(stream=torch.cuda.current_stream().cuda_stream, synchronous=False)
    if c["kind"] == "rotate":
        event = eh.OpRope(view(s["q"]), out(s["q_out"]), view(s["positions"]), _sections(c), k=view(s["k"]), k_out=out(s["k_out"]),
                          factors=view(s["factors"]) if c["factors"] else None, base=c["base"], adjacent=c["adjacent"], in_turn=c["in_turn"],
                          own_frequencies=c["own_frequencies"], backward=c["backward"])
        return kernel, [event]
    if c["kind"] == "attend":
        return kernel, [eh.OpPagedAttention(view(s["q"]), pages(s["k_pages"], c["k_type"], eh.TensorView), pages(s["v_pages"], c["v_type"], eh.TensorView),
                                            view(s["table"]), view(s["lengths"]), out(s["y"]), scale=1.0 / math.sqrt(c["dim"]), window=c["window"],
                                            soft_cap=c["cap"])]
    read = eh.OpPagedKvRead(pages(s["k_pages"], c["k_type"], eh.TensorView), pages(s["v_pages"], c["v_type"], eh.TensorView), view(s["slots"]),
                            out(s["k_out"]), out(s["v_out"]))
    if c["kind"] == "read":
        return kernel, [read]
    return kernel, [eh.OpPagedKvAppend(view(s["k"]), view(s["v"]), view(s["slots"]), pages(s["k_pages"], c["k_type"], eh.TensorViewMut),
                                       pages(s["v_pages"], c["v_type"], eh.TensorViewMut)), read]


# ---- their plain form -------------------------------------------------------------------------


def _encode(kind, x):
    """Rows of f32 values as packed bytes.  Of a block's 32 values the scale is the largest magnitude / 127, or the value
    of the largest magnitude (the first of equal ones) / -8, rounded to f32 and then to f16; a value is the nearest
    whole number of scales, ties to even, within the format's range.  Numbers come first, by eights: the first eight
    of every block, then the second, the third and the fourth; the blocks' scales follow."""
    b = x.reshape(-1, 32)
    size = b.abs().amax(1)
    if kind == "q8_0":
        d = size.double() / torch.full_like(size, 127.0).double()
    else:
        d = b.gather(1, b.abs().eq(size[:, None]).to(torch.int8).argmax(1, keepdim=True))[:, 0] * -0.125
    d = d.float().clamp(-65504.0, 65504.0).half()
    n = torch.where(d[:, None] == 0, 0.0, torch.round(b.double() / d.double()[:, None]))  # 64 bits tell which side of a half a quotient is
    if kind == "q8_0":
        q = n.clamp(-127, 127).to(torch.int8).view(torch.uint8)
    else:  # of an eight: values 0, 2, 4, 6, then 1, 3, 5, 7, four bits each
        q = (n.clamp(-8, 7) + 8).to(torch.uint8).view(-1, 8)[:, NIBBLES]
        q = q[:, 0::2] | (q[:, 1::2] << 4)
    blocks = x.shape[-1] // 32
    rows = torch.cat([q.reshape(x.numel() // x.shape[-1], blocks, 4, -1).transpose(1, 2).flatten(1), d.view(-1, blocks).view(torch.uint8)], 1)
    return rows.view(*x.shape[:-1], -1)


def _decode(kind, b):
    """Packed rows as f32 values."""
    blocks = b.shape[-1] // BLOCK[kind]
    rows = b.reshape(-1, b.shape[-1])
    d, q = rows[:, -2 * blocks:].contiguous().view(torch.float16).float(), rows[:, :-2 * blocks]
    if kind == "q8_0":
        v = q.contiguous().view(torch.int8).float()
    else:
        q = q.reshape(-1, 4)
        v = torch.empty(q.shape[0], 8, device=b.device)
        v[:, NIBBLES] = torch.stack([q & 15, q >> 4], 2).flatten(1).float() - 8.0
    v = v.view(-1, 4, blocks, 8).transpose(1, 2).flatten(2)  # [rows, blocks, 32]
    return (v * d[:, :, None]).view(*b.shape[:-1], -1)


def _pairs(c):
    """Of each pair: its axis, its number and the count that its frequency's exponent is a quotient of."""
    left, axis = _sections(c), []
    if c["in_turn"]:
        while any(left):
            for a in range(len(left)):
                if left[a]:
                    axis.append(a)
                    left[a] -= 1
    else:
        axis = [a for a, n in enumerate(left) for _ in range(n)]
    if not c["own_frequencies"]:
        return axis, list(range(len(axis))), [len(axis)] * len(axis)
    return axis, [axis[:i].count(a) for i, a in enumerate(axis)], [_sections(c)[a] for a in axis]


def _rotated(c, s, x, cos, sin):
    """x [tokens, heads, dim] with its pairs turned by the angles of cos and sin [tokens, 1, pairs]."""
    n = cos.shape[-1]
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if c["adjacent"] else (slice(0, n), slice(n, 2 * n))
    a, b, y = x[..., first], x[..., second], x.clone()
    y[..., first], y[..., second] = a * cos - b * sin, a * sin + b * cos
    return y


def run(s):
    c = s["case"]
    if own:
        if "events" not in s:  # built once, as a program that serves tokens keeps them
            s["kernel"], s["events"] = _events(c, s)
        for event in s["events"]:
            status = s["kernel"].process_event(event)
            if status != 0:
                raise RuntimeError(status.name)
        return [s["q_out"], s["k_out"]] if c["kind"] == "rotate" else s["y"] if c["kind"] == "attend" else [s["k_out"], s["v_out"]]
    if c["kind"] == "rotate":
        axis, j, n = (torch.tensor(t, device="cuda") for t in _pairs(c))
        freq = torch.exp(j.double() / n * -math.log(c["base"]))
        if c["factors"]:
            freq = freq / s["factors"].double()
        angle = s["positions"].double()[axis].t()[:, None] * freq  # far positions lose their angle in 32 bits
        sin = torch.sin(angle).float()
        return [_rotated(c, s, x, torch.cos(angle).float(), -sin if c["backward"] else sin) for x in (s["q"], s["k"])]
    if c["kind"] == "write" or c["kind"] == "read":
        at = s["slots"].long()
        live = at >= 0
        page, tok = at[live] // c["page"], at[live] % c["page"]
        outs = []
        for new, pool, kind, dst in (("k", "k_pages", c["k_type"], "k_out"), ("v", "v_pages", c["v_type"], "v_out")):
            if c["kind"] == "write":
                s[pool][page, :, tok] = _encode(kind, s[new][live])
            s[dst][live] = _decode(kind, s[pool][page, :, tok])
            outs.append(s[dst])
        return outs
    k, v = (_decode(kind, s[pool][s["table"].long()].transpose(2, 3)) for pool, kind in (("k_pages", c["k_type"]), ("v_pages", c["v_type"])))
    k, v = (t.reshape(c["seqs"], -1, c["kv_heads"], c["dim"]) for t in (k, v))  # [seqs, positions, kv_heads, dim]
    q = s["q"].view(c["seqs"], c["kv_heads"], -1, c["dim"])
    score = (q @ k.permute(0, 2, 3, 1).contiguous()) * (1.0 / math.sqrt(c["dim"]))
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    at, n = torch.arange(k.shape[1], device="cuda"), s["lengths"][:, None, None, None]
    seen = (at < n) & (at >= n - c["window"] if c["window"] else at >= 0)
    score = torch.where(seen, score, -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    return ((e / e.sum(-1, keepdim=True)) @ v.transpose(1, 2).contiguous()).view(c["seqs"], c["heads"], c["dim"])


# ---- what a pass cannot do without, and its outputs in 64 bits ------------------------------------


def work(c):
    if c["kind"] == "rotate":
        n = c["tokens"] * (c["heads"] + c["kv_heads"])
        return {"bytes": 8 * n * c["dim"] + 4 * c["tokens"] * len(_sections(c)), "flops": 6 * n * sum(_sections(c))}
    packed = (BLOCK[c["k_type"]] + BLOCK[c["v_type"]]) / 32  # of a key's value and a value's
    if c["kind"] == "attend":
        t = sum(min(n, c["window"]) if c["window"] else n for n in _lengths(c))
        return {"bytes": int(t * c["kv_heads"] * c["dim"] * packed) + 8 * c["seqs"] * c["heads"] * c["dim"] + 4 * (t // c["page"] + c["seqs"]),
                "flops": 4 * t * c["heads"] * c["dim"]}
    n = c["tokens"] * c["kv_heads"] * c["dim"]
    return {"bytes": int(n * (packed + (16 if c["kind"] == "write" else 8))) + 4 * c["tokens"], "flops": 0}


def exact(c, seed):
    s = prepare(c, seed)

    def values(kind, rows):
        """Packed rows [..., bytes] in 64 bits, a value at a time."""
        b = rows.reshape(-1, rows.shape[-1]).to(torch.int32)
        blocks = rows.shape[-1] // BLOCK[kind]
        out = torch.empty(b.shape[0], 32 * blocks, dtype=torch.float64, device="cuda")
        for i in range(32 * blocks):
            j, eight, at = i // 32, i % 32 // 8, i % 8
            low = (32 if kind == "q8_0" else 16) * blocks + 2 * j
            d = (b[:, low] | (b[:, low + 1] << 8)).to(torch.int16).view(torch.float16).double()
            if kind == "q8_0":
                q = b[:, 8 * (eight * blocks + j) + at]
                out[:, i] = d * (q - 256 * (q // 128))
            else:  # even values in the first two bytes, odd ones in the last two
                q = b[:, 4 * (eight * blocks + j) + 2 * (at % 2) + at // 4]
                out[:, i] = d * ((q // 16 if at // 2 % 2 else q % 16) - 8)
        return out.view(*rows.shape[:-1], -1)

    def rounded(kind, x):
        """What f32 rows stand for once they are packed: whole numbers of the scale, nearest first."""
        b = x.reshape(-1, 32).double()
        out = torch.empty_like(b)
        if kind == "q8_0":
            low, high, d = -127, 127, b.abs().amax(1) / 127.0
        else:
            top, bottom = b.amax(1), b.amin(1)
            m = torch.where(top > -bottom, top, bottom)
            for i in torch.nonzero(top == -bottom)[:, 0].tolist():  # both signs: the first of them
                m[i] = next(v for v in b[i].tolist() if abs(v) == float(top[i]))
            low, high, d = -8, 7, m / -8.0
        d = d.float().half().double()
        for j in range(32):
            n = torch.where(d == 0, 0.0, b[:, j] / d)
            f = torch.floor(n)
            up = (n - f > 0.5) | ((n - f == 0.5) & (f % 2 == 1))
            out[:, j] = d * torch.clamp(f + up, low, high)
        return out.view_as(x)

    if c["kind"] == "rotate":
        axis, j, n = _pairs(c)
        outs = []
        for x in (s["q"].double(), s["k"].double()):
            y = x.clone()
            for i in range(len(axis)):
                p, r = (2 * i, 2 * i + 1) if c["adjacent"] else (i, i + len(axis))
                freq = c["base"] ** (-j[i] / n[i]) / (float(s["factors"][i].double()) if c["factors"] else 1.0)
                turn = s["positions"][axis[i]].double()[:, None] * freq * (-1.0 if c["backward"] else 1.0)
                y[..., p] = x[..., p] * torch.cos(turn) - x[..., r] * torch.sin(turn)
                y[..., r] = x[..., p] * torch.sin(turn) + x[..., r] * torch.cos(turn)
            outs.append(y)
        return outs
    if c["kind"] == "write":
        idle = s["slots"] < 0
        return [rounded(kind, s[x]).masked_fill(idle[:, None, None], 0.0) for kind, x in ((c["k_type"], "k"), (c["v_type"], "v"))]
    if c["kind"] == "read":
        at = s["slots"].long()
        return [values(kind, s[pool][at // c["page"], :, at % c["page"]]) for kind, pool in ((c["k_type"], "k_pages"), (c["v_type"], "v_pages"))]
    out = torch.zeros(c["seqs"], c["heads"], c["dim"], dtype=torch.float64, device="cuda")
    group = c["heads"] // c["kv_heads"]
    for i, n in enumerate(s["lengths"].tolist()):
        at = torch.arange(max(0, n - c["window"]) if c["window"] else 0, n, device="cuda")
        page = s["table"][i].long()[at // c["page"]]
        k, v = (values(kind, s[pool][page, :, at % c["page"]]) for kind, pool in ((c["k_type"], "k_pages"), (c["v_type"], "v_pages")))
        for h in range(c["kv_heads"]):
            z = s["q"][i, h * group:(h + 1) * group].double() @ k[:, h].t() / math.sqrt(c["dim"])
            if c["cap"]:
                z = c["cap"] * torch.tanh(z / c["cap"])
            out[i, h * group:(h + 1) * group] = torch.softmax(z, -1) @ v[:, h]
    return out
