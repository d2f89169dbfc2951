"""A served token's operators over packed weights and a paged cache, as cases that can be timed and compared.

One case is one pass through one operator, as a decoder's step calls it: products with 4-bit weights, the
new tokens' keys and values written into a paged cache, one new token's attention over that cache, and the
logits' penalties, biases and grammar mask ahead of the sampler.  Sizes are those of this repository's
benchmark (hidden 4096, MLP 11008, 32 heads of 128, 151936 logits) and generic ones around them.

  listed()           the named cases
  draw(rng)          one more case of the same ranges
  prepare(c, seed)   inputs on the GPU, made from the seed, and the views and events a program keeps
  run(state)         one pass; returns every output it writes
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

PAGE_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
# values and bytes of one block of each packed format
BLOCK = {"q4_0": (32, 18), "q4_k": (256, 144)}


def listed():
    return [
        # One token of one sequence through a square projection: the smallest product of a step, where latency counts.
        {"name": "project_one", "kind": "product", "format": "q4_0", "k": 4096, "m": 4096, "n": 1},
        # The same token through the MLP's second product, in the other format.
        {"name": "mlp_down_one", "kind": "product", "format": "q4_k", "k": 11008, "m": 4096, "n": 1},
        # The output head of three sequences served together.
        {"name": "head_few", "kind": "product", "format": "q4_k", "k": 4096, "m": 151936, "n": 3},
        # The MLP's first product for a batch of sequences, one of its slots empty.
        {"name": "mlp_up_batch", "kind": "product", "format": "q4_0", "k": 4096, "m": 11008, "n": 15},
        # The step's new keys and values of a batch, some slots of it idle.
        {"name": "append_step", "kind": "append", "type": "bf16", "tokens": 64, "kv_heads": 8, "dim": 128, "page": 16, "pages": 4096, "order": "token"},
        # A long prompt's keys and values.
        {"name": "append_prompt", "kind": "append", "type": "f16", "tokens": 8001, "kv_heads": 8, "dim": 128, "page": 64, "pages": 512, "order": "head"},
        # One sequence, a few thousand tokens in: few rows, so the cache's length is what can be shared out.
        {"name": "attend_one", "kind": "attend", "type": "f16", "heads": 32, "kv_heads": 8, "dim": 128, "seqs": 1, "low": 4001, "high": 4001,
         "page": 16, "order": "token", "window": 0, "cap": 0.0},
        # A batch of sequences of very different lengths.
        {"name": "attend_batch", "kind": "attend", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "seqs": 64, "low": 90, "high": 9000,
         "page": 16, "order": "token", "window": 0, "cap": 0.0},
        # Two sequences over a long document, every head with keys of its own.
        {"name": "attend_long", "kind": "attend", "type": "f16", "heads": 32, "kv_heads": 32, "dim": 128, "seqs": 2, "low": 40001, "high": 60001,
         "page": 64, "order": "head", "window": 0, "cap": 0.0},
        # Wide heads, a sliding window and capped scores.
        {"name": "attend_window", "kind": "attend", "type": "bf16", "heads": 16, "kv_heads": 2, "dim": 256, "seqs": 17, "low": 500, "high": 20000,
         "page": 32, "order": "head", "window": 1024, "cap": 50.0},
        # One sequence's logits: the penalties of its history and a few biases.
        {"name": "logits_one", "kind": "logits", "card": 151936, "rows": 1, "history": 700, "biases": 12, "mask": False},
        # A batch under a grammar.
        {"name": "logits_batch", "kind": "logits", "card": 151936, "rows": 64, "history": 2048, "biases": 64, "mask": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["product", "product", "attend", "attend", "append", "logits"])
    if kind == "product":
        form = rng.choice(["q4_0", "q4_k"])
        unit = BLOCK[form][0]
        k = unit * _log(rng, 512 // unit, 16384 // unit)
        m = min(_log(rng, 256, 151936), 620_000_000 // k)
        n = min(_log(rng, 1, 64), max(1, 1_800_000_000 // (k * m)))
        return {"kind": kind, "format": form, "k": k, "m": m, "n": n}
    if kind == "append":
        return {"kind": kind, "type": rng.choice(["f16", "bf16"]), "tokens": _log(rng, 1, 8000), "kv_heads": rng.choice([1, 2, 4, 8]),
                "dim": rng.choice([64, 80, 96, 128]), "page": rng.choice([8, 16, 24, 64]), "pages": rng.randint(1100, 1400), "order": rng.choice(["token", "head"])}
    if kind == "attend":
        kv = rng.choice([1, 2, 4, 8, 16])
        heads = kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
        dim, seqs = rng.choice([64, 80, 96, 128, 192, 256]), _log(rng, 1, 128)
        high = min(_log(rng, 1, 60000), max(1, 180_000_000 // (kv * dim * seqs)), max(1, 60_000_000 // (heads * seqs)))
        return {"kind": kind, "type": rng.choice(["f16", "bf16"]), "heads": heads, "kv_heads": kv, "dim": dim, "seqs": seqs,
                "low": min(high, _log(rng, 1, 4000)), "high": high, "page": rng.choice([1, 8, 16, 24, 64, 256]), "order": rng.choice(["token", "head"]),
                "window": rng.choice([0, 0, 0, _log(rng, 1, 8192)]), "cap": rng.choice([0.0, 0.0, 30.0])}
    return {"kind": kind, "card": _log(rng, 1000, 151936), "rows": _log(rng, 1, 64), "history": _log(rng, 1, 2048), "biases": rng.choice([0, _log(rng, 1, 64)]),
            "mask": rng.random() < 0.5}


# ---- inputs -------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, scale=1.0):
    return torch.empty(*shape, device="cuda").normal_(0.0, scale, generator=g)


def _scales(g, count, size):
    """f16 scales spread around `size`, as bytes [count, 2]."""
    return (size * torch.exp(_normal(g, count, scale=0.3))).half().view(torch.uint8).view(count, 2)


def _packed(c, g):
    """Packed rows of normal weights around 1/sqrt(k), as bytes [m, bytes of a row]."""
    values, size = BLOCK[c["format"]]
    blocks = c["m"] * c["k"] // values
    out = torch.empty(blocks, size, dtype=torch.uint8, device="cuda")
    low = torch.empty(blocks, values // 2, device="cuda").normal_(8.0, 2.7, generator=g).round_().clamp_(0, 15).to(torch.uint8)
    high = torch.empty(blocks, values // 2, device="cuda").normal_(8.0, 2.7, generator=g).round_().clamp_(0, 15).to(torch.uint8)
    out[:, size - values // 2:] = low | (high << 4)
    if c["format"] == "q4_0":
        out[:, :2] = _scales(g, blocks, 0.37 / math.sqrt(c["k"]))
    else:  # six-bit scales and minima around 32, so that a value is near 32 d (q - 8)
        out[:, :2] = _scales(g, blocks, 0.0116 / math.sqrt(c["k"]))
        out[:, 2:4] = _scales(g, blocks, 8 * 0.0116 / math.sqrt(c["k"]))
        out[:, 4:16] = torch.randint(0, 256, (blocks, 12), dtype=torch.uint8, device="cuda", generator=g)
    return out.view(c["m"], -1)


def _lengths(c, g):
    """Lengths spread evenly over the logarithm of the range, in an order of the seed's."""
    n = c["seqs"]
    at = [0.5] if n == 1 else [i / (n - 1) for i in range(n)]
    lens = [int(round(c["low"] * (c["high"] / c["low"]) ** x)) for x in at]
    return torch.tensor(lens, dtype=torch.int32, device="cuda")[torch.randperm(n, device="cuda", generator=g)]


def _pages(c, count, g=None):
    """A pool of pages [pages, kv_heads, page, dim]; "token" order keeps a token's heads side by side in memory."""
    shape = (count, c["kv_heads"], c["page"], c["dim"]) if c["order"] == "head" else (count, c["page"], c["kv_heads"], c["dim"])
    t = torch.zeros(shape, dtype=PAGE_TYPES[c["type"]], device="cuda") if g is None else _normal(g, *shape).to(PAGE_TYPES[c["type"]])
    return t if c["order"] == "head" else t.transpose(1, 2)


def prepare(c, seed):
    g = _gen(seed)
    s = {"case": c}
    if c["kind"] == "product":
        s["w"], s["x"] = _packed(c, g), _normal(g, c["n"], c["k"])
        s["y"] = torch.empty(c["n"], c["m"], device="cuda")
    elif c["kind"] == "append":
        shape = (c["tokens"], c["kv_heads"], c["dim"])
        s["k"], s["v"] = _normal(g, *shape), _normal(g, *shape)
        s["k_pages"], s["v_pages"] = _pages(c, c["pages"]), _pages(c, c["pages"])
        slots = torch.randperm(c["page"] * c["pages"], device="cuda", generator=g)[:c["tokens"]].to(torch.int32)
        s["slots"] = torch.where(torch.rand(c["tokens"], device="cuda", generator=g) < 0.05, -1, slots).to(torch.int32)
    elif c["kind"] == "attend":
        s["lengths"] = _lengths(c, g)
        per = -(-c["high"] // c["page"])
        count = c["seqs"] * per
        s["q"] = _normal(g, c["seqs"], c["heads"], c["dim"], scale=1.5)
        s["k_pages"], s["v_pages"] = _pages(c, count, g), _pages(c, count, g)
        s["table"] = torch.randperm(count, device="cuda", generator=g).to(torch.int32).view(c["seqs"], per)
        s["y"] = torch.empty(c["seqs"], c["heads"], c["dim"], device="cuda")
    else:
        rows, card = c["rows"], c["card"]
        s["logits"] = _normal(g, rows, card, scale=3.0)
        # text repeats itself: ids thin out towards the end of the vocabulary
        s["history"] = (card * torch.rand(rows, c["history"], device="cuda", generator=g) ** 4).to(torch.int32).clamp_(max=card - 1)
        s["used"] = torch.randint(c["history"] // 2, c["history"] + 1, (rows,), device="cuda", generator=g).to(torch.int32)
        s["repeat"] = torch.empty(rows, device="cuda").uniform_(1.0, 1.3, generator=g)
        s["frequency"] = torch.empty(rows, device="cuda").uniform_(0.0, 0.5, generator=g)
        s["presence"] = torch.empty(rows, device="cuda").uniform_(0.0, 0.5, generator=g)
        if c["biases"]:
            ids = torch.rand(rows, card, device="cuda", generator=g).topk(min(c["biases"], card)).indices
            s["bias_ids"], s["bias"] = ids.to(torch.int32), _normal(g, *ids.shape, scale=4.0)
        if c["mask"]:  # one bit a token, an eighth of them allowed
            words = (rows, -(-card // 32))
            s["allowed"] = _words(g, words) & _words(g, words) & _words(g, words)
        s["y"] = torch.empty(rows, card, device="cuda")
    return s


def _words(g, shape):
    return torch.randint(-2**31, 2**31, shape, device="cuda", generator=g).to(torch.int32)


# ---- the library's operators -----------------------------------------------------------------


def _event(c, s):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "emel.rs_amd"))
    import emel_hip as eh

    def layout(t):
        kind = {torch.float32: eh.DType.F32, torch.int32: eh.DType.I32, torch.float16: eh.DType.F16, torch.bfloat16: eh.DType.BF16}[t.dtype]
        shape, strides = (1,) * (4 - t.dim()) + tuple(t.shape), [st * t.element_size() for st in t.stride()]
        strides = [strides[0] * t.shape[0]] * (4 - t.dim()) + strides
        return eh.Layout(kind, shape[::-1], strides[::-1])

    def view(t):
        return eh.TensorView(t, layout(t))

    def out(t):
        return eh.TensorViewMut(t, layout(t))

    kernel = eh.Kernel(stream=torch.cuda.current_stream().cuda_stream, synchronous=False)
    if c["kind"] == "product":
        code, event = (eh.DType.Q4_0, eh.OpMulMatQ4_0) if c["format"] == "q4_0" else (eh.DType.Q4_K, eh.OpMulMatQ4K)
        return kernel, event(eh.TensorView(s["w"], eh.Layout.packed(code, [c["k"], c["m"], 1, 1])), view(s["x"]), out(s["y"]))
    if c["kind"] == "append":
        return kernel, eh.OpPagedKvAppend(view(s["k"]), view(s["v"]), view(s["slots"]), out(s["k_pages"]), out(s["v_pages"]))
    if c["kind"] == "attend":
        return kernel, eh.OpPagedAttention(view(s["q"]), view(s["k_pages"]), view(s["v_pages"]), view(s["table"]), view(s["lengths"]), out(s["y"]),
                                           scale=1.0 / math.sqrt(c["dim"]), window=c["window"], soft_cap=c["cap"])
    more = {"bias_ids": view(s["bias_ids"]), "bias": view(s["bias"])} if c["biases"] else {}
    if c["mask"]:
        more["allowed"] = view(s["allowed"])
    return kernel, eh.OpLogitsAdjust(view(s["logits"]), out(s["y"]), history=view(s["history"]), history_len=view(s["used"]), repeat=view(s["repeat"]),
                                     frequency=view(s["frequency"]), presence=view(s["presence"]), **more)


# ---- their plain form -------------------------------------------------------------------------


def _half(pair):
    return pair.contiguous().view(torch.float16).float()


def _weights(c, w):
    """The f32 values [m, k] of packed rows."""
    values, size = BLOCK[c["format"]]
    b = w.view(-1, size)
    q = b[:, size - values // 2:]
    d = _half(b[:, :2])
    if c["format"] == "q4_0":  # a block's low nibbles are its first 16 values
        q = torch.cat([q & 15, q >> 4], 1).float()
        return ((q - 8.0) * d).view(c["m"], c["k"])
    q = q.view(-1, 4, 32)  # 64 values a quarter: low nibbles, then high
    q = torch.stack([q & 15, q >> 4], 2).view(-1, 8, 32).float()
    a, n, e = b[:, 4:8], b[:, 8:12], b[:, 12:16]
    sc = torch.cat([a & 63, (e & 15) | (a >> 6 << 4)], 1).float()
    mn = torch.cat([n & 63, (e >> 4) | (n >> 6 << 4)], 1).float()
    return (q * (d * sc)[:, :, None] - (_half(b[:, 2:4]) * mn)[:, :, None]).view(c["m"], c["k"])


def _cached(pages, table, page):
    """Every position's vectors [seqs, positions, kv_heads, dim] in f32."""
    rows = pages[table.long()].transpose(2, 3)
    return rows.reshape(table.shape[0], table.shape[1] * page, rows.shape[3], rows.shape[4]).float()


def run(s):
    c = s["case"]
    if own:
        if "event" not in s:  # built once, as a program that serves tokens keeps it
            s["kernel"], s["event"] = _event(c, s)
        status = s["kernel"].process_event(s["event"])
        if status != 0:
            raise RuntimeError(status.name)
        return [s["k_pages"], s["v_pages"]] if c["kind"] == "append" else s["y"]
    if c["kind"] == "product":
        return s["x"] @ _weights(c, s["w"]).t()
    if c["kind"] == "append":
        at = s["slots"].long()
        keep = at >= 0
        at, page = at[keep], c["page"]
        s["k_pages"][at // page, :, at % page] = s["k"][keep].to(s["k_pages"].dtype)
        s["v_pages"][at // page, :, at % page] = s["v"][keep].to(s["v_pages"].dtype)
        return [s["k_pages"], s["v_pages"]]
    if c["kind"] == "attend":
        k, v = _cached(s["k_pages"], s["table"], c["page"]), _cached(s["v_pages"], s["table"], c["page"])
        q = s["q"].view(c["seqs"], c["kv_heads"], -1, c["dim"])
        score = (q @ k.permute(0, 2, 3, 1).contiguous()) * (1.0 / math.sqrt(c["dim"]))
        if c["cap"]:
            score = c["cap"] * torch.tanh(score / c["cap"])
        at, n = torch.arange(k.shape[1], device="cuda"), s["lengths"][:, None, None, None]
        seen = (at < n) & (at >= n - c["window"] if c["window"] else at >= 0)
        score = torch.where(seen, score, -math.inf)
        e = torch.exp(score - score.amax(-1, keepdim=True))
        return ((e / e.sum(-1, keepdim=True)) @ v.transpose(1, 2).contiguous()).view(c["seqs"], c["heads"], c["dim"])
    l, rows = s["logits"], torch.arange(c["rows"], device="cuda")[:, None]
    used = torch.arange(c["history"], device="cuda") < s["used"][:, None]
    count = torch.zeros_like(l).index_put_((rows, s["history"].long()), used.float(), accumulate=True)
    pen = torch.where(l > 0, l / s["repeat"][:, None], l * s["repeat"][:, None]) - count * s["frequency"][:, None] - s["presence"][:, None]
    l = torch.where(count > 0, pen, l)
    if c["biases"]:
        l[rows, s["bias_ids"].long()] += s["bias"]
    if c["mask"]:
        at = torch.arange(c["card"], device="cuda")
        l = torch.where((s["allowed"][:, at >> 5] >> (at & 31)) & 1 == 1, l, -math.inf)
    return l


# ---- what a pass cannot do without, and its outputs in 64 bits ------------------------------------


def _tokens(c):
    n = c["seqs"]
    at = [0.5] if n == 1 else [i / (n - 1) for i in range(n)]
    lens = [int(round(c["low"] * (c["high"] / c["low"]) ** x)) for x in at]
    return sum(min(x, c["window"]) if c["window"] else x for x in lens)


def work(c):
    if c["kind"] == "product":
        k, m, n = c["k"], c["m"], c["n"]
        values, size = BLOCK[c["format"]]
        return {"bytes": m * k // values * size + 4 * n * (k + m), "flops": 2 * m * k * n}
    if c["kind"] == "append":
        return {"bytes": 2 * c["tokens"] * c["kv_heads"] * c["dim"] * (4 + 2) + 4 * c["tokens"], "flops": 0}
    if c["kind"] == "attend":
        t = _tokens(c)
        return {"bytes": 2 * t * c["kv_heads"] * c["dim"] * 2 + 8 * c["seqs"] * c["heads"] * c["dim"] + 4 * (t // c["page"] + c["seqs"]),
                "flops": 4 * t * c["heads"] * c["dim"]}
    cells = c["rows"] * c["card"]
    return {"bytes": 8 * cells + (cells // 8 if c["mask"] else 0) + 4 * c["rows"] * (c["history"] + 2 * c["biases"]), "flops": 0}


def exact(c, seed):
    s = prepare(c, seed)

    def product():
        values, size = BLOCK[c["format"]]
        x = s["x"].double()
        out = torch.empty(c["n"], c["m"], dtype=torch.float64, device="cuda")
        step = max(1, 100_000_000 // c["k"])
        for r in range(0, c["m"], step):
            b = s["w"][r:r + step].reshape(-1, size).to(torch.int32)
            half = lambda i: (b[:, i] | (b[:, i + 1] << 8)).to(torch.int16).view(torch.float16).double()  # noqa: E731
            w = torch.empty(b.shape[0], values, dtype=torch.float64, device="cuda")
            if c["format"] == "q4_0":
                for j in range(16):
                    w[:, j] = half(0) * ((b[:, 2 + j] % 16) - 8)
                    w[:, 16 + j] = half(0) * ((b[:, 2 + j] // 16) - 8)
            else:
                for j in range(8):
                    if j < 4:
                        sc, mn = b[:, 4 + j] % 64, b[:, 8 + j] % 64
                    else:
                        sc, mn = b[:, 8 + j] % 16 + 16 * (b[:, j] // 64), b[:, 8 + j] // 16 + 16 * (b[:, 4 + j] // 64)
                    q = b[:, 16 + 32 * (j // 2):48 + 32 * (j // 2)]
                    q = q // 16 if j % 2 else q % 16
                    w[:, 32 * j:32 * j + 32] = (half(0) * sc)[:, None] * q - (half(2) * mn)[:, None]
            out[:, r:r + step] = x @ w.view(-1, c["k"]).t()
        return out

    def attend():
        out = torch.zeros(c["seqs"], c["heads"], c["dim"], dtype=torch.float64, device="cuda")
        group = c["heads"] // c["kv_heads"]
        for i, n in enumerate(s["lengths"].tolist()):
            first = max(0, n - c["window"]) if c["window"] else 0
            at = torch.arange(first, n, device="cuda")
            page = s["table"][i].long()[at // c["page"]]
            k, v = s["k_pages"][page, :, at % c["page"]].double(), s["v_pages"][page, :, at % c["page"]].double()  # [positions, kv_heads, dim]
            for h in range(c["kv_heads"]):
                z = s["q"][i, h * group:(h + 1) * group].double() @ k[:, h].t() / math.sqrt(c["dim"])
                if c["cap"]:
                    z = c["cap"] * torch.tanh(z / c["cap"])
                out[i, h * group:(h + 1) * group] = torch.softmax(z, -1) @ v[:, h]
        return out

    if c["kind"] == "product":
        return product()
    if c["kind"] == "append":
        pair = []
        for new, pages in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
            pool = torch.zeros(pages.shape[0] * c["page"], c["kv_heads"], c["dim"], dtype=torch.float64, device="cuda")
            live = s["slots"] >= 0
            pool[s["slots"][live].long()] = new[live].double()
            pair.append(pool.view(-1, c["page"], c["kv_heads"], c["dim"]).transpose(1, 2))
        return pair
    if c["kind"] == "attend":
        return attend()
    out = s["logits"].double()
    for r in range(c["rows"]):
        ids, count = s["history"][r, :int(s["used"][r])].long().unique(return_counts=True)
        v = out[r, ids]
        v = torch.where(v > 0, v / s["repeat"][r].double(), v * s["repeat"][r].double())
        out[r, ids] = v - count * s["frequency"][r].double() - s["presence"][r].double()
        if c["biases"]:
            out[r, s["bias_ids"][r].long()] += s["bias"][r].double()
        if c["mask"]:
            bits = (s["allowed"][r].long()[:, None] >> torch.arange(32, device="cuda")) & 1
            out[r, bits.view(-1)[:c["card"]] == 0] = -math.inf
    return out
