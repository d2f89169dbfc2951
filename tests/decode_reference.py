"""The served-token operators from their formulas, in 64 bits with numpy, each with the size of the terms that it
sums (what a rounding error is relative to); and the packed rows, pools and views that their tests share."""
from __future__ import annotations

import numpy as np

import emel_hip as eh
from helpers import rng

BLOCK = {"q4_0": (32, 18), "q4_k": (256, 144)}


def packed_rows(seed, form, k, m):
    """m random packed rows of k values, as bytes [m, row bytes]: every nibble, six-bit scale and minimum occurs."""
    values, size = BLOCK[form]
    g = rng(seed)
    b = g.integers(0, 256, (m * k // values, size), dtype=np.uint8)
    for at in (0, 2)[: 1 if form == "q4_0" else 2]:
        d = (g.standard_normal(b.shape[0]) * 0.02).astype(np.float16)
        b[:, at:at + 2] = d.view(np.uint8).reshape(-1, 2)
    return b.reshape(m, -1)


def weight_terms(form, rows):
    """(scaled nibbles, what is subtracted from them) of packed rows, each [m, k] in f64."""
    values, size = BLOCK[form]
    m = rows.shape[0]
    b = rows.reshape(-1, size)
    half = lambda i: np.ascontiguousarray(b[:, i:i + 2]).view(np.float16).astype(np.float64)  # noqa: E731
    if form == "q4_0":
        q = np.concatenate([b[:, 2:] & 15, b[:, 2:] >> 4], 1)
        with np.errstate(invalid="ignore"):  # an infinite scale times 8 - 8
            return (half(0) * (q - 8.0)).reshape(m, -1), np.zeros((m, rows.size // m // size * values))
    hi, lo = np.zeros((b.shape[0], 256)), np.zeros((b.shape[0], 256))
    for j in range(8):
        s = b[:, 4:16].astype(np.int64)
        sc, mn = (s[:, j] & 63, s[:, j + 4] & 63) if j < 4 else ((s[:, j + 4] & 15) + 16 * (s[:, j - 4] >> 6), (s[:, j + 4] >> 4) + 16 * (s[:, j] >> 6))
        q = b[:, 16 + 32 * (j // 2):48 + 32 * (j // 2)]
        hi[:, 32 * j:32 * j + 32] = half(0) * sc[:, None] * (q >> 4 if j % 2 else q & 15)
        lo[:, 32 * j:32 * j + 32] = half(2) * mn[:, None]
    return hi.reshape(m, -1), lo.reshape(m, -1)


def product(form, rows, x):
    """(y [n, m], its tolerance) for x [n, k] f32.

    x is taken as hi + lo halves of 11 bits each, an error of 2^-23 of the value, or of 2^-39 of the column's
    largest value where lo is subnormal; products of a half and a nibble are exact; sums of up to k / 32 + 128 f32
    terms in a row (a block's in the matrix unit, then blocks, then waves), each off by at most 2^-23 of the sum of
    magnitudes so far.  As digits, x is off by 2^-30 of the largest of its 256 instead, T: sum |w| T 2^-30 is within the
    first term where T is below 2^14 times the run's mean weighted size, as in a run of 256 normal values (T about 3) or
    of those with one 1000 times as large."""
    hi, lo = weight_terms(form, rows)
    x = x.astype(np.float64)
    k = x.shape[1]
    y = x @ (hi - lo).T
    size = np.abs(x) @ (np.abs(hi) + np.abs(lo)).T
    floor = np.abs(x).max(1, keepdims=True) * (np.abs(hi) + np.abs(lo)).sum(1)
    return y, size * (k / 32 + 128) * 2.0**-23 + floor * 2.0**-39


def attention(q, k, v, scale, cap):
    """(out [heads, dim], tolerance) of one sequence: q [heads, dim], k and v [positions, kv_heads, dim] (the values
    that the pools hold), f64.

    A score sums dim products with q to 22 bits, each step off by 2^-23 of the magnitudes: dz = |q||k| (dim + 4) 2^-23,
    then scale, cap and the base-two exponent's argument, 2^-22 of its size; a weight is off by exp's relative error,
    that of its argument and 2^-22; the output is a weighted mean: twice a weight's error, and a sum of n + 64 steps."""
    heads, dim = q.shape
    n, kv = k.shape[:2]
    out, tol = np.zeros((heads, dim)), np.zeros((heads, dim))
    for h in range(heads):
        kk, vv = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        z = scale * (kk @ q[h])
        dz = abs(scale) * (np.abs(kk) @ np.abs(q[h])) * (dim + 4) * 2.0**-23
        if cap:
            z = cap * np.tanh(z / cap)
        with np.errstate(invalid="ignore"):
            e = np.exp(z - z.max())
            p = e / e.sum()
        dz = dz + (np.abs(z) + np.abs(z.max())) * 2.0**-21
        out[h] = p @ vv
        tol[h] = (2 * (dz.max() + 2.0**-21) + (n + 64) * 2.0**-23) * (p @ np.abs(vv))
    return out, tol


def adjusted(logits, history=None, history_len=None, repeat=None, frequency=None, presence=None, bias_ids=None, bias=None, allowed=None):
    """The definition step by step in f32, as include/emel_hip.h states it: bit-exact."""
    f = np.float32
    out = logits.astype(f).copy()
    rows, card = out.shape
    pick = lambda t, r: t[r if len(t) > 1 else 0]  # noqa: E731
    for r in range(rows):
        if history is not None:
            ids = pick(history, r)
            if history_len is not None:
                ids = ids[: int(np.clip(pick(history_len, r), 0, len(ids)))]
            rep, fr, pr = (f(1) if repeat is None else pick(repeat, r), f(0) if frequency is None else pick(frequency, r), f(0) if presence is None else pick(presence, r))
            for t, n in zip(*np.unique(ids[(ids >= 0) & (ids < card)], return_counts=True)):
                with np.errstate(all="ignore"):
                    l = out[r, t] / rep if out[r, t] > 0 else out[r, t] * rep
                    out[r, t] = (l - f(n) * fr) - pr
        if bias_ids is not None:
            last = {int(t): b for t, b in zip(pick(bias_ids, r), pick(bias, r)) if 0 <= t < card}
            for t, b in last.items():
                out[r, t] = out[r, t] + b
        if allowed is not None:
            bits = (pick(allowed, r).view(np.uint32)[:, None] >> np.arange(32, dtype=np.uint32)) & 1
            out[r, bits.reshape(-1)[:card] == 0] = -np.inf
    return out


# ---- views of torch tensors -----------------------------------------------------------------


def layout(t):
    """The layout of a torch tensor, its dimensions innermost first and padded to four."""
    import torch

    kind = {torch.float32: eh.DType.F32, torch.int32: eh.DType.I32, torch.float16: eh.DType.F16, torch.bfloat16: eh.DType.BF16}[t.dtype]
    shape, nb = list(t.shape)[::-1], [s * t.element_size() for s in t.stride()][::-1]
    while len(shape) < 4:
        nb.append(max(nb[-1] * shape[-1], t.element_size()))
        shape.append(1)
    return eh.Layout(kind, shape, nb)


def view(t):
    return eh.TensorView(t, layout(t))


def out(t):
    return eh.TensorViewMut(t, layout(t))


def packed(t, form, k, m):
    return eh.TensorView(t, eh.Layout.packed(eh.DType.Q4_0 if form == "q4_0" else eh.DType.Q4_K, [k, m, 1, 1]))
