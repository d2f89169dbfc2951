"""Packed rows of the paged cache from their definition, with numpy: bit for bit as they are stored, and their values in
64 bits; and the pools that the tests share."""
from __future__ import annotations

import numpy as np

import emel_hip as eh
from helpers import rng

SIZE = {"q8_0": 34, "q4_0": 18}
TYPES = {"q8_0": eh.DType.Q8_0, "q4_0": eh.DType.Q4_0}
NIBBLE_OF = [0, 4, 1, 5, 2, 6, 3, 7]  # of an eight's values, lowest bits first


def encode(kind, x):
    """Rows of f32 [..., dim] as bytes [..., bytes of a row]."""
    shape = x.shape
    x = x.reshape(-1, shape[-1]).astype(np.float32)
    blocks = shape[-1] // 32
    out = np.zeros((len(x), blocks * SIZE[kind]), np.uint8)
    b = x.reshape(len(x), blocks, 32)
    fine = np.isfinite(b).all(2)
    safe = np.where(fine[..., None], b, np.float32(0))
    size = np.abs(safe).max(2)
    if kind == "q8_0":
        d = (size.astype(np.float64) / 127.0).astype(np.float32)
    else:
        first = np.abs(safe).argmax(2)  # the first of equal ones
        d = np.take_along_axis(safe, first[..., None], 2)[..., 0] * np.float32(-0.125)
    d = np.clip(d, np.float32(-65504), np.float32(65504)).astype(np.float16)
    wide = d.astype(np.float64)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        n = np.where(wide == 0, 0.0, np.rint(safe.astype(np.float64) / wide))  # exact enough to tell every tie
    d[~fine] = np.uint16(0x7E00).view(np.float16)
    n[~fine] = 0
    for j in range(blocks):
        for i in range(32):
            unit, at = i // 8 * blocks + j, i % 8
            if kind == "q8_0":
                out[:, 8 * unit + at] = np.clip(n[:, j, i], -127, 127).astype(np.int8).view(np.uint8)
            else:
                nib = NIBBLE_OF[at]
                out[:, 4 * unit + nib // 2] |= (np.clip(n[:, j, i], -8, 7) + 8).astype(np.uint8) << (4 * (nib % 2))
    out[:, -2 * blocks:] = np.ascontiguousarray(d).view(np.uint8).reshape(len(x), -1)
    return out.reshape(*shape[:-1], -1)


def decode(kind, rows):
    """The values [..., dim] of packed rows, f64."""
    shape = rows.shape
    b = rows.reshape(-1, shape[-1])
    blocks = shape[-1] // SIZE[kind]
    d = np.ascontiguousarray(b[:, -2 * blocks:]).view(np.float16).astype(np.float64)
    d[~np.isfinite(d)] = np.nan
    out = np.empty((len(b), 32 * blocks))
    for j in range(blocks):
        for i in range(32):
            unit, at = i // 8 * blocks + j, i % 8
            if kind == "q8_0":
                n = b[:, 8 * unit + at].astype(np.int8).astype(np.float64)
            else:
                nib = NIBBLE_OF[at]
                n = (b[:, 4 * unit + nib // 2] >> (4 * (nib % 2)) & 15) - 8.0
            out[:, 32 * j + i] = d[:, j] * n
    return out.reshape(*shape[:-1], -1)


def random_rows(seed, kind, count, dim, size=0.05):
    """Rows with every whole number, scales of both signs spread over a factor of some hundred."""
    g = rng(seed)
    blocks = dim // 32
    rows = g.integers(0, 256, (count, blocks * SIZE[kind]), dtype=np.uint8)
    if kind == "q8_0":  # -128 is none of the format's numbers
        rows[:, : 32 * blocks][rows[:, : 32 * blocks] == 128] = 0
    d = (g.standard_normal((count, blocks)) * size * np.exp(g.standard_normal((count, blocks)))).astype(np.float16)
    rows[:, -2 * blocks:] = d.view(np.uint8)
    return rows


def pool_tensors(device, kinds, pages, kv, page, dim, order, seed=None, fill=0xAA):
    """Pools of keys and values as byte tensors [pages, kv, page, bytes of a row] and everything that they lie in.

    "head": a head's tokens side by side; "token": a token's heads; "both": keys and values of a page interleaved by
    rows; "apart": rows, heads and pages with gaps, at odd multiples of two bytes."""
    import torch

    row = [dim // 32 * SIZE[k] for k in kinds]
    if order == "both":
        store = torch.full((pages, kv, page, sum(row)), fill, dtype=torch.uint8, device=device)
        both = [store[..., : row[0]], store[..., row[0]:]]
    elif order == "apart":
        store = torch.full((2, pages, kv, page, max(row) + 6), fill, dtype=torch.uint8, device=device)
        both = [store[i, ..., 2: 2 + row[i]] for i in range(2)]
    else:
        store = torch.full((pages * kv * page * sum(row) + 2,), fill, dtype=torch.uint8, device=device)
        first = pages * kv * page * row[0]
        flat = store[2: 2 + first], store[2 + first:]
        shape = lambda i: (pages, kv, page, row[i]) if order == "head" else (pages, page, kv, row[i])  # noqa: E731
        both = [flat[i].view(shape(i)) if order == "head" else flat[i].view(shape(i)).transpose(1, 2) for i in range(2)]
    if seed is not None:
        for i, t in enumerate(both):
            rows = random_rows(seed + i, kinds[i], pages * kv * page, dim).reshape(pages, kv, page, row[i])
            t.copy_(torch.from_numpy(rows).to(device))
    return both[0], both[1], store


def pages_view(t, kind, dim, mut=False):
    """The view of a byte tensor [pages, kv, page, bytes of a row]."""
    lay = eh.Layout(TYPES[kind], [dim, t.shape[2], t.shape[1], t.shape[0]], [1, t.stride(2), t.stride(1), t.stride(0)])
    return (eh.TensorViewMut if mut else eh.TensorView)(t, lay)
