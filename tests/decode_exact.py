"""Cases of the served-token operators whose result is exact: small whole numbers times powers of two, of which no
partial sum, in whatever order, passes 24 bits.  So a kernel that sums in f32 gives the result itself, and one that
loses a value, a part of one or a token does not."""
from __future__ import annotations

import numpy as np

from decode_reference import BLOCK, weight_terms
from helpers import rng

SCALE = 2.0**-6  # of every packed block


def exact_rows(seed, form, k, m, zeros=()):
    """m packed rows with weights SCALE (q - 8), or SCALE (sc q - mn) with sc and mn up to 3; zero at `zeros`."""
    values, size = BLOCK[form]
    g = rng(seed)
    b = g.integers(0, 256, (m, k // values, size), dtype=np.uint8)
    half = np.array([SCALE], np.float16).view(np.uint8)
    b[..., :2] = half
    at = np.asarray(zeros, np.int64)
    if form == "q4_0":
        place, high = at % 32 % 16, at % 32 // 16
        keep, none = np.where(high, 0x0F, 0xF0).astype(np.uint8), np.where(high, 0x80, 0x08).astype(np.uint8)
        for i, p, mask, bits in zip(at // 32, place, keep, none):
            b[:, i, 2 + p] = (b[:, i, 2 + p] & mask) | bits
        return b.reshape(m, -1)
    b[..., 2:4] = half
    # six-bit scales and minima up to 3: those of groups 0-3 in bytes 4-11, of 4-7 in the nibbles of bytes 12-15
    b[..., 4:12] &= 3
    b[..., 12:16] &= 0x33
    for i, j, p in zip(at // 256, at % 256 // 32, at % 32):
        q = 16 + 32 * (j // 2) + p
        b[:, i, q] &= 0x0F if j % 2 else 0xF0
        if j < 4:
            b[:, i, 8 + j] = 0
        else:
            b[:, i, 8 + j] &= 0x0F
    return b.reshape(m, -1)


def exact_product(form, rows, x, quantum=1.0):
    """[n, m], for x whose values are multiples of `quantum` (those that meet a weight, at least)."""
    hi, lo = weight_terms(form, rows)
    live = (hi != 0) | (lo != 0)
    x = x.astype(np.float64)
    size = np.where(live.any(0), np.abs(x), 0) @ (np.abs(hi) + np.abs(lo)).T
    assert size.max() < 2.0**23 * SCALE * quantum, "sums of this case may round"
    return x @ (hi - lo).T


def whole_columns(seed, form, k, n):
    """[n, k] f32: values of up to 3, and one in some dozens odd and of 13 bits, which an 11-bit half does not hold."""
    g = rng(seed)
    x = g.integers(-3, 4, (n, k))
    gap = max(16, k // (256 if form == "q4_0" else 96) + 1)
    for c in range(n):
        at = np.arange(int(g.integers(0, min(gap, k))), k, gap)
        x[c, at] = (2 * g.integers(2048, 4096, at.size) + 1) * g.choice([-1, 1], at.size)
    return x.astype(np.float32)


def outlier_columns(seed, k, n, big):
    """([n, k] f32, where the outliers are): multiples of 2^-14 up to 2^-7, and one value of about `big` in 50, which is to
    meet a weight of zero."""
    g = rng(seed)
    x = (g.integers(-127, 128, (n, k)) * 2.0**-14).astype(np.float32)
    at = np.arange(int(g.integers(0, min(50, k))), k, 50)
    x[:, at] = np.float32(big) * g.uniform(1, 2, (n, at.size)).astype(np.float32) * g.choice([-1, 1], (n, at.size)).astype(np.float32)
    return x, at
