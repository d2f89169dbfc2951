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
    gap = max(16, k // (200 if form == "q4_0" else 48) + 1)
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


# ---- attention ------------------------------------------------------------------------------


def flat_values(seed, seqs, kv, positions, dim):
    """Whole numbers of up to 3 for every position and dim: the flat mean over any positions names them."""
    return rng(seed).integers(-3, 4, (seqs, kv, positions, dim)).astype(np.float32)


def flat_means_differ(got, v, n, window=0):
    """Where `got` [heads, dim] is not the mean of v [kv_heads, positions, dim] over the window's positions.

    With scores of zero every weight is one (or 2^14), sums of whole numbers below 2^24 are exact, and what is left is the
    reciprocal of the number of positions and the product with it, each off by half a step: 2^-24 of the mean.  A position
    more or less changes a sum of at most 3 n, below 2^20, by 1 or more, which is 2^-20 of it."""
    start = max(0, n - window) if window else 0
    total = v[:, start:n].sum(1, dtype=np.float64).repeat(len(got) // len(v), 0)
    count = n - start
    assert 3 * count < 2**20
    return ~(np.abs(got.astype(np.float64) * count - total) <= np.abs(total) * 2.0**-22)


def exact_scale(power):
    """An f32 scale whose f32 product with f32's log2(e) is 2^power exactly."""
    log2e = np.float32(1.4426950408889634)
    s = np.float32(2.0**power / 1.4426950408889634)
    for s in (s, np.nextafter(s, np.float32(0)), np.nextafter(s, np.float32(1))):
        if s * log2e == np.float32(2.0**power):
            return float(s)
    raise AssertionError("no such scale")


POWER = -17


def cancelling(seed, kv, heads, positions, dim):
    """(q [heads, dim], k [kv, positions, dim], v): q odd whole numbers of 20 bits, keys of one 1 and one -1 each, so
    that scores are differences of q's values times 2^POWER: exact in f32, below 4, and wrong wherever a part of q is lost."""
    g = rng(seed)
    q = (2 * g.integers(1 << 18, 1 << 19, (heads, dim)) + 1).astype(np.float32)
    k = np.zeros((kv, positions, dim), np.float32)
    j = np.arange(positions)
    for h in range(kv):
        a = (j * 3 + seed + h) % dim
        b = (a + 1 + g.integers(0, dim - 1, positions)) % dim
        k[h, j, a], k[h, j, b] = 1, -1
    return q, k, g.integers(-9, 10, (kv, positions, dim)).astype(np.float32)


def cancelling_attention(q, k, v, n, q_part=lambda x: x, p_part=lambda x: x):
    """(out [heads, dim], tolerance) in f64; q_part and p_part stand for what a kernel keeps of q and of the weights.

    Scores are exact but for the rounding of the scale's product with log2(e).  A weight is off by 2^-23 (exp2) and 2^-22
    (two halves of 11 bits); numerator and denominator are sums of up to 32 products in an instruction, then of n / 128
    steps, four waves and a row's parts, each step 2^-24 of the terms so far."""
    rounding = abs(exact_scale(POWER) / 2.0**POWER / np.log(2.0) - 1)
    h, kv = len(q), len(k)
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(h):
        kk, vv = k[i // (h // kv), :n].astype(np.float64), v[i // (h // kv), :n].astype(np.float64)
        z = kk @ q_part(q[i].astype(np.float64)) * exact_scale(POWER)
        e = np.exp(z - z.max())
        out[i] = (p_part(e) @ vv) / e.sum()
        tol[i] = (2 * (np.abs(z).max() * rounding + 2.0**-23 + 2.0**-22) + 2 * (min(n, 32) + n / 128 + 8) * 2.0**-24) * (e @ np.abs(vv)) / e.sum()
    return out, tol
