"""Rotary positions of several axes from their formula, in 64 bits with numpy."""
from __future__ import annotations

import numpy as np


def pairs_of(sections, in_turn=False, own=False):
    """[(axis, exponent's number, its count)] of each pair, as include/emel_hip.h deals them out."""
    left, axis = list(sections), []
    if in_turn:
        while any(left):
            for a, n in enumerate(left):
                if n:
                    axis.append(a)
                    left[a] -= 1
    else:
        for a, n in enumerate(left):
            axis += [a] * n
    total = len(axis)
    return [(a, axis[:i].count(a), sections[a]) if own else (a, i, total) for i, a in enumerate(axis)]


def rope(x, positions, sections, *, base=1e4, scale=1.0, magnitude=1.0, factors=None, adjacent=False, in_turn=False, own=False, backward=False):
    """(out [tokens, heads, dim], tolerance) for x [tokens, heads, dim] f32 and positions [axes, tokens].

    The library's cos and sin are off by 2^-23 at most: their argument, below 0.8, is rounded to f32 (2^-25), the series'
    terms and their sum once each (2^-24.7 and 2^-25 for cos, the larger one), what the series leaves out is below 2^-28;
    magnitude, the products and the sum round once more each: 2^-22 of magnitude (|x| + |y|) holds all of it.  An
    exponent's rounding, of up to 24, is 2^-48 of it, a frequency's then 2^-46 with its product's and quotient's."""
    x = x.astype(np.float64)
    y, tol = x.copy(), np.zeros_like(x)
    plan = pairs_of(sections, in_turn, own)
    n = len(plan)
    f32 = lambda v: np.float64(np.float32(v))  # noqa: E731
    for i, (a, j, count) in enumerate(plan):
        p, r = (2 * i, 2 * i + 1) if adjacent else (i, i + n)
        freq = f32(scale) * f32(base) ** (-j / count) / (1.0 if factors is None else np.float64(factors[i]))
        angle = positions[a].astype(np.float64)[:, None] * freq
        c, s = np.cos(angle), np.sin(-angle if backward else angle)
        y[..., p] = f32(magnitude) * (x[..., p] * c - x[..., r] * s)
        y[..., r] = f32(magnitude) * (x[..., p] * s + x[..., r] * c)
        tol[..., p] = tol[..., r] = abs(f32(magnitude)) * (np.abs(x[..., p]) + np.abs(x[..., r])) * (2.0**-22 + np.abs(angle) * 2.0**-46) + 2.0**-148
    return y, tol
