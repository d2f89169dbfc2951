"""CPU: that the exact cases notice what they are for, on results with a mistake planted in them, and what the
operators launch for very many tokens, rows or columns."""
import ctypes
import re

import numpy as np
import pytest

import emel_hip as eh
from decode_exact import cancelling, cancelling_attention, exact_product, exact_rows, flat_means_differ, flat_values, outlier_columns, whole_columns
from decode_reference import weight_terms
from launch_recorder import Recorder
from launch_recorder import view as wide_view


@pytest.fixture(scope="module")
def rec():
    return Recorder()


def fixed_point(x, bits):
    """x as multiples of 2^-bits of each run's largest power of two."""
    k = x.shape[1]
    runs = np.pad(x.astype(np.float64), ((0, 0), (0, -k % 256))).reshape(len(x), -1, 256)
    unit = 2.0 ** (np.floor(np.log2(np.abs(runs).max(2, keepdims=True))) - bits + 1)
    return (np.rint(runs / unit) * unit).reshape(len(x), -1)[:, :k]


@pytest.mark.parametrize("form", ["q4_0", "q4_k"])
def test_weights_of_exact_rows(form):
    zeros = [0, 17, 100, 255, 300, 511]
    hi, lo = weight_terms(form, exact_rows(1, form, 512, 40, zeros))
    w = (hi - lo) * 64
    assert (w[:, zeros] == 0).all() and (w == np.rint(w)).all() and np.abs(w).max() <= 48
    assert (np.delete(w, zeros, 1) != 0).mean() > 0.7


@pytest.mark.parametrize("form", ["q4_0", "q4_k"])
@pytest.mark.parametrize("big", [2.0**20, 2.0**30])
def test_thirty_bits_are_too_few_beside_towering_values(form, big):
    x, at = outlier_columns(3, 3840, 2, big)
    rows = exact_rows(4, form, 3840, 70, at)
    want = exact_product(form, rows, x, 2.0**-14)
    hi, lo = weight_terms(form, rows)
    assert (fixed_point(x, 30) @ (hi - lo).T != want).mean() > 0.95
    assert np.array_equal(fixed_point(x, 60) @ (hi - lo).T, want)


@pytest.mark.parametrize("tokens,launches", [(1 << 17, 1), ((1 << 17) + 1, 2), (1 << 20, 8), ((1 << 31) - 1, 1 << 14)])
def test_append_looks_through_no_more_tokens_than_a_launch_takes(rec, tokens, launches):
    """Each workgroup looks through all later slots of its launch, so a launch's tokens bound what a token costs."""
    kv = [wide_view(i, [8, 1, tokens, 1]) for i in (0, 1)]
    pools = [wide_view(i, [8, 16, 1, 9000], dtype=eh.DType.F16, mut=True) for i in (2, 3)]
    got = rec.launches(eh.OpPagedKvAppend(*kv, wide_view(4, [tokens, 1, 1, 1], dtype=eh.DType.I32), *pools))
    per = [int(re.search(r", (\d)u,", g.name).group(1)) for g in got]
    assert len(got) == launches and sum(g.grid * p for g, p in zip(got, per)) in range(tokens, tokens + 8)
    assert max(g.grid * p for g, p in zip(got, per)) == 1 << 17


@pytest.mark.parametrize("k,m,n", [(1 << 26, 300, 16), (1 << 26, 300, 12), (1 << 26, 300, 5), (1 << 26, 17, 70), (3 << 24, 200, 16), (1 << 25, 200, 16),
                                   (11008, 1 << 22, 32), (4096, 151936, 102), (64, 33, 1 << 21)])
def test_partial_sums_stay_within_256_mb(rec, k, m, n):
    w = eh.TensorView(1 << 43, eh.Layout.packed(eh.DType.Q4_0, [k, m, 1, 1]), 1 << 62)
    stream = ctypes.c_void_p(0x1000 + 16 * (k + m + n))  # its own: a stream's workspace only grows
    event = eh.OpMulMatQ4_0(w, wide_view(1, [k, n, 1, 1]), wide_view(2, [m, n, 1, 1], mut=True))
    assert eh.Status(event._call(rec.lib, stream)) == eh.Status.OK
    work, counters = ctypes.c_uint64(), ctypes.c_uint64()
    assert rec.lib.emel_stream_workspace(stream, ctypes.byref(work), ctypes.byref(counters)) == 0
    assert 1 << 20 <= work.value <= 256 << 20


def nearest(x, bits):
    """x to `bits` significant bits."""
    with np.errstate(divide="ignore"):
        unit = 2.0 ** (np.floor(np.log2(np.abs(np.where(x == 0, 1, x)))) - bits + 1)
    return np.rint(x / unit) * unit


def cut(x, bits):
    """x cut after `bits` significant bits."""
    unit = 2.0 ** (np.floor(np.log2(np.abs(np.where(x == 0, 1, x)))) - bits + 1)
    return np.trunc(x / unit) * unit


@pytest.mark.parametrize("form,k", [("q4_0", 4096), ("q4_0", 32768), ("q4_k", 4096), ("q4_k", 11008)])
def test_lost_low_halves_and_lost_values_show(form, k):
    """Columns to 11 bits, or without one value, differ from the exact results nearly everywhere."""
    x, rows = whole_columns(1, form, k, 5), exact_rows(2, form, k, 60)
    want = exact_product(form, rows, x)
    hi, lo = weight_terms(form, rows)
    assert (nearest(x, 11) @ (hi - lo).T != want).mean() > 0.95
    without = x.copy()
    without[:, k // 2] = 0
    changed = (hi - lo)[:, k // 2] != 0
    assert ((without @ (hi - lo).T != want) == ((x[:, k // 2] != 0)[:, None] & changed)).all()


@pytest.mark.parametrize("n", [1, 33, 20000, 150000])
def test_a_lost_or_doubled_position_shows(n):
    v = flat_values(n, 1, 1, n, 16)[0]
    mean = v.sum(1, dtype=np.float64) / n
    assert not flat_means_differ(mean.astype(np.float32), v, n).any()
    for j in {0, n // 2, n - 1}:
        for sign in (1, -1):
            off = (mean + sign * v[:, j] / n).astype(np.float32)
            assert np.array_equal(flat_means_differ(off, v, n)[0], v[0, j] != 0)


@pytest.mark.parametrize("dim", [8, 64, 136, 256])
@pytest.mark.parametrize("part", ["q: f16, one half", "q: bf16, two parts", "weights: f16, one half", "weights: bf16, two parts"])
def test_lost_parts_of_queries_and_weights_show(dim, part):
    kept = (lambda x: nearest(x, 11)) if "f16, one" in part else (lambda x: cut(x, 16))
    seen = []
    for seed in range(8):
        q, k, v = cancelling(seed, 1, 4, 3, dim)
        want, tol = cancelling_attention(q, k, v, 3)
        got, _ = cancelling_attention(q, k, v, 3, **{"q_part" if part[0] == "q" else "p_part": kept})
        seen.append((abs(got - want) > tol).mean())
    assert min(seen) > 0.1, seen
