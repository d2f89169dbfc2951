"""CPU: that the exact cases notice what they are for, on results with a mistake planted in them, and what the
operators launch for very many tokens, rows or columns."""
import ctypes
import re

import numpy as np
import pytest

import emel_hip as eh
from decode_exact import exact_product, exact_rows, outlier_columns
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
