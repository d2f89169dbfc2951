"""CPU: that the exact cases notice what they are for, on results with a mistake planted in them."""
import numpy as np
import pytest

from decode_exact import exact_product, exact_rows, outlier_columns
from decode_reference import weight_terms


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
