"""CPU: what the served-token operators refuse, and in which order, before anything is launched."""
import ctypes

import pytest

import emel_hip as eh
from emel_hip.abi import SIGNATURES
from launch_recorder import LIB

S, F32, F16, BF16, I32, Q4_0, Q4_K = eh.Status, eh.DType.F32, eh.DType.F16, eh.DType.BF16, eh.DType.I32, eh.DType.Q4_0, eh.DType.Q4_K


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(str(LIB))
    for name in SIGNATURES:
        getattr(lib, name).argtypes = SIGNATURES[name]
        getattr(lib, name).restype = ctypes.c_int
    lib.record_count.restype = ctypes.c_uint64
    return lib


def v(slot, ne, dtype=F32, nb=None, mut=False, offset=0, size=1 << 43, packed=False):
    lay = eh.Layout.packed(dtype, ne) if packed else eh.Layout.dense(dtype, ne) if nb is None else eh.Layout(dtype, ne, nb)
    return (eh.TensorViewMut if mut else eh.TensorView)((slot + 1) * (1 << 43) + offset, lay, size)


def status(lib, event):
    lib.record_clear()
    got = S(event._call(lib, None))
    assert (lib.record_count() > 0) == (got == S.OK)
    return got


def null(view):
    view.ptr = 0
    return view


@pytest.mark.parametrize("event,dtype,unit", [(eh.OpMulMatQ4_0, Q4_0, 32), (eh.OpMulMatQ4K, Q4_K, 256)])
def test_product_refusals(lib, event, dtype, unit):
    k, m, n = 2 * unit, 6, 3
    w, x, y = v(0, [k, m, 1, 1], dtype, packed=True), v(1, [k, n, 1, 1]), v(2, [m, n, 1, 1], mut=True)
    ask = lambda a=w, b=x, c=y: status(lib, event(a, b, c))  # noqa: E731
    assert ask() == S.OK
    assert ask(a=None) == ask(b=None) == ask(c=None) == S.INVALID_ARGUMENT
    assert ask(a=null(v(0, [k, m, 1, 1], dtype, packed=True))) == ask(b=v(1, [k, n, 1, 1], offset=2)) == ask(c=v(2, [m, n, 1, 1], mut=True, offset=1)) == S.INVALID_ARGUMENT
    other = Q4_K if dtype == Q4_0 else Q4_0
    assert ask(a=v(0, [256, m, 1, 1], other, packed=True)) == S.INVALID_VIEW
    lay = eh.Layout.packed(dtype, [k, m, 1, 1])
    assert ask(a=eh.TensorView(1 << 43, lay, lay.nb[1] * m - 1)) == S.INVALID_VIEW
    assert ask(a=eh.TensorView(1 << 43, eh.Layout(dtype, [k, m, 1, 1], [1, lay.nb[1] + 2, lay.nb[2], lay.nb[3]]), 1 << 43)) == S.INVALID_VIEW
    assert ask(a=eh.TensorView(1 << 43, eh.Layout(dtype, [k + 16, m, 1, 1], lay.nb), 1 << 43)) == S.INVALID_VIEW
    assert ask(b=v(1, [k, n, 1, 1], size=4 * k * n - 1)) == ask(b=v(1, [k, n, 1, 1], F16)) == ask(b=v(1, [k, 0, 1, 1])) == S.INVALID_VIEW
    assert ask(b=v(1, [k + 1, n, 1, 1])) == ask(b=v(1, [k, n, 2, 1])) == ask(c=v(2, [m, n + 1, 1, 1], mut=True)) == ask(c=v(2, [n, m, 1, 1], mut=True)) == S.SHAPE_MISMATCH
    assert ask(a=v(0, [k, m, 2, 1], dtype, packed=True)) == S.SHAPE_MISMATCH
    assert ask(c=v(1, [m, n, 1, 1], mut=True, offset=4 * k * n - 4)) == ask(c=v(0, [m, n, 1, 1], mut=True, offset=4)) == S.INVALID_VIEW
    assert ask(c=v(2, [m, n, 1, 1], nb=[4, 4, 4 * m, 4 * m], mut=True)) == S.INVALID_VIEW
    assert ask(b=v(1, [k, 1 << 31, 1, 1])) == S.UNSUPPORTED_OPERATION
    big = 1 << 24
    assert ask(a=v(0, [k, big, 1, 1], dtype, packed=True), c=v(2, [big, n, 1, 1], mut=True)) == S.OK
    assert ask(b=v(1, [k, big, 1, 1]), c=v(2, [m, big, 1, 1], mut=True)) == S.OK


def test_append_refusals(lib):
    d, h, t = 64, 2, 5
    parts = dict(k=v(0, [d, h, t, 1]), v=v(1, [d, h, t, 1]), slots=v(2, [t, 1, 1, 1], I32),
                 k_pages=v(3, [d, 16, h, 9], F16, mut=True), v_pages=v(4, [d, 16, h, 9], F16, mut=True))

    def ask(**other):
        return status(lib, eh.OpPagedKvAppend(**{**parts, **other}))

    assert ask() == S.OK
    for name in parts:
        assert ask(**{name: None}) == S.INVALID_ARGUMENT
    assert ask(k_pages=v(3, [d, 16, h, 9], F16, mut=True, offset=1)) == ask(slots=v(2, [t, 1, 1, 1], I32, offset=2)) == S.INVALID_ARGUMENT
    assert ask(k_pages=v(3, [d, 16, h, 9], F32, mut=True)) == ask(slots=v(2, [t, 1, 1, 1])) == ask(k=v(0, [d, h, t, 1], F16)) == S.INVALID_VIEW
    assert ask(k_pages=v(3, [d, 16, h, 9], F16, mut=True, size=d * 16 * h * 9 * 2 - 1)) == S.INVALID_VIEW
    assert ask(k_pages=v(3, [d, 16, h, 9], F16, [4, 256, 4096, 8192], mut=True)) == S.INVALID_VIEW
    assert ask(k_pages=v(3, [d, 16, h, 9], F16, [2, 127, 4096, 8192], mut=True)) == S.INVALID_VIEW
    assert ask(v_pages=v(4, [d, 16, h, 9], BF16, mut=True)) == ask(v_pages=v(4, [d, 16, h, 8], F16, mut=True)) == S.SHAPE_MISMATCH
    assert ask(k=v(0, [d, h + 1, t, 1])) == ask(v=v(1, [d, h, t + 1, 1])) == ask(slots=v(2, [t + 1, 1, 1, 1], I32)) == S.SHAPE_MISMATCH
    assert ask(v_pages=parts["k_pages"]) == ask(k=v(3, [d, h, t, 1])) == ask(slots=v(4, [t, 1, 1, 1], I32, offset=64)) == S.INVALID_VIEW
    assert ask(k_pages=v(3, [d, 16, h, 9], F16, [2, 64, 1024, 2048], mut=True)) == S.INVALID_VIEW  # its own slots overlap
    # keys and values side by side in every page, and not quite
    nb = [2, 128, 2048, 8192]
    side = lambda at: ask(k_pages=v(3, [d, 16, h, 9], F16, nb, mut=True), v_pages=v(3, [d, 16, h, 9], F16, nb, mut=True, offset=at))  # noqa: E731
    assert side(4096) == S.OK and side(4094) == side(2048) == side(128) == S.INVALID_VIEW
    assert ask(slots=v(2, [1 << 31, 1, 1, 1], I32)) == S.UNSUPPORTED_OPERATION


def test_attention_refusals(lib):
    d, h, kv, s = 64, 6, 2, 5
    parts = dict(q=v(0, [d, h, s, 1]), k_pages=v(1, [d, 16, kv, 9], BF16), v_pages=v(2, [d, 16, kv, 9], BF16), page_table=v(3, [7, s, 1, 1], I32),
                 lengths=v(4, [s, 1, 1, 1], I32), output=v(5, [d, h, s, 1], mut=True), scale=0.1, window=0, soft_cap=0.0)

    def ask(**other):
        return status(lib, eh.OpPagedAttention(**{**parts, **other}))

    assert ask() == ask(window=2**63, soft_cap=1.0, scale=-1.0) == S.OK
    for name in ("q", "k_pages", "v_pages", "page_table", "lengths", "output"):
        assert ask(**{name: None}) == S.INVALID_ARGUMENT
    assert ask(v_pages=v(2, [d, 16, kv, 9], BF16, offset=1)) == ask(q=v(0, [d, h, s, 1], offset=2)) == S.INVALID_ARGUMENT
    assert ask(k_pages=v(1, [d, 16, kv, 9])) == ask(lengths=v(4, [s, 1, 1, 1])) == ask(q=v(0, [d, h, s, 1], size=4 * d * h * s - 4)) == S.INVALID_VIEW
    assert ask(page_table=v(3, [7, s, 1, 1], I32, size=4 * 7 * s - 4)) == ask(lengths=v(4, [0, 1, 1, 1], I32)) == S.INVALID_VIEW
    assert ask(v_pages=v(2, [d, 16, kv, 9], F16)) == ask(v_pages=v(2, [d, 16, kv, 10], BF16)) == ask(q=v(0, [d, 5, s, 1]), output=v(5, [d, 5, s, 1], mut=True)) == S.SHAPE_MISMATCH
    assert ask(page_table=v(3, [7, s + 1, 1, 1], I32)) == ask(lengths=v(4, [s - 1, 1, 1, 1], I32)) == ask(output=v(5, [d, h, s, 2], mut=True)) == S.SHAPE_MISMATCH
    assert ask(scale=float("nan")) == ask(scale=float("inf")) == ask(soft_cap=-1.0) == ask(soft_cap=float("nan")) == S.INVALID_PARAMETERS
    for dim in (4, 60, 264):
        pool = v(1, [dim, 16, kv, 9], BF16), v(2, [dim, 16, kv, 9], BF16)
        assert ask(q=v(0, [dim, h, s, 1]), k_pages=pool[0], v_pages=pool[1], output=v(5, [dim, h, s, 1], mut=True)) == S.UNSUPPORTED_OPERATION
    assert ask(page_table=v(3, [1 << 27, s, 1, 1], I32)) == S.UNSUPPORTED_OPERATION
    for at in range(5):
        assert ask(output=v(at, [d, h, s, 1], mut=True)) == S.INVALID_VIEW
    assert ask(output=v(5, [d, h, s, 1], nb=[4, 4, 4 * d, 4 * d * s], mut=True)) == S.INVALID_VIEW


def test_logits_adjust_refusals(lib):
    card, rows = 100, 3
    parts = dict(history=v(2, [9, rows, 1, 1], I32), history_len=v(3, [rows, 1, 1, 1], I32), repeat=v(4, [rows, 1, 1, 1]), frequency=v(5, [rows, 1, 1, 1]),
                 presence=v(6, [1, 1, 1, 1]), bias_ids=v(7, [4, rows, 1, 1], I32), bias=v(8, [4, rows, 1, 1]), allowed=v(9, [4, 1, 1, 1], I32))
    x, y = v(0, [card, rows, 1, 1]), v(1, [card, rows, 1, 1], mut=True)

    def ask(logits=x, adjusted=y, **other):
        return status(lib, eh.OpLogitsAdjust(logits, adjusted, **{**parts, **other}))

    assert ask() == ask(adjusted=v(0, [card, rows, 1, 1], mut=True)) == S.OK
    assert status(lib, eh.OpLogitsAdjust(x, y)) == S.OK
    assert ask(logits=None) == ask(adjusted=None) == ask(bias=v(8, [4, rows, 1, 1], offset=2)) == S.INVALID_ARGUMENT
    assert lib.emel_logits_adjust(None, None) == S.INVALID_ARGUMENT
    assert ask(bias=None) == ask(bias_ids=None) == ask(history=None) == S.INVALID_REQUEST
    reserved = eh.OpLogitsAdjust(x, y)
    reserved._args[0]._obj.reserved = 1
    assert status(lib, reserved) == S.INVALID_REQUEST
    assert ask(history=v(2, [9, rows, 1, 1])) == ask(repeat=v(4, [rows, 1, 1, 1], I32)) == ask(logits=v(0, [card, rows, 1, 1], size=4 * card * rows - 1)) == S.INVALID_VIEW
    assert ask(logits=v(0, [card, rows + 1, 1, 1])) == ask(history=v(2, [9, 2, 1, 1], I32)) == ask(repeat=v(4, [2, 1, 1, 1])) == S.SHAPE_MISMATCH
    assert ask(bias=v(8, [5, rows, 1, 1])) == ask(bias=v(8, [4, 1, 1, 1])) == ask(allowed=v(9, [3, 1, 1, 1], I32)) == ask(allowed=v(9, [5, 1, 1, 1], I32)) == S.SHAPE_MISMATCH
    assert ask(adjusted=v(0, [card, rows, 1, 1], mut=True, offset=4)) == ask(adjusted=v(9, [card, rows, 1, 1], mut=True)) == S.INVALID_VIEW
    assert ask(adjusted=v(1, [card, rows, 1, 1], nb=[4, 8, 1200, 1200], mut=True)) == S.INVALID_VIEW
    assert ask(history=v(2, [1 << 31, 1, 1, 1], I32)) == S.UNSUPPORTED_OPERATION
