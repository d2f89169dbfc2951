"""A served token's events over packed weights and a paged key-value cache.

    kernel.process_event(OpMulMatQ4K(TensorView(w, Layout.packed(DType.Q4_K, [k, m, 1, 1])),
                                     TensorView(x, ...), TensorViewMut(y, ...)))
    kernel.process_event(OpPagedKvAppend(k, v, slots, k_pages, v_pages))
    kernel.process_event(OpPagedAttention(q, k_pages, v_pages, page_table, lengths, out, scale=dim ** -0.5))
    kernel.process_event(OpLogitsAdjust(logits, logits, history=ids, repeat=r, allowed=bits))

None has a counterpart in the reference's events; include/emel_hip.h holds
their formulas, layouts and guards.  Every view is device memory.  An event
may be kept and processed again: it then reads and writes the same views,
with what they hold by then.  Its operands' C views are laid out once, on
construction, so an event is immutable (a call of six views takes the host
3.9 us, 6.3 us with the event built anew).
"""
from __future__ import annotations

import ctypes

from .abi import CLogitsAdjustRequest
from .views import TensorView, TensorViewMut


class _Event:
    """Keeps the views (and so their memory) and the C arguments of one call."""

    __slots__ = ("_views", "_args")
    _fn = ""

    def _bind(self, views, *more):
        self._views = views
        self._args = tuple(None if v is None else ctypes.byref(v.c()) for v in views[:-1]) + more
        self._args += (None if views[-1] is None else ctypes.byref(views[-1].c()),)

    def _call(self, lib, s):
        return getattr(lib, self._fn)(*self._args, s)


class OpMulMatQ4_0(_Event):
    """dst[r, c] = sum_k W[r, k] x[k, c], W packed Q4_0 rows (emel_op_mul_mat_q4_0)."""

    __slots__ = ()
    _fn = "emel_op_mul_mat_q4_0"

    def __init__(self, weights: TensorView, x: TensorView, dst: TensorViewMut):
        self._bind((weights, x, dst))


class OpMulMatQ4K(OpMulMatQ4_0):
    """OpMulMatQ4_0 over packed Q4_K rows (emel_op_mul_mat_q4_k)."""

    __slots__ = ()
    _fn = "emel_op_mul_mat_q4_k"


class OpPagedKvAppend(_Event):
    """Writes new tokens' keys and values into their slots of the page pools (emel_op_paged_kv_append)."""

    __slots__ = ()
    _fn = "emel_op_paged_kv_append"

    def __init__(self, k: TensorView, v: TensorView, slots: TensorView, k_pages: TensorViewMut, v_pages: TensorViewMut):
        self._bind((k, v, slots, k_pages, v_pages))


class OpPagedAttention(_Event):
    """Attention of one new token per sequence over its cached pages (emel_op_paged_attention).

    window 0 attends to every position, soft_cap 0 leaves the scores as they are."""

    __slots__ = ()
    _fn = "emel_op_paged_attention"

    def __init__(self, q: TensorView, k_pages: TensorView, v_pages: TensorView, page_table: TensorView,
                 lengths: TensorView, output: TensorViewMut, scale: float, window: int = 0, soft_cap: float = 0.0):
        self._bind((q, k_pages, v_pages, page_table, lengths, output), scale, window, soft_cap)


class OpLogitsAdjust(_Event):
    """Penalties, biases and a token mask on rows of logits (emel_logits_adjust); adjusted may be logits itself."""

    __slots__ = ()

    def __init__(self, logits: TensorView, adjusted: TensorViewMut, *, history: TensorView | None = None,
                 history_len: TensorView | None = None, repeat: TensorView | None = None,
                 frequency: TensorView | None = None, presence: TensorView | None = None,
                 bias_ids: TensorView | None = None, bias: TensorView | None = None,
                 allowed: TensorView | None = None):
        r = CLogitsAdjustRequest()
        self._views = (logits, adjusted, history, history_len, repeat, frequency, presence, bias_ids, bias, allowed)
        for (name, _), view in zip(CLogitsAdjustRequest._fields_, self._views):
            if view is not None:
                setattr(r, name, ctypes.pointer(view.c()))
        self._args = (ctypes.byref(r),)

    _fn = "emel_logits_adjust"
