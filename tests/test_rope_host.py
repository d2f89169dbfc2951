"""CPU: what rotary positions refuse, in which order, what they launch, and how pairs are dealt out."""
import ctypes

import pytest

import emel_hip as eh
from launch_recorder import Recorder, view
from rope_reference import pairs_of

S, F16, I32 = eh.Status, eh.DType.F16, eh.DType.I32


@pytest.fixture(scope="module")
def rec():
    return Recorder()


def parts(dim=64, heads=6, kv=2, tokens=5, axes=3):
    return dict(q=view(0, [dim, heads, tokens, 1]), q_out=view(1, [dim, heads, tokens, 1], mut=True), k=view(2, [dim, kv, tokens, 1]),
                k_out=view(3, [dim, kv, tokens, 1], mut=True), positions=view(4, [tokens, axes, 1, 1], dtype=I32),
                factors=view(5, [20, 1, 1, 1]), sections=[8, 6, 6])


def ask(rec, **other):
    lib = rec.lib
    lib.record_clear()
    got = S(eh.OpRope(**{**parts(), **other})._call(lib, None))
    assert (lib.record_count() > 0) == (got == S.OK)
    return got


def null(v):
    v.ptr = 0
    return v


def test_refusals(rec):
    d, h, kv, t = 64, 6, 2, 5
    out = lambda slot, ne, **kw: view(slot, ne, mut=True, **kw)  # noqa: E731
    assert ask(rec) == ask(rec, factors=None) == ask(rec, k=None, k_out=None) == S.OK
    for name in ("q", "q_out", "positions"):
        assert ask(rec, **{name: None}) == S.INVALID_ARGUMENT
    assert rec.lib.emel_op_rope(None, None) == S.INVALID_ARGUMENT
    assert ask(rec, q=null(view(0, [d, h, t, 1]))) == ask(rec, k=view(2, [d, kv, t, 1], offset=2)) == ask(rec, factors=view(5, [20, 1, 1, 1], offset=1)) == S.INVALID_ARGUMENT
    assert ask(rec, k=None) == ask(rec, k_out=None) == S.INVALID_REQUEST
    for flags in (16, 1 << 31):
        event = eh.OpRope(**parts())
        event._args[0]._obj.flags = flags
        assert event._call(rec.lib, None) == S.INVALID_REQUEST
    assert ask(rec, q=view(0, [1 << 31, h, t, 1])) == ask(rec, positions=view(4, [1 << 31, 3, 1, 1], dtype=I32)) == S.UNSUPPORTED_OPERATION
    big = (1 << 24) + 2
    assert ask(rec, q=view(0, [big, h, t, 1]), q_out=out(1, [big, h, t, 1]), k=None, k_out=None) == S.UNSUPPORTED_OPERATION
    many = (1 << 31) - 1
    assert ask(rec, q=view(0, [2, many, 1, 1]), q_out=out(1, [2, many, 1, 1]), k=view(2, [2, 1, 1, 1]), k_out=out(3, [2, 1, 1, 1]), factors=None,
               positions=view(4, [1, 1, 1, 1], dtype=I32), sections=[1]) == S.UNSUPPORTED_OPERATION
    assert ask(rec, q=view(0, [d, h, t, 1], dtype=F16)) == ask(rec, positions=view(4, [t, 3, 1, 1])) == ask(rec, factors=view(5, [20, 1, 1, 1], dtype=I32)) == S.INVALID_VIEW
    assert ask(rec, q=view(0, [d, h, 0, 1])) == S.INVALID_VIEW
    assert ask(rec, q_out=out(1, [d, h, t + 1, 1])) == ask(rec, k=view(2, [d + 2, kv, t, 1])) == ask(rec, k_out=out(3, [d, kv + 1, t, 1])) == S.SHAPE_MISMATCH
    assert ask(rec, positions=view(4, [t + 1, 3, 1, 1], dtype=I32)) == ask(rec, positions=view(4, [t, 5, 1, 1], dtype=I32)) == ask(rec, factors=view(5, [21, 1, 1, 1])) == S.SHAPE_MISMATCH
    assert ask(rec, q=view(0, [d, h, t, 2]), q_out=out(1, [d, h, t, 2])) == S.SHAPE_MISMATCH
    assert ask(rec, sections=[8, 6, 5, 1]) == ask(rec, sections=[], factors=None) == ask(rec, sections=[20, 7, 6], factors=None) == S.INVALID_PARAMETERS
    assert ask(rec, sections=[2**32 - 1, 2**32 - 1, 2], factors=None) == S.INVALID_PARAMETERS
    for bad in (float("nan"), float("inf")):
        assert ask(rec, base=bad) == ask(rec, scale=bad) == ask(rec, magnitude=bad) == S.INVALID_PARAMETERS
    assert ask(rec, base=0.0) == ask(rec, base=-2.0) == S.INVALID_PARAMETERS
    assert ask(rec, sections=[0, 20, 0]) == ask(rec, sections=[20, 12, 0], factors=None) == ask(rec, scale=0.0, magnitude=-1.0, base=0.5) == S.OK


def test_overlaps(rec):
    d, h, kv, t = 64, 6, 2, 5
    p = parts()
    out = lambda v: eh.TensorViewMut(v.ptr, v.layout, v.data_bytes)  # noqa: E731
    assert ask(rec, q_out=out(p["q"])) == ask(rec, q_out=out(p["q"]), k_out=out(p["k"])) == S.OK
    assert ask(rec, q_out=out(view(0, [d, h, t, 1], offset=4))) == ask(rec, q_out=out(view(4, [d, h, t, 1]))) == ask(rec, q_out=out(view(5, [d, h, t, 1]))) == S.INVALID_VIEW
    assert ask(rec, q_out=out(view(2, [d, h, t, 1]))) == ask(rec, k_out=out(view(0, [d, kv, t, 1]))) == ask(rec, k_out=out(view(1, [d, kv, t, 1]))) == S.INVALID_VIEW
    assert ask(rec, q_out=out(view(1, [d, h, t, 1], nb=[4, 4, 4 * d * h, 4 * d * h * t]))) == S.INVALID_VIEW
    # queries, keys and values of a token side by side, in place
    nb = [4, 4 * d, 4 * d * (h + 2 * kv), 4 * d * (h + 2 * kv) * t]
    fused = lambda at, heads: view(0, [d, heads, t, 1], nb=nb, offset=4 * d * at)  # noqa: E731
    q, k = fused(0, h), fused(h, kv)
    assert ask(rec, q=q, q_out=out(q), k=k, k_out=out(k)) == ask(rec, q=k, q_out=out(k), k=q, k_out=out(q)) == S.OK
    late = fused(h - 1, kv)
    assert ask(rec, q=q, q_out=out(q), k=late, k_out=out(late)) == S.INVALID_VIEW
    past = fused(h + 2 * kv - 1, kv)  # its second head is the next token's first
    assert ask(rec, q=q, q_out=out(q), k=past, k_out=out(past)) == S.INVALID_VIEW
    # the other heads of a buffer twice as wide, which is not in place
    wide = lambda at: view(0, [d, h, t, 1], nb=[4, 4 * d, 8 * d * h, 8 * d * h * t], offset=at)  # noqa: E731
    assert ask(rec, q=wide(0), q_out=out(wide(4 * d * h))) == S.OK
    assert ask(rec, q=wide(0), q_out=out(wide(4 * d * h - 4))) == ask(rec, q=wide(0), q_out=out(wide(4 * d * h + 4))) == S.INVALID_VIEW


@pytest.mark.parametrize("sections,own,want", [
    ([3, 1, 2], False, [(0, 0, 6), (1, 1, 6), (2, 2, 6), (0, 3, 6), (2, 4, 6), (0, 5, 6)]),
    ([0, 2, 2, 0], True, [(1, 0, 2), (2, 0, 2), (1, 1, 2), (2, 1, 2)])])
def test_pairs_taken_in_turn(sections, own, want):
    assert pairs_of(sections, True, own) == want


def test_shapes_that_take_vectors(rec):
    def vec(dim=64, sections=(32,), **kw):
        got, = rec.launches(eh.OpRope(view(0, [dim, 6, 5, 1], **kw), view(1, [dim, 6, 5, 1], mut=True), view(4, [5, len(sections), 1, 1], dtype=I32), list(sections)))
        return "k_rope<true" in got.name

    assert vec() and vec(80, (20, 20)) and vec(96, (16, 16, 8)) and vec(96, (20, 7, 17))
    assert not vec(80, (33,)) and not vec(66, (32,)) and not vec(nb=[8, 544, 3264, 16320])


def test_every_head_is_in_some_step(rec):
    for dim, heads, tokens in ((2, 1000, 3), (1024, 5, 1), (4096, 3, 7), (1 << 24, 1, 1), (6, 1, 100000)):
        got, = rec.launches(eh.OpRope(view(0, [dim, heads, tokens, 1]), view(1, [dim, heads, tokens, 1], mut=True), view(4, [tokens, 1, 1, 1], dtype=I32), [1]))
        assert got.block == 256 and got.grid > 0


@pytest.mark.parametrize("dim,tokens,launches", [(64, 100000, 1), (64, (1 << 31) - 1, 16), (2048, (1 << 22) + 1, 2)])
def test_very_many_tokens_run_in_parts(rec, dim, tokens, launches):
    """A launch counts its threads in 32 bits."""
    big = lambda at, mut=False: (eh.TensorViewMut if mut else eh.TensorView)(at << 58, eh.Layout.dense(eh.DType.F32, [dim, 1, tokens, 1]), 1 << 57)  # noqa: E731
    got = rec.launches(eh.OpRope(big(1), big(2, True), view(4, [tokens, 1, 1, 1], dtype=I32), [dim // 2]))
    assert len(got) == launches and all(g.grid * g.block < 1 << 32 for g in got)
