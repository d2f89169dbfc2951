"""CPU: what a packed paged cache refuses, what it launches, and the definition of its rows."""
import ctypes
import re

import numpy as np
import pytest

import emel_hip as eh
from helpers import rng
from launch_recorder import Recorder
from packed_cache_reference import SIZE, decode, encode, random_rows

S, F32, F16, BF16, I32, Q4_0, Q8_0, Q4_K = eh.Status, eh.DType.F32, eh.DType.F16, eh.DType.BF16, eh.DType.I32, eh.DType.Q4_0, eh.DType.Q8_0, eh.DType.Q4_K


@pytest.fixture(scope="module")
def rec():
    return Recorder()


def v(slot, ne, dtype=F32, nb=None, mut=False, offset=0, size=1 << 43):
    packed = dtype in (Q4_0, Q8_0, Q4_K)
    lay = eh.Layout(dtype, ne, nb) if nb else eh.Layout.packed(dtype, ne) if packed else eh.Layout.dense(dtype, ne)
    return (eh.TensorViewMut if mut else eh.TensorView)((slot + 1) * (1 << 43) + offset, lay, size)


def status(rec, event):
    rec.lib.record_clear()
    got = S(event._call(rec.lib, None))
    assert (rec.lib.record_count() > 0) == (got == S.OK)
    return got


D, H, P, N, T = 64, 2, 16, 9, 5


def pool(slot, dtype, dim=D, **kw):
    return v(slot, [dim, P, H, N], dtype, **kw)


@pytest.mark.parametrize("kd", [Q4_0, Q8_0])
@pytest.mark.parametrize("vd", [Q4_0, Q8_0])
def test_append_and_read_refusals(rec, kd, vd):
    sources = dict(k=v(0, [D, H, T, 1]), v=v(1, [D, H, T, 1]), slots=v(2, [T, 1, 1, 1], I32))

    def append(**other):
        return status(rec, eh.OpPagedKvAppend(**{**sources, "k_pages": pool(3, kd, mut=True), "v_pages": pool(4, vd, mut=True), **other}))

    outs = dict(k=v(0, [D, H, T, 1], mut=True), v=v(1, [D, H, T, 1], mut=True), slots=v(2, [T, 1, 1, 1], I32))

    def read(**other):
        return status(rec, eh.OpPagedKvRead(**{**outs, "k_pages": pool(3, kd), "v_pages": pool(4, vd), **other}))

    for ask, mut in ((append, True), (read, False)):
        assert ask() == S.OK
        for name in ("k", "v", "slots", "k_pages", "v_pages"):
            assert ask(**{name: None}) == S.INVALID_ARGUMENT
        assert ask(k_pages=pool(3, kd, mut=mut, offset=1)) == ask(slots=v(2, [T, 1, 1, 1], I32, offset=2)) == S.INVALID_ARGUMENT
        assert ask(k_pages=pool(3, F32, mut=mut)) == ask(k_pages=v(3, [256, P, H, N], Q4_K, mut=mut)) == S.INVALID_VIEW
        row = D // 32 * SIZE["q8_0" if kd == Q8_0 else "q4_0"]
        nb = [1, row, row * P, row * P * H]
        assert ask(k_pages=pool(3, kd, mut=mut, nb=nb, size=row * P * H * N)) == S.OK
        assert ask(k_pages=pool(3, kd, mut=mut, nb=nb, size=row * P * H * N - 1)) == ask(k_pages=pool(3, kd, mut=mut, nb=[2] + nb[1:])) == S.INVALID_VIEW
        assert ask(k_pages=pool(3, kd, mut=mut, nb=[1, row + 1] + nb[2:])) == ask(k_pages=pool(3, kd, mut=mut, dim=48, nb=nb)) == S.INVALID_VIEW
        assert ask(v_pages=pool(4, F16, mut=mut)) == ask(v_pages=pool(4, vd, dim=96, mut=mut)) == ask(v_pages=v(4, [D, P, H, N + 1], vd, mut=mut)) == S.SHAPE_MISMATCH
        assert ask(k=v(0, [D, H + 1, T, 1], mut=not mut)) == ask(v=v(1, [D, H, T + 1, 1], mut=not mut)) == ask(slots=v(2, [T + 1, 1, 1, 1], I32)) == S.SHAPE_MISMATCH
        assert ask(k=v(3, [D, H, T, 1], mut=not mut)) == ask(v=v(4, [D, H, T, 1], mut=not mut, offset=64)) == S.INVALID_VIEW
        assert ask(slots=v(2, [1 << 31, 1, 1, 1], I32)) == S.UNSUPPORTED_OPERATION
        wide = lambda t: v(3 + t, [1 << 13, 1, (1 << 13) + 1, 1], (kd, vd)[t], mut=mut)  # noqa: E731
        flat = lambda t: v(t, [1 << 13, (1 << 13) + 1, 1, 1], mut=not mut)  # noqa: E731
        assert ask(k=flat(0), v=flat(1), slots=v(2, [1, 1, 1, 1], I32), k_pages=wide(0), v_pages=wide(1)) == S.UNSUPPORTED_OPERATION
    assert append(v_pages=eh.TensorViewMut(4 * (1 << 43), eh.Layout.packed(kd, [D, P, H, N]), 1 << 43)) == S.INVALID_VIEW
    assert append(slots=v(4, [T, 1, 1, 1], I32, offset=64)) == append(k_pages=pool(3, kd, mut=True, nb=[1, row - 2] + nb[2:])) == S.INVALID_VIEW
    assert read(v=v(0, [D, H, T, 1], mut=True)) == read(k=v(2, [D, H, T, 1], mut=True)) == read(k=v(0, [D, H, T, 1], nb=[4, 4, 4 * D, 4 * D * T], mut=True)) == S.INVALID_VIEW
    # keys and values of a token side by side
    kv_nb = [4, 4 * D, 8 * D * H, 8 * D * H * T]
    assert read(k=v(0, [D, H, T, 1], nb=kv_nb, mut=True), v=v(0, [D, H, T, 1], nb=kv_nb, mut=True, offset=4 * D * H)) == S.OK
    assert read(k=v(0, [D, H, T, 1], nb=kv_nb, mut=True), v=v(0, [D, H, T, 1], nb=kv_nb, mut=True, offset=4 * D * H - 4)) == S.INVALID_VIEW


@pytest.mark.parametrize("kd,vd", [(Q8_0, Q4_0), (Q4_0, Q8_0), (Q4_0, Q4_0)])
def test_pools_interleaved_in_one_allocation(rec, kd, vd):
    kr, vr = (D // 32 * (34 if t == Q8_0 else 18) for t in (kd, vd))
    step = kr + vr
    nb = [1, step, step * P, step * P * H]

    def side(at, stride=step):
        n = [1, stride, stride * P, stride * P * H]
        return status(rec, eh.OpPagedKvAppend(v(0, [D, H, T, 1]), v(1, [D, H, T, 1]), v(2, [T, 1, 1, 1], I32), pool(3, kd, nb=n, mut=True), pool(3, vd, nb=n, mut=True, offset=at)))

    assert side(kr) == S.OK and side(kr - 2) == side(kr, step - 2) == side(kr + 2) == S.INVALID_VIEW
    assert side(kr + 2, step + 2) == S.OK
    low = status(rec, eh.OpPagedKvAppend(v(0, [D, H, T, 1]), v(1, [D, H, T, 1]), v(2, [T, 1, 1, 1], I32), pool(3, kd, nb=nb, mut=True, offset=vr), pool(3, vd, nb=nb, mut=True)))
    assert low == S.OK


def test_attention_refusals(rec):
    h, s = 6, 5
    parts = dict(q=v(0, [D, h, s, 1]), k_pages=pool(1, Q8_0), v_pages=pool(2, Q4_0), page_table=v(3, [7, s, 1, 1], I32), lengths=v(4, [s, 1, 1, 1], I32),
                 output=v(5, [D, h, s, 1], mut=True), scale=0.1)

    def ask(**other):
        return status(rec, eh.OpPagedAttention(**{**parts, **other}))

    assert ask() == ask(v_pages=pool(2, Q8_0)) == ask(k_pages=pool(1, Q4_0)) == S.OK
    assert ask(k_pages=pool(1, F16)) == ask(v_pages=pool(2, BF16)) == S.SHAPE_MISMATCH
    assert ask(k_pages=pool(1, Q4_0, dim=48, nb=[1, 64, 1024, 2048])) == S.INVALID_VIEW
    wide = lambda slot, t: v(slot, [288, P, H, N], t)  # noqa: E731
    assert ask(q=v(0, [288, h, s, 1]), k_pages=wide(1, Q8_0), v_pages=wide(2, Q4_0), output=v(5, [288, h, s, 1], mut=True)) == S.UNSUPPORTED_OPERATION
    assert ask(output=v(1, [D, h, s, 1], mut=True)) == ask(output=v(2, [D, h, s, 1], mut=True)) == S.INVALID_VIEW


def test_halves_are_read_too(rec):
    for kind, dim, kernel in ((F16, 64, "k_pa_read<true>"), (BF16, 20, "k_pa_read<false>"), (F16, 256, "k_pa_read_wide")):
        event = eh.OpPagedKvRead(v(3, [dim, P, H, N], kind), v(4, [dim, P, H, N], kind), v(2, [T, 1, 1, 1], I32), v(0, [dim, H, T, 1], mut=True), v(1, [dim, H, T, 1], mut=True))
        got, = rec.launches(event)
        assert kernel in got.name
    mixed = eh.OpPagedKvRead(pool(3, F16), pool(4, BF16), v(2, [T, 1, 1, 1], I32), v(0, [D, H, T, 1], mut=True), v(1, [D, H, T, 1], mut=True))
    assert status(rec, mixed) == S.SHAPE_MISMATCH


@pytest.mark.parametrize("tokens,launches", [(1, 1), (1 << 17, 1), (1 << 25, 1), ((1 << 25) + 1, 2), ((1 << 31) - 1, 64)])
def test_reads_of_many_tokens_run_in_parts(rec, tokens, launches):
    """A launch counts its threads in 32 bits."""
    event = eh.OpPagedKvRead(v(3, [32, 16, 1, 9000], Q4_0), v(4, [32, 16, 1, 9000], Q8_0), v(2, [tokens, 1, 1, 1], I32), v(0, [32, 1, tokens, 1], mut=True, size=1 << 50),
                             eh.TensorViewMut(1 << 60, eh.Layout.dense(F32, [32, 1, tokens, 1]), 1 << 50))
    got = rec.launches(event)
    assert len(got) == launches and all(g.grid * g.block < 1 << 32 for g in got)


@pytest.mark.parametrize("items", [1, 4, 16])
def test_wide_tokens_share_a_workgroups_waves(rec, items):
    for dim, kv, tokens in ((128, items, 5000), (256, items, 3)):
        event = eh.OpPagedKvAppend(v(0, [dim, kv, tokens, 1]), v(1, [dim, kv, tokens, 1]), v(2, [tokens, 1, 1, 1], I32), v(3, [dim, 16, kv, 900], Q4_0, mut=True),
                                   v(4, [dim, 16, kv, 900], Q8_0, mut=True))
        got, = rec.launches(event)
        assert ("wide" in got.name) == (dim // 8 * kv >= 64) and got.grid == (-(-tokens // 8) if tokens >= 2048 else tokens)


@pytest.mark.parametrize("tokens,launches", [(1, 1), (1 << 17, 1), ((1 << 17) + 1, 2)])
def test_appends_of_many_tokens_run_in_parts(rec, tokens, launches):
    event = eh.OpPagedKvAppend(v(0, [32, 1, tokens, 1]), v(1, [32, 1, tokens, 1]), v(2, [tokens, 1, 1, 1], I32), v(3, [32, 16, 1, 9000], Q4_0, mut=True),
                               v(4, [32, 16, 1, 9000], Q8_0, mut=True))
    assert len(rec.launches(event)) == launches


@pytest.mark.parametrize("kind,low,high", [("q8_0", -127, 127), ("q4_0", -8, 7)])
def test_the_definition_of_a_row(kind, low, high):
    """Nearest numbers to the stored scale, within half of it, by comparison with every other number."""
    x = (rng(1).standard_normal((40, 96)) * np.exp(3 * rng(2).standard_normal((40, 1)))).astype(np.float32)
    x[0, :32], x[1, 40] = 0, 60000
    rows = encode(kind, x)
    d = rows[:, -6:].copy().view(np.float16).astype(np.float64)
    got = decode(kind, rows).reshape(40, 3, 32)
    all_of = d[..., None, None] * np.arange(low, high + 1)  # [row, block, 1, number]
    best = np.abs(all_of - x.astype(np.float64).reshape(40, 3, 32, 1)).min(3)
    assert np.array_equal(np.abs(got - x.reshape(40, 3, 32)), best)
    size = np.abs(x.reshape(40, 3, 32)).max(2)
    # the largest value becomes the end of the scale, but for f16's rounding of it
    end = np.abs(got).max(2)
    assert (np.abs(end - size) <= size * 2.0**-11 + 127 * 2.0**-25 + np.abs(d) * 0.5 * (kind == "q8_0")).all()


@pytest.mark.parametrize("kind", ["q8_0", "q4_0"])
def test_rows_come_back_as_they_were(kind):
    """Packing a row's own values gives the same values, as every block of them holds its scale's end."""
    rows = random_rows(5, kind, 60, 64)
    if kind == "q8_0":
        rows[:, 0], rows[:, 8] = 127, 129
    else:
        rows[:, 0] &= 0xF0
        rows[:, 4] &= 0x0F
    d = np.abs(rows[:, -4:].copy().view(np.float16))
    rows[:, -4:] = np.where(d < 0.002, np.float16(0.002), d).view(np.uint8)
    want = decode(kind, rows)
    assert np.array_equal(decode(kind, encode(kind, want.astype(np.float32))), want)


@pytest.mark.parametrize("kd,vd", [(Q8_0, Q8_0), (Q8_0, Q4_0), (Q4_0, Q8_0), (Q4_0, Q4_0)])
@pytest.mark.parametrize("dim", range(32, 257, 32))
def test_attentions_lds_is_its_kernels(rec, kd, vd, dim):
    """The launch's LDS holds what the kernel that it picks lays out there, by the columns a head that its name gives: score
    operands of each set of blocks, the waves' parts of a head's values, and a weight for each part of a row."""
    for group in list(range(1, 18)) + [31, 32, 33, 48]:
        for kv, s in ((1, 3), (8, 70)):
            heads = group * kv
            event = eh.OpPagedAttention(v(0, [dim, heads, s, 1]), v(1, [dim, 16, kv, 900], kd), v(2, [dim, 16, kv, 900], vd), v(3, [7, s, 1, 1], I32), v(4, [s, 1, 1, 1], I32),
                                        v(5, [dim, heads, s, 1], mut=True), scale=0.1)
            got, = rec.launches(event)
            blocks, values, fold = (int(n) for n in re.search(r"k_pa_attn<.*, (\d+), (\d+), (\d+)>", got.name).groups())
            assert 32 * blocks == dim and values == 2 * blocks
            shared = min(group, 16)
            assert shared * fold <= 16 and (fold == 1 or fold < 2 * blocks)
            operands, parts = -(-blocks // fold) * 2 * 65 * 16, 4 * 4 * shared * (dim + 4)
            assert got.lds >= max(operands, parts) and got.lds + 4096 + 1024 * blocks <= 160 * 1024 and got.grid % 256 == 0


@pytest.mark.parametrize("group", [1 << 28, (1 << 28) + 1, 1 << 29, (1 << 29) + 2, 3 << 29, (1 << 31) - 1])
def test_any_number_of_heads_to_a_cache_head(rec, group):
    """Sixteen heads of a row leave each one column, however many groups of sixteen there are."""
    event = eh.OpPagedAttention(v(0, [256, group, 1, 1]), v(1, [256, 16, 1, 9], Q8_0), v(2, [256, 16, 1, 9], Q4_0), v(3, [1, 1, 1, 1], I32), v(4, [1, 1, 1, 1], I32),
                                v(5, [256, group, 1, 1], mut=True), scale=0.1)
    got, = rec.launches(event)
    assert re.search(r"k_pa_attn<.*, 8, 16, 1>", got.name), got.name
