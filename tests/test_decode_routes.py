"""CPU: which kernels the served-token operators launch, and in how many launches; nothing runs."""
import re

import pytest

import emel_hip as eh
from launch_recorder import Recorder, view

F16, BF16, I32, Q4_0, Q4_K = eh.DType.F16, eh.DType.BF16, eh.DType.I32, eh.DType.Q4_0, eh.DType.Q4_K


@pytest.fixture(scope="module")
def rec():
    return Recorder()


def kernels(got):
    return [re.search(r"k_\w+", g.name).group() for g in got]


def product(rec, k, m, n, q4k=False, nb=None):
    w = eh.TensorView(1 << 43, eh.Layout.packed(Q4_K if q4k else Q4_0, [k, m, 1, 1]), 1 << 62)
    return rec.launches((eh.OpMulMatQ4K if q4k else eh.OpMulMatQ4_0)(w, view(1, [k, n, 1, 1]), view(2, [m, n, 1, 1], mut=True)))


@pytest.mark.parametrize("q4k", [False, True])
@pytest.mark.parametrize("n,fits,alone", [(1, 18688, 26112), (2, 8704, 12544), (3, 5376, 7936), (4, 3840, 5632)])
def test_up_to_four_columns_are_digits_where_they_fit(rec, q4k, n, fits, alone):
    digits, halves = ["k_qm_digits"], ["k_qm_halves", "k_qm_sum"]
    for m, k in ((11008, fits), (4096, alone)):  # two workgroups a compute unit, or one with a tile to each
        assert kernels(product(rec, k, m, n, q4k)) == digits
        assert kernels(product(rec, k + 256, m, n, q4k)) == halves
    assert kernels(product(rec, 256, 4096, n + 4, q4k)) == halves


@pytest.mark.parametrize("k,m,n,launches", [
    (64, 33, 1 << 16, 1), (64, 33, (1 << 16) + 5, 2), (64, 33, 1 << 21, 32),  # columns, by a grid's second axis
    (4096, 11008, 64, 1), (4096, 11008, 2000, 2), (4096, 151936, 64, 1), (4096, 151936, 102, 2),  # by the partial sums' 256 MB
    (32, 1 << 22, 16, 1), (32, (1 << 22) + 1, 16, 2), (11008, 1 << 22, 32, 24), (1 << 26, 300, 5, 3)])  # rows
def test_large_products_run_in_parts(rec, k, m, n, launches):
    assert kernels(product(rec, k, m, n)) == ["k_qm_halves", "k_qm_sum"] * launches


def test_columns_left_over_are_digits(rec):
    assert kernels(product(rec, 64, 33, (1 << 16) + 2)) == ["k_qm_halves", "k_qm_sum", "k_qm_digits"]


@pytest.mark.parametrize("k,m,n,lds,grid", [
    (4096, 151936, 5, 4, 4 * 128), (4096, 40000, 16, 4, 4 * 128),  # four units a chunk, two workgroups a compute unit
    (4096, 11008, 15, 2, 8 * 32), (4096, 4096, 8, 2, 8 * 32),       # two, and one
    (1024, 2000, 12, 1, 4 * 16), (256, 16, 5, 1, 1)])               # where that leaves compute units idle
def test_chunks_of_many_columns(rec, k, m, n, lds, grid):
    halves = product(rec, k, m, n)[0]
    assert (halves.lds, halves.grid) == (lds * 17472, grid)


@pytest.mark.parametrize("dim,strided", [(64, False), (60, False), (64, True)])
def test_append_takes_eight_tokens_a_workgroup_of_many(rec, dim, strided):
    for tokens, per in ((1, 1), (2047, 1), (2048, 8), (100001, 8)):
        kv = [view(i, [dim, 2, tokens, 1], [8, 8 * dim, 16 * dim, 16 * dim * tokens] if strided else None) for i in (0, 1)]
        pools = [view(i, [dim, 16, 2, 9000], dtype=F16, mut=True) for i in (2, 3)]
        got, = rec.launches(eh.OpPagedKvAppend(*kv, view(4, [tokens, 1, 1, 1], dtype=I32), *pools))
        assert f", {per}u," in got.name and got.grid == -(-tokens // per)
        assert ("true>" in got.name) == (dim % 8 == 0 and not strided)


def attention(rec, seqs, max_pages, page=16, kv=2, heads=6, dim=64):
    pools = [view(i, [dim, page, kv, 9], dtype=BF16) for i in (0, 1)]
    return rec.launches(eh.OpPagedAttention(view(2, [dim, heads, seqs, 1]), *pools, view(3, [max_pages, seqs, 1, 1], dtype=I32),
                                            view(4, [seqs, 1, 1, 1], dtype=I32), view(5, [dim, heads, seqs, 1], mut=True), scale=0.1))


def test_attention_runs_in_one_launch_of_what_fits_at_once(rec):
    grids = {attention(rec, seqs, 100, dim=dim)[0].grid for seqs in (1, 64, 1000) for dim in (64,)}
    assert len(grids) == 1
    assert len(attention(rec, 1000, 100)) == 1


def test_attention_with_more_units_than_are_counted_runs_in_parts(rec):
    # 2^22 tokens at most: 2^15 + 1 units a sequence and cache head
    assert len(attention(rec, 32000, 1 << 18)) == 1
    assert len(attention(rec, 33000, 1 << 18)) == 2
    assert len(attention(rec, 1100, 1 << 14, page=256, kv=64, heads=64, dim=8)) == 2
    assert len(attention(rec, 70, (1 << 27) - 1, kv=127, heads=127)) == 70
    with pytest.raises(RuntimeError, match="UNSUPPORTED_OPERATION"):
        attention(rec, 1, (1 << 27) - 1, kv=128, heads=128)


def test_append_with_too_wide_tokens_is_refused(rec):
    ask = lambda dim, kv: rec.launches(eh.OpPagedKvAppend(  # noqa: E731
        view(0, [dim, kv, 1, 1]), view(1, [dim, kv, 1, 1]), view(2, [1, 1, 1, 1], dtype=I32), *(view(i, [dim, 1, kv, 1], dtype=F16, mut=True) for i in (3, 4))))
    assert len(ask(1 << 13, 1 << 13)) == 1
    with pytest.raises(RuntimeError, match="UNSUPPORTED_OPERATION"):
        ask(1 << 13, (1 << 13) + 1)


@pytest.mark.parametrize("history,biases,packed", [(65535, 65534, True), (65536, 1, False), (1, 65535, False)])
def test_logits_counts_and_entries_share_a_word_where_they_fit(rec, history, biases, packed):
    t = lambda slot, ne, dtype=I32: view(slot, ne, dtype=dtype)  # noqa: E731
    got, = rec.launches(eh.OpLogitsAdjust(view(0, [1000, 2, 1, 1]), view(1, [1000, 2, 1, 1], mut=True), history=t(2, [history, 2, 1, 1]),
                                          bias_ids=t(3, [biases, 2, 1, 1]), bias=t(4, [biases, 2, 1, 1], eh.DType.F32)))
    assert ("u, true, true, false>" in got.name) == packed


def test_logits_rows_out_of_step_are_not_read_by_fours(rec):
    def vec(nb_x, nb_y, rows=3, at=0):
        got, = rec.launches(eh.OpLogitsAdjust(view(0, [1000, rows, 1, 1], nb_x), view(1, [1000, rows, 1, 1], nb_y, mut=True, offset=at)))
        return re.search(r"k_la_adjust<\w+, \w+, (\w+), false", got.name).group(1) == "true"

    dense = [4, 4000, 12000, 12000]
    assert vec(None, None) and vec(dense, [4, 4016, 12048, 12048]) and vec(None, None, rows=1)
    assert not vec(dense, [4, 4004, 12012, 12012]) and not vec([8, 8000, 24000, 24000], None) and not vec(None, None, at=4)


@pytest.mark.parametrize("card,rows,tokens", [(151936, 13, 1024), (151936, 14, 4096), (1 << 21, 1, 1024), ((1 << 21) + 1, 1, 4096), (5, 1000, 1024)])
def test_logits_that_run_at_once_take_shorter_runs(rec, card, rows, tokens):
    got, = rec.launches(eh.OpLogitsAdjust(view(0, [card, rows, 1, 1]), view(1, [card, rows, 1, 1], mut=True)))
    assert f"k_la_adjust<{tokens // 1024}u," in got.name
