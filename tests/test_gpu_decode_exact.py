"""GPU: the served-token operators on cases whose result is exact."""
import numpy as np
import pytest

import emel_hip as eh
from decode_exact import (POWER, cancelling, cancelling_attention, exact_product, exact_rows, exact_scale, flat_means_differ, flat_values,
                          outlier_columns, whole_columns)
from decode_reference import attention as reference
from decode_reference import out, packed, view
from helpers import rng

pytestmark = pytest.mark.gpu

EVENT = {"q4_0": eh.OpMulMatQ4_0, "q4_k": eh.OpMulMatQ4K}


def run(event):
    status = eh.Kernel().process_event(event)
    assert status == eh.Status.OK, eh.last_error()


def product(gpu, form, rows, x):
    import torch

    (n, k), m = x.shape, len(rows)
    y = torch.full((n, m), 7.0, device=gpu)
    run(EVENT[form](packed(torch.from_numpy(rows).to(gpu), form, k, m), view(torch.from_numpy(x).to(gpu)), out(y)))
    return y.cpu().numpy()


@pytest.mark.parametrize("form,k", [("q4_0", 64), ("q4_0", 4128), ("q4_0", 3840), ("q4_k", 256), ("q4_k", 3840)])
@pytest.mark.parametrize("n", [1, 2, 3, 4])
@pytest.mark.parametrize("big", [2.0**-3, 1.0, 2.0**12, 2.0**20, 2.0**30, 2.0**40])
def test_product_beside_values_that_tower_over_the_rest(gpu, form, k, n, big):
    """Values that meet zero weights take nothing from the precision of the others."""
    x, at = outlier_columns(k + n, k, n, big)
    rows = exact_rows(n, form, k, 70, at)
    got = product(gpu, form, rows, x)
    assert np.array_equal(got, exact_product(form, rows, x, 2.0**-14))


@pytest.mark.parametrize("form", ["q4_0", "q4_k"])
@pytest.mark.parametrize("m,n", [(17000, 1), (9001, 3), (40000, 4)])
def test_product_of_many_rows_beside_towering_values(gpu, form, m, n):
    x, at = outlier_columns(m, 512, n, 2.0**18)
    rows = exact_rows(n, form, 512, m, at)
    assert np.array_equal(product(gpu, form, rows, x), exact_product(form, rows, x, 2.0**-14))


@pytest.mark.parametrize("form", ["q4_0", "q4_k"])
def test_product_with_one_towering_and_one_infinite_column(gpu, form):
    x, at = outlier_columns(5, 1024, 3, 2.0**25)
    rows = exact_rows(6, form, 1024, 90, at)
    want = exact_product(form, rows, x, 2.0**-14)
    x[1, 77], x[2, 900] = np.inf, np.nan
    got = product(gpu, form, rows, x)
    assert np.array_equal(got[0], want[0]) and np.isnan(got[2]).all()
    plain = exact_product(form, rows[:, :], np.where(np.arange(1024) == 77, 1, 0)[None].astype(np.float32))[0]
    assert np.array_equal(np.isnan(got[1]), plain == 0)
    assert np.array_equal(got[1][plain != 0], np.sign(plain[plain != 0]) * np.inf)


@pytest.mark.parametrize("k,n", [(1 << 26, 16), (1 << 26, 1), (3 << 24, 11)])
def test_product_of_the_longest_rows(gpu, k, n):
    """Rows so long that a part of the product has fewer tiles than a workgroup has waves."""
    import torch

    m, g = 70, torch.Generator(gpu).manual_seed(k + n)
    w = torch.randint(0, 256, (m, k // 32, 18), dtype=torch.uint8, device=gpu, generator=g)
    w[:, :, 0], w[:, :, 1] = 0x00, 0x24  # the f16 2^-6
    at = torch.randint(0, k, (4000,), device=gpu, generator=g)
    at[:3] = torch.tensor([0, k - 1, k // 2], device=gpu)
    at = at.unique()
    x = torch.zeros(n, k, device=gpu)
    x[:, at] = torch.randint(-400, 401, (n, at.numel()), device=gpu, generator=g).float()
    y = torch.full((n, m), 7.0, device=gpu)
    run(eh.OpMulMatQ4_0(packed(w, "q4_0", k, m), view(x), out(y)))
    byte = w[:, at // 32, 2 + at % 16].int()
    q = torch.where(at % 32 < 16, byte & 15, byte >> 4) - 8
    want = x[:, at].double() @ q.double().t().contiguous() / 64
    assert (x[:, at].abs().double() @ q.abs().double().t().contiguous()).max() < 2**23
    assert torch.equal(y.double(), want)


@pytest.mark.parametrize("tokens", [(1 << 17) - 1, (1 << 17) + 1, (1 << 17) + 3000, (1 << 18) + 9])
def test_append_of_more_tokens_than_a_launch_takes(gpu, tokens):
    """Slots named again within a launch and by later ones: the last token is stored, whichever launch has it."""
    import torch

    pages, page, dim = 500, 100, 8
    g = rng(tokens)
    slots = g.integers(-5, pages * page + 5, tokens).astype(np.int32)
    slots[[3, 70000, tokens - 1]] = 77
    k = torch.arange(tokens, device=gpu, dtype=torch.int32)[:, None, None].expand(tokens, 1, dim).contiguous()
    k = k % 2039 + torch.arange(dim, device=gpu)  # whole numbers that f16 holds
    v = (k // 7 - 100).float()
    pool = torch.full((2, pages, 1, page, dim), -5.0, device=gpu, dtype=torch.float16)
    run(eh.OpPagedKvAppend(view(k.float()), view(v), view(torch.from_numpy(slots).to(gpu)), out(pool[0]), out(pool[1])))
    last = np.full(pages * page, -1)
    live = np.flatnonzero((slots >= 0) & (slots < pages * page))
    last[slots[live]] = live  # numpy stores the last of equal indices
    at = torch.from_numpy(last).to(gpu)
    for got, src in zip(pool.view(2, pages * page, dim), (k[:, 0].half(), v[:, 0].half())):
        assert torch.equal(got, torch.where((at < 0)[:, None], torch.full_like(got, -5.0), src[at.clamp(min=0)]))


def attention(gpu, kind, q, k, v, lengths, scale=0.0, page=16, **more):
    """The operator over keys and values [seqs, kv_heads, positions, dim] put into pages in a mixed order."""
    import torch

    seqs, kv, most, dim = k.shape
    per = -(-most // page)
    ids = torch.from_numpy(rng(most).permutation(seqs * per)).to(gpu)
    pools = []
    for src in (k, v):
        pad = torch.zeros(seqs, kv, per * page, dim, device=gpu, dtype=kind)
        pad[:, :, :most] = src.to(kind)
        pool = torch.empty(seqs * per, kv, page, dim, device=gpu, dtype=kind)
        pool[ids] = pad.view(seqs, kv, per, page, dim).transpose(1, 2).reshape(seqs * per, kv, page, dim)
        pools.append(pool)
    y = torch.full(q.shape, 7.0, device=gpu)
    run(eh.OpPagedAttention(view(q), view(pools[0]), view(pools[1]), view(ids.view(seqs, per).int()), view(torch.tensor(lengths, dtype=torch.int32, device=gpu)),
                            out(y), scale=scale, **more))
    return y


@pytest.mark.parametrize("lengths", [[2, 5, 40], [300, 1, 4000], [20000, 3, 33]])
@pytest.mark.parametrize("dim", [8, 128, 256])
def test_attention_of_values_whose_sum_overflows(gpu, dim, lengths):
    """The mean of values near bf16's largest is finite, though their sum is not; the means are exact (flat scores)."""
    import torch

    seqs, kv, heads, most = 3, 2, 4, max(lengths)
    v = torch.full((seqs, kv, most, dim), 3 * 2.0**126, device=gpu)  # three quarters of the largest power of two
    v[:, :, :, 1::2] = -(2.0**127)
    v[:, 1, 1::2, 2::4] = 0.0  # every other position
    v[2] = 2.0**-60
    q = torch.ones(seqs, heads, dim, device=gpu)
    got = attention(gpu, torch.bfloat16, q, v[:, :, :, :] * 0, v, lengths).double().cpu()
    for s, n in enumerate(lengths):
        want = v[s, :, :n].double().mean(1).repeat_interleave(heads // kv, 0).cpu()
        # a product with the reciprocal of a sum, each off by half a step, and the join's weighted parts
        assert (abs(got[s] - want) <= abs(want) * 2.0**-21).all(), (s, n)


@pytest.mark.parametrize("where", [0, 1999])
def test_attention_of_one_value_that_overflows_beside_small_ones(gpu, where):
    """Waves with huge sums and others are joined at one scale."""
    import torch

    v = torch.ones(1, 1, 2000, 64, device=gpu)
    v[0, 0, where] = 2.0**127
    v[0, 0, where - 1, 5] = -(2.0**127)
    got = attention(gpu, torch.bfloat16, torch.ones(1, 4, 64, device=gpu), v * 0, v, [2000]).double().cpu()
    want = v[0, 0].double().mean(0).cpu().expand(4, 64)
    assert (abs(got[0] - want) <= abs(v[0, 0].double()).mean(0).cpu() * 2.0**-21).all()


@pytest.mark.parametrize("form", ["q4_0", "q4_k"])
@pytest.mark.parametrize("n,idle", [(1, [0]), (3, [1]), (4, [0, 3]), (15, [14]), (16, [2, 3, 7]), (33, [0, 16, 32])])
def test_product_beside_columns_that_nobody_filled(gpu, form, n, idle):
    """Columns of NaN, or with one, are NaN in every row, whatever weights they meet; the others are as without them."""
    x = whole_columns(n, form, 1024, n)
    rows = exact_rows(n, form, 1024, 200)
    want = exact_product(form, rows, x)
    for i, c in enumerate(idle):
        x[c, :: 1 if i % 2 == 0 else 1024] = np.nan
        want[c] = np.nan
    rows.reshape(200, -1, 18 if form == "q4_0" else 144)[7, 0, :2] = np.array([np.inf], np.float16).view(np.uint8)
    got = product(gpu, form, rows, x)
    assert np.isnan(got[idle]).all()
    rest = [c for c in range(n) if c not in idle]
    got, want = np.delete(got[rest], 7, 1), np.delete(want[rest], 7, 1)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (20, 1, 72), (3, 3, 8), (4, 2, 256)])
def test_attention_beside_queries_that_nobody_filled(gpu, bf16, heads, kv, dim):
    """A head whose query holds a NaN is NaN, unless its sequence is empty; the others are as without it."""
    import torch

    kind, lengths = (torch.bfloat16, torch.float16)[not bf16], [700, 0, 33, 5000, 1]
    g = torch.Generator(gpu).manual_seed(dim)
    v = torch.randint(-9, 10, (5, kv, 5000, dim), device=gpu, generator=g).float()
    q = torch.randn(5, heads, dim, device=gpu, generator=g)
    plain = attention(gpu, kind, q, v * 0, v, lengths, scale=1.0)
    q[0, heads - 1, dim - 1] = q[3, 0, 3] = q[4, 0] = float("nan")
    q[1] = float("nan")
    got = attention(gpu, kind, q, v * 0, v, lengths, scale=1.0)
    filled = ~q.isnan().any(2)
    filled[1] = True
    assert torch.equal(got[filled], plain[filled]) and got[~filled].isnan().all()
    assert (got[1] == 0).all()


@pytest.mark.parametrize("form,k", [("q4_0", 32), ("q4_0", 288), ("q4_0", 4096), ("q4_0", 4128), ("q4_0", 11008), ("q4_0", 18688), ("q4_0", 32768),
                                    ("q4_k", 256), ("q4_k", 1280), ("q4_k", 4096), ("q4_k", 11008), ("q4_k", 16384)])
@pytest.mark.parametrize("m,n", [(70, 1), (257, 2), (33, 3), (100, 4), (47, 5), (64, 13), (31, 16), (50, 33)])
def test_product_keeps_every_bit_of_whole_numbers(gpu, form, k, m, n):
    x, rows = whole_columns(k + n, form, k, n), exact_rows(m, form, k, m)
    assert np.array_equal(product(gpu, form, rows, x), exact_product(form, rows, x))


@pytest.mark.parametrize("form", ["q4_0", "q4_k"])
@pytest.mark.parametrize("m,n", [(40000, 1), (20000, 4), (40000, 7), (11008, 15), (9000, 64)])
def test_product_of_many_rows_keeps_every_bit(gpu, form, m, n):
    x, rows = whole_columns(m, form, 1024, n), exact_rows(n, form, 1024, m)
    assert np.array_equal(product(gpu, form, rows, x), exact_product(form, rows, x))


FLAT = [(1, 1, 64), (8, 1, 128), (17, 1, 8), (4, 2, 40), (6, 3, 104), (2, 1, 136), (5, 1, 200), (16, 1, 256), (32, 8, 128)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kv,dim", FLAT)
def test_attention_counts_every_position_once(gpu, bf16, heads, kv, dim):
    """Flat scores, values that name their positions: lengths around units, waves and the runs of workgroups."""
    import torch

    lengths = [1, 2, 31, 32, 33, 127, 128, 129, 255, 256, 257, 0, 500, 639, 641, 1500, 2047, 2049, 3000]
    v = flat_values(dim, len(lengths), kv, max(lengths), dim)
    q = torch.ones(len(lengths), heads, dim, device=gpu)
    vt = torch.from_numpy(v).to(gpu)
    for window in (0, 1, 32, 100, 1000):
        got = attention(gpu, (torch.float16, torch.bfloat16)[bf16], q, vt * 0, vt, lengths, scale=0.0, page=(24, 1, 16, 7, 256)[window % 5], window=window).cpu().numpy()
        for s, n in enumerate(lengths):
            if n:
                assert not flat_means_differ(got[s], v[s], n, window).any(), (n, window)
            else:
                assert (got[s] == 0).all()


@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 128), (1, 1, 64), (20, 1, 8), (4, 2, 256), (32, 8, 128), (3, 1, 96)])
@pytest.mark.parametrize("positions", [[8191], [12000, 1], [20000], [33000, 5, 129], [70001], [150000]])
def test_attention_counts_every_position_of_long_sequences_once(gpu, heads, kv, dim, positions):
    """As above, with rows of more than 64 parts."""
    import torch

    v = flat_values(positions[0] + dim, len(positions), kv, positions[0], dim)
    vt = torch.from_numpy(v).to(gpu)
    got = attention(gpu, torch.float16, torch.ones(len(positions), heads, dim, device=gpu), vt * 0, vt, positions, scale=0.0, page=64).cpu().numpy()
    for s, n in enumerate(positions):
        assert not flat_means_differ(got[s], v[s], n).any(), n


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("dim", list(range(8, 257, 8)))
def test_attention_keeps_every_part_of_queries_and_weights(gpu, bf16, dim):
    """Scores that are differences of large numbers in q, in every dim, over three positions and over some hundreds."""
    import torch

    heads, kv, most = 4, 2, dim + 200
    lengths = [3] * 24 + [dim + 9, most]
    cases = [cancelling(dim + s, kv, heads, most, dim) for s in range(len(lengths))]
    q, k, v = (torch.from_numpy(np.stack(t)).to(gpu) for t in zip(*cases))
    got = attention(gpu, (torch.float16, torch.bfloat16)[bf16], q, k, v, lengths, scale=exact_scale(POWER)).double().cpu().numpy()
    for s, n in enumerate(lengths):
        want, tol = cancelling_attention(*cases[s], n)
        assert (np.abs(got[s] - want) <= tol).all(), (n, (np.abs(got[s] - want) / np.maximum(tol, 1e-30)).max())


@pytest.mark.parametrize("dim", [8, 128, 256])
@pytest.mark.parametrize("size", [2.0**-24, 2.0**-20, 2.0**-17])
def test_attention_over_subnormal_halves(gpu, dim, size):
    """F16 values below 2^-14 count to 2^-38 of their weights, each instruction's largest: 2^-37 of the sum, at most."""
    import torch

    lengths, most = [1, 33, 700], 700
    g = rng(dim)
    k = g.standard_normal((3, 2, most, dim)).astype(np.float16)
    v = (g.integers(-7, 8, (3, 2, most, dim)) * size).astype(np.float16)
    q = g.standard_normal((3, 4, dim)).astype(np.float32)
    up = lambda t: torch.from_numpy(t.astype(np.float32)).to(gpu)  # noqa: E731
    got = attention(gpu, torch.float16, up(q), up(k), up(v), lengths, scale=dim**-0.5).double().cpu().numpy()
    for s, n in enumerate(lengths):
        want, tol = reference(q[s].astype(np.float64), *(t[s, :, :n].astype(np.float64).transpose(1, 0, 2) for t in (k, v)), dim**-0.5, 0.0)
        assert (np.abs(got[s] - want) <= tol + 2.0**-37).all(), (n, np.abs(got[s] - want).max())


@pytest.mark.parametrize("form", ["q4_0", "q4_k"])
@pytest.mark.parametrize("n", [1, 4, 9])
def test_a_captured_product_follows_its_columns(gpu, form, n):
    """What a replay finds in its columns decides how it goes: whole numbers, towering values, NaN, and whole numbers again."""
    import torch

    k, m = 1024, 300
    tower, at = outlier_columns(n, k, n, 2.0**20)
    rows = exact_rows(n, form, k, m, at)
    whole = whole_columns(n, form, k, n)
    plain = (whole, exact_product(form, rows, whole))
    empty = whole.copy()
    empty[n - 1] = np.nan
    with_empty = plain[1].copy()
    with_empty[n - 1] = np.nan
    w, x, y = torch.from_numpy(rows).to(gpu), torch.zeros(n, k, device=gpu), torch.zeros(n, m, device=gpu)
    stream = torch.cuda.Stream()
    kernel = eh.Kernel(stream.cuda_stream, synchronous=False)
    event = EVENT[form](packed(w, form, k, m), view(x), out(y))
    torch.cuda.synchronize()
    assert kernel.process_event(event) == eh.Status.OK  # sizes the stream's workspace
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        assert kernel.process_event(event) == eh.Status.OK
    steps = [plain, (empty, with_empty), plain, plain]
    if n <= 4:  # more columns keep 22 bits beside such values
        steps[1:1] = [(tower, exact_product(form, rows, tower, 2.0**-14)), plain]
    for values, want in steps:
        x.copy_(torch.from_numpy(values))
        y.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(y.cpu().numpy(), want, equal_nan=True)


def test_a_captured_append_of_several_launches_follows_its_slots(gpu):
    import torch

    tokens, pages, page, dim = (1 << 17) + 500, 40, 64, 8
    k = (torch.arange(tokens, device=gpu) % 2039).float()[:, None, None].expand(tokens, 1, dim).contiguous()
    slots = torch.zeros(tokens, dtype=torch.int32, device=gpu)
    pool = torch.zeros(2, pages, 1, page, dim, device=gpu, dtype=torch.bfloat16)
    stream = torch.cuda.Stream()
    kernel = eh.Kernel(stream.cuda_stream, synchronous=False)
    event = eh.OpPagedKvAppend(view(k), view(-k), view(slots), out(pool[0]), out(pool[1]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        assert kernel.process_event(event) == eh.Status.OK
    for seed in range(3):
        ids = rng(seed).integers(-9, pages * page, tokens).astype(np.int32)
        slots.copy_(torch.from_numpy(ids))
        pool.fill_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        last = np.full(pages * page, -1)
        last[ids[ids >= 0]] = np.flatnonzero(ids >= 0)
        want = torch.where(torch.from_numpy(last < 0).to(gpu)[:, None], torch.ones(1, device=gpu), k[torch.from_numpy(last).to(gpu).clamp(min=0), 0]).bfloat16()
        assert torch.equal(pool[0].view(-1, dim), want) and (pool[1].view(-1, dim) == -want)[torch.from_numpy(last >= 0).to(gpu)].all()
