"""GPU: the served-token operators against their formulas in 64 bits, and a decoder's step through them."""
import numpy as np
import pytest

import emel_hip as eh
from decode_reference import BLOCK, adjusted, attention, out, packed, packed_rows, product, view, weight_terms
from helpers import assert_bits_equal, rng

pytestmark = pytest.mark.gpu

EVENT = {"q4_0": eh.OpMulMatQ4_0, "q4_k": eh.OpMulMatQ4K}


def run(event, stream=None):
    status = eh.Kernel(stream).process_event(event)
    assert status == eh.Status.OK, eh.last_error()


def within(got, want, tol, what):
    got = np.asarray(got, np.float64)
    off = np.abs(got - want)
    assert got.shape == want.shape
    ok = (off <= tol) | (np.isnan(got) & np.isnan(want)) | (got == want)
    assert ok.all(), f"{what}: {int((~ok).sum())} outside; worst {np.nanmax(off / np.maximum(tol, 1e-300)):.3g} of the tolerance"


# ---- products -----------------------------------------------------------------------------------


def inputs(seed, form, k, m, n):
    rows = packed_rows(seed, form, k, m)
    x = rng(seed + 1).standard_normal((n, k)).astype(np.float32)
    return rows, x


@pytest.mark.parametrize("form,k", [("q4_0", 32), ("q4_0", 64), ("q4_0", 96), ("q4_0", 480), ("q4_0", 4096), ("q4_0", 4128), ("q4_0", 11008),
                                    ("q4_k", 256), ("q4_k", 768), ("q4_k", 4096), ("q4_k", 11008), ("q4_k", 16384)])
@pytest.mark.parametrize("m,n", [(1, 1), (16, 1), (33, 1), (257, 2), (100, 4), (47, 5), (64, 13), (31, 16), (50, 17), (18, 70)])
def test_product_matches_the_formula(gpu, form, k, m, n):
    import torch

    rows, x = inputs(k + m + n, form, k, m, n)
    w, xt = torch.from_numpy(rows).to(gpu), torch.from_numpy(x).to(gpu)
    y = torch.full((n, m), 7.0, device=gpu)
    run(EVENT[form](packed(w, form, k, m), view(xt), out(y)))
    within(y.cpu().numpy(), *product(form, rows, x), f"{form} {k}x{m}x{n}")
    again = torch.full((n, m), 9.0, device=gpu)
    run(EVENT[form](packed(w, form, k, m), view(xt), out(again)))
    assert torch.equal(y, again)


@pytest.mark.parametrize("form", ["q4_0", "q4_k"])
@pytest.mark.parametrize("k,m,n", [(18688, 4112, 1), (18944, 4112, 1), (26112, 20, 1), (26368, 20, 1), (12544, 33, 2), (12800, 33, 2), (5632, 20, 4), (5888, 20, 4), (32768, 50, 7)])
def test_product_at_the_limits_of_its_lds(gpu, form, k, m, n):
    import torch

    rows, x = inputs(k + m, form, k, m, n)
    y = torch.empty(n, m, device=gpu)
    run(EVENT[form](packed(torch.from_numpy(rows).to(gpu), form, k, m), view(torch.from_numpy(x).to(gpu)), out(y)))
    within(y.cpu().numpy(), *product(form, rows, x), f"{k} {m} {n}")


@pytest.mark.parametrize("form", ["q4_0", "q4_k"])
@pytest.mark.parametrize("m,n", [(40000, 1), (40000, 3), (9000, 16), (5000, 64)])
def test_product_of_many_rows(gpu, form, m, n):
    import torch

    rows, x = inputs(m + n, form, 512, m, n)
    w, xt = torch.from_numpy(rows).to(gpu), torch.from_numpy(x).to(gpu)
    y = torch.empty(n, m, device=gpu)
    run(EVENT[form](packed(w, form, 512, m), view(xt), out(y)))
    within(y.cpu().numpy(), *product(form, rows, x), f"{form} {m}x{n}")


@pytest.mark.parametrize("form", ["q4_0", "q4_k"])
@pytest.mark.parametrize("n", [1, 6, 20])
@pytest.mark.parametrize("shift", [0, 1, 2, 4])
def test_product_strides_and_alignment(gpu, form, n, shift):
    """x and dst by columns, by steps, and inside larger buffers; packed rows at any byte."""
    import torch

    k, m = 512, 37
    rows, x = inputs(5 + n, form, k, m, n)
    store = torch.zeros(rows.size + shift, dtype=torch.uint8, device=gpu)
    store[shift:] = torch.from_numpy(rows.reshape(-1)).to(gpu)
    want, tol = product(form, rows, x)
    src = torch.from_numpy(x).to(gpu)
    for xt in (src.t().contiguous().t(), torch.stack([src, src * 0 + 5], 2)[:, :, 0], torch.cat([src[:, :1] * 0, src], 1)[:, 1:]):
        assert torch.equal(xt, src)
        for yt, keep in ((torch.full((m, n), 3.0, device=gpu).t(), None), (torch.full((n, 2 * m + 1), 3.0, device=gpu)[:, 1::2], None)):
            base = yt._base if yt._base is not None else yt
            run(EVENT[form](packed(store[shift:], form, k, m), view(xt), out(yt)))
            within(yt.cpu().numpy(), want, tol, "strided")
            if base.numel() > m * n:
                rest = base.clone()
                rest[:, 1::2] = 3.0
                assert (rest == 3.0).all()  # what lies between dst's elements is left as it was


@pytest.mark.parametrize("form", ["q4_0", "q4_k"])
@pytest.mark.parametrize("n", [1, 7])
def test_product_range_of_values(gpu, form, n):
    """Columns of very different sizes, with outliers, zeros and subnormals; each column keeps its own precision."""
    import torch

    k, m = 1024, 50
    rows, x = inputs(77 + n, form, k, m, n)
    x *= (10.0 ** np.linspace(-38, 34, n)[:, None]).astype(np.float32) if n > 1 else np.float32(1e-30)
    x[:, 3] *= 1000
    x[0, 256:600] = 0
    y = torch.empty(n, m, device=gpu)
    run(EVENT[form](packed(torch.from_numpy(rows).to(gpu), form, k, m), view(torch.from_numpy(x).to(gpu)), out(y)))
    want, tol = product(form, rows, x)
    within(y.cpu().numpy(), want, tol + 2.0**-140, "range")


@pytest.mark.parametrize("form", ["q4_0", "q4_k"])
@pytest.mark.parametrize("n", [1, 4, 6])
def test_product_of_values_near_the_smallest(gpu, form, n):
    """Runs whose largest value is below 2^-97 keep an absolute precision of 2^-127 a value."""
    import torch

    k, m = 512, 40
    rows, x = inputs(88 + n, form, k, m, n)
    x *= np.float32(2.0**-110)
    y = torch.empty(n, m, device=gpu)
    run(EVENT[form](packed(torch.from_numpy(rows).to(gpu), form, k, m), view(torch.from_numpy(x).to(gpu)), out(y)))
    want, tol = product(form, rows, x)
    hi, lo = weight_terms(form, rows)
    within(y.cpu().numpy(), want, tol + (np.abs(hi) + np.abs(lo)).sum(1) * 2.0**-127 + 2.0**-140, "small")


def test_product_of_more_columns_than_a_launch_takes(gpu):
    """Columns run in parts; more than 65535 groups of 16 of them would not fit a grid."""
    import torch

    k, m, n = 32, 5, (1 << 20) + 3
    rows = packed_rows(3, "q4_0", k, m)
    x = torch.randn(n, k, device=gpu, generator=torch.Generator(gpu).manual_seed(5))
    y = torch.empty(n, m, device=gpu)
    run(EVENT["q4_0"](packed(torch.from_numpy(rows).to(gpu), "q4_0", k, m), view(x), out(y)))
    want, tol = product("q4_0", rows, x.cpu().numpy())
    within(y.cpu().numpy(), want, tol, "columns")


def test_product_of_more_rows_than_a_launch_takes(gpu):
    """Rows run in parts of 2^22 where k is short; the rows on both sides of the cut, the ends and some between."""
    import torch

    k, m, n = 32, (1 << 22) + 37, 5
    some = packed_rows(4, "q4_0", k, 4096)
    pick = np.arange(m) % 4093
    rows = torch.from_numpy(some).to(gpu)[torch.from_numpy(pick).to(gpu)].contiguous()
    x = rng(6).standard_normal((n, k)).astype(np.float32)
    y = torch.empty(n, m, device=gpu)
    run(EVENT["q4_0"](packed(rows, "q4_0", k, m), view(torch.from_numpy(x).to(gpu)), out(y)))
    want, tol = product("q4_0", some, x)
    got = y.cpu().numpy()
    for a, b in ((0, 5000), ((1 << 21) - 7, (1 << 21) + 300), ((1 << 22) - 300, m)):
        within(got[:, a:b], want[:, pick[a:b]], tol[:, pick[a:b]], f"rows {a}")


@pytest.mark.parametrize("form", ["q4_0", "q4_k"])
@pytest.mark.parametrize("n", [1, 3, 9])
def test_product_infinities_and_nan_as_in_the_formula(gpu, form, n):
    import torch

    values, size = BLOCK[form]
    k, m = 1024, 40
    rows, x = inputs(31 + n, form, k, m, n)
    x[0, 700], x[n - 1, 17] = np.inf, -np.inf
    if n > 2:
        x[1, 5] = np.nan
    b = rows.reshape(m, -1, size)
    b[3, 1, :2] = np.array([np.inf], np.float16).view(np.uint8)
    b[4, 0, :2] = np.array([np.nan], np.float16).view(np.uint8)
    y = torch.empty(n, m, device=gpu)
    run(EVENT[form](packed(torch.from_numpy(rows).to(gpu), form, k, m), view(torch.from_numpy(x).to(gpu)), out(y)))
    hi, lo = weight_terms(form, rows)
    with np.errstate(all="ignore"):
        want = np.stack([((hi - lo) * c.astype(np.float64)).sum(1) for c in x])
    got = y.cpu().numpy()
    special = ~np.isfinite(want)
    assert special.any() and np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)].astype(np.float32))


# ---- the paged cache -------------------------------------------------------------------------------


def pools(gpu, bf16, pages, kv, page, dim, order, seed=None):
    """Key and value pools [pages, kv, page, dim], laid out by tokens, by heads, or both pools side by side."""
    import torch

    kind = torch.bfloat16 if bf16 else torch.float16
    shape = {"head": (2, pages, kv, page, dim), "token": (2, pages, page, kv, dim), "both": (pages, 2, kv, page, dim), "apart": (2, pages, kv, page, dim + 8)}[order]
    t = torch.from_numpy(rng(seed or 0).standard_normal(shape).astype(np.float32)).to(gpu).to(kind)
    if seed is None:
        t.fill_(3.0)
    if order == "token":
        return t[0].transpose(1, 2), t[1].transpose(1, 2), t
    if order == "both":
        return t[:, 0], t[:, 1], t
    return t[0][..., :dim], t[1][..., :dim], t


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("order", ["head", "token", "both", "apart"])
@pytest.mark.parametrize("kv,page,dim,tokens", [(1, 1, 1, 1), (2, 16, 64, 5), (3, 7, 20, 100), (8, 16, 128, 64), (1, 64, 250, 700)])
def test_append_stores_each_token_and_nothing_else(gpu, bf16, order, kv, page, dim, tokens):
    import torch

    pages = tokens // page + 3
    kp, vp, store = pools(gpu, bf16, pages, kv, page, dim, order)
    g = rng(tokens)
    k, v = (torch.from_numpy(g.standard_normal((tokens, kv, dim)).astype(np.float32)).to(gpu) for _ in range(2))
    slots = g.permutation(pages * page)[:tokens].astype(np.int32)
    slots[::7] = -1
    slots[3::11] = pages * page + 5
    if tokens > 4:
        slots[tokens - 1] = slots[1]  # the later token is stored
        k[2, 0, 0], v[2, -1, -1] = float("inf"), float("nan")
    before = store.clone()
    run(eh.OpPagedKvAppend(view(k), view(v), view(torch.from_numpy(slots).to(gpu)), out(kp), out(vp)))
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            for pool, src in ((kp, k), (vp, v)):
                place = [t for t, x in enumerate(slots.tolist()) if x == s][-1]
                assert torch.equal(pool[s // page, :, s % page].view(torch.int16), src[place].to(pool.dtype).view(torch.int16)) or \
                    torch.isnan(src[place]).any()
    # every other slot, and what lies between the pools' elements, is as it was
    for pool in (kp, vp):
        for s in slots.tolist():
            if 0 <= s < pages * page:
                pool[s // page, :, s % page] = 3.0
    assert torch.equal(store, before)


@pytest.mark.parametrize("tokens", [2, 300, 5000])
def test_append_of_one_slot_named_by_all(gpu, tokens):
    import torch

    kp, vp, _ = pools(gpu, False, 4, 2, 8, 64, "token")
    k = torch.arange(tokens, device=gpu, dtype=torch.float32)[:, None, None].expand(tokens, 2, 64).contiguous()
    run(eh.OpPagedKvAppend(view(k), view(-k), view(torch.full((tokens,), 9, dtype=torch.int32, device=gpu)), out(kp), out(vp)))
    assert (kp[1, :, 1] == (tokens - 1)).all() and (vp[1, :, 1] == 1 - tokens).all()


def attend_case(gpu, bf16, heads, kv, dim, page, lengths, order, seed, spare=2):
    import torch

    most = max(1, max(-(-n // page) for n in lengths)) + 1
    pages = len(lengths) * most + spare
    kp, vp, _ = pools(gpu, bf16, pages, kv, page, dim, order, seed)
    g = rng(seed + 9)
    table = g.permutation(pages)[: len(lengths) * most].reshape(len(lengths), most).astype(np.int32)
    q = (g.standard_normal((len(lengths), heads, dim)) * 2).astype(np.float32)
    return {"q": torch.from_numpy(q).to(gpu), "kp": kp, "vp": vp, "table": torch.from_numpy(table).to(gpu),
            "lengths": torch.tensor(lengths, dtype=torch.int32, device=gpu), "y": torch.full(q.shape, 5.0, device=gpu)}


def attend_event(c, **more):
    more.setdefault("scale", c["q"].shape[-1] ** -0.5)
    return eh.OpPagedAttention(view(c["q"]), view(c["kp"]), view(c["vp"]), view(c["table"]), view(c["lengths"]), out(c["y"]), **more)


def cached(c, s, window=0):
    """Keys and values [positions, kv, dim] of sequence s, f64."""
    import torch

    n, page = int(c["lengths"][s]), c["kp"].shape[2]
    at = torch.arange(max(0, n - window) if window else 0, n, device=c["q"].device)
    ids = c["table"][s].long()[at // page]
    return tuple(p[ids, :, at % page].double().cpu().numpy() for p in (c["kp"], c["vp"]))


def check_attention(c, window=0, cap=0.0, scale=None, skip=()):
    got, dim = c["y"].cpu().numpy(), c["q"].shape[-1]
    for s, n in enumerate(c["lengths"].tolist()):
        if s in skip:
            continue
        if n == 0:
            assert (got[s] == 0).all(), f"sequence {s} of length 0"
            continue
        want, tol = attention(c["q"][s].double().cpu().numpy(), *cached(c, s, window), dim ** -0.5 if scale is None else scale, cap)
        within(got[s], want, tol, f"sequence {s} of length {n}")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 8), (4, 4, 64), (8, 2, 80), (32, 8, 128), (5, 1, 96), (40, 2, 64), (16, 1, 256), (6, 2, 200), (17, 1, 136), (7, 7, 128)])
@pytest.mark.parametrize("page,order", [(16, "token"), (1, "head"), (24, "both"), (64, "apart")])
def test_attention_matches_the_formula(gpu, bf16, heads, kv, dim, page, order):
    lengths = [1, 0, 15, 16, 17, 63, 64, 65, 129, 700]
    c = attend_case(gpu, bf16, heads, kv, dim, page, lengths, order, heads + dim)
    run(attend_event(c))
    check_attention(c)
    first = c["y"].clone()
    c["y"].fill_(-1)
    run(attend_event(c))
    assert (first == c["y"]).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("window,cap,scale", [(1, 0.0, None), (16, 0.0, 0.3), (100, 20.0, None), (1000, 0.0, None), (5000, 3.0, 1.0), (0, 50.0, -0.5), (2**40, 0.0, 0.0)])
def test_attention_windows_caps_and_scales(gpu, bf16, window, cap, scale):
    c = attend_case(gpu, bf16, 8, 2, 128, 16, [3, 100, 101, 0, 2500, 1000, 1], "token", 3)
    run(attend_event(c, window=window, soft_cap=cap, **({} if scale is None else {"scale": scale})))
    check_attention(c, window if window < 2**31 else 0, cap, scale)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("seqs,low,high,heads,kv,dim", [(1, 20000, 20000, 8, 1, 128), (1, 9001, 9001, 32, 8, 128), (3, 1, 12000, 8, 8, 64), (300, 0, 90, 8, 2, 64), (130, 1, 300, 24, 1, 256)])
def test_attention_of_long_and_many_sequences(gpu, bf16, seqs, low, high, heads, kv, dim):
    lengths = [low + (high - low) * i // max(1, seqs - 1) for i in range(seqs)]
    c = attend_case(gpu, bf16, heads, kv, dim, 32, lengths, "token", seqs)
    run(attend_event(c))
    check_attention(c)


def test_attention_reads_nothing_behind_a_sequence(gpu):
    """What a page holds behind the last token, and before the window, changes nothing, NaN and infinities included."""
    import torch

    c = attend_case(gpu, False, 8, 2, 128, 16, [1, 19, 33, 250], "head", 5)
    run(attend_event(c, window=30))
    want = c["y"].clone()
    for s, n in enumerate(c["lengths"].tolist()):
        for j in [j for j in range(c["table"].shape[1] * 16) if j >= n or j < n - 30]:
            c["kp"][c["table"][s, j // 16], :, j % 16] = float("nan")
            c["vp"][c["table"][s, j // 16], :, j % 16] = float("inf")
    # ids of pages that are not reached may be anything
    for s, n in enumerate(c["lengths"].tolist()):
        c["table"][s, -(-n // 16):] = 2**31 - 1
    c["y"].fill_(0)
    run(attend_event(c, window=30))
    assert torch.equal(c["y"], want)


def test_attention_infinities_and_nan_of_the_cache(gpu):
    """An infinite score of one sign takes no part or all of it, as softmax has it; NaN stays with its own heads."""
    import torch

    c = attend_case(gpu, False, 4, 2, 64, 16, [40, 40, 40, 200], "head", 6)
    place = lambda s, j: (int(c["table"][s, j // 16]), j % 16)  # noqa: E731
    p, i = place(0, 7)
    c["vp"][p, 0, i, 3] = float("inf")  # an infinite value: that dim alone
    p, i = place(1, 7)
    c["kp"][p, 1, i, 5] = float("nan")  # NaN scores: the heads that read cache head 1
    p, i = place(2, 39)
    c["q"][2, :, 5] = 1.0
    c["kp"][p, 0, i] = 0.0
    c["kp"][p, 0, i, 5] = -float("inf")  # a score of -inf: the position takes no part
    p, i = place(3, 70)
    c["vp"][p, 1, i, 9] = float("nan")
    run(attend_event(c))
    got = c["y"].cpu().numpy()
    assert np.isposinf(got[0, :2, 3]).all() and np.isfinite(np.delete(got[0], 3, -1)).all() and np.isfinite(got[0, 2:]).all()
    assert np.isnan(got[1, 2:]).all() and np.isfinite(got[1, :2]).all()
    k, v = cached(c, 2)
    want, tol = attention(c["q"][2].double().cpu().numpy(), np.delete(k, 39, 0), np.delete(v, 39, 0), 1 / 8, 0.0)
    within(got[2, :2], want[:2], tol[:2], "-inf score")
    assert np.isnan(got[3, 2:, 9]).all() and np.isfinite(np.delete(got[3], 9, -1)).all()


def test_attention_without_any_finite_score(gpu):
    """Every score -inf is 0 / 0, as soft_max of such a row gives."""
    c = attend_case(gpu, True, 2, 1, 32, 4, [9, 500], "head", 8)
    c["q"][:, :, 0] = 1.0
    c["kp"][..., 0] = -float("inf")
    run(attend_event(c))
    assert c["y"].isnan().all()


def test_attention_refuses_to_read_outside_the_pool(gpu):
    """A page id outside the pool, and a length past the table or below zero: NaN for that sequence alone."""
    lengths = [40, 300, 50, 60, 3, 70]
    c = attend_case(gpu, False, 4, 2, 64, 16, lengths, "token", 4)
    c["table"][0, 1], c["table"][1, 17], c["table"][2, 0] = -1, c["kp"].shape[0], -(2**31)
    good = c["lengths"].clone()
    c["lengths"][3], c["lengths"][4] = 2**31 - 1, -5
    run(attend_event(c))
    for s in range(5):
        assert c["y"][s].isnan().all(), s
    c["lengths"].copy_(good)
    check_attention(c, skip=range(5))


def test_cache_past_32_bit_offsets(gpu):
    """Pools of more than 2^32 halves: tokens appended to their first and last pages, and attention over those."""
    import torch

    kv, page, dim, tokens = 4, 64, 128, 300
    pages = (1 << 17) + 9  # of 2^15 halves
    kp, vp = (torch.empty(pages, kv, page, dim, dtype=torch.float16, device=gpu) for _ in range(2))
    assert kp.numel() > 1 << 32
    table = torch.tensor([[0, pages - 1, 1, pages - 2, pages // 2], [pages - 5, 2, pages - 4, pages - 3, pages - 6]], dtype=torch.int32, device=gpu)
    q = torch.from_numpy(rng(70).standard_normal((2, 8, dim)).astype(np.float32)).to(gpu)
    c = {"q": q, "kp": kp, "vp": vp, "table": table, "lengths": torch.tensor([tokens, tokens - 7], dtype=torch.int32, device=gpu), "y": torch.empty_like(q)}
    at = torch.arange(tokens, device=gpu)
    for s in range(2):
        k, v = (torch.from_numpy(rng(71 + 2 * s + i).standard_normal((tokens, kv, dim)).astype(np.float32)).to(gpu) for i in range(2))
        slots = (table[s][at // page] * page + at % page).to(torch.int32)
        run(eh.OpPagedKvAppend(view(k), view(v), view(slots), out(kp), out(vp)))
        where = table[s].long()[at // page]
        assert torch.equal(kp[where, :, at % page], k.half()) and torch.equal(vp[where, :, at % page], v.half())
    run(attend_event(c))
    check_attention(c)


def test_attention_in_parts_of_a_batch(gpu):
    """A table so wide that its units, counted before the lengths are known, pass 2^31: the batch runs in parts."""
    import torch

    seqs, heads = 1100, 64
    few = attend_case(gpu, False, heads, heads, 8, 256, [int(n) for n in rng(81).integers(0, 500, 40)], "head", 80)
    at = torch.arange(seqs, device=gpu) * 7 % 40
    table = torch.full((seqs, 1 << 14), -1, dtype=torch.int32, device=gpu)
    table[:, :few["table"].shape[1]] = few["table"][at]
    q = torch.from_numpy(rng(82).standard_normal((seqs, heads, 8)).astype(np.float32)).to(gpu)
    c = {**few, "q": q, "table": table, "lengths": few["lengths"][at].contiguous(), "y": torch.full_like(q, 5.0)}
    run(attend_event(c))
    check_attention(c, skip=set(range(seqs)) - {*range(0, 60), *range(1000, 1100)})
    assert c["y"].isfinite().all() and not (c["y"] == 5.0).any()


@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (3, 1, 40)])
def test_attention_strides(gpu, heads, kv, dim):
    """q and dst with heads and dims in other orders, the index tensors by columns, pools that start at any half."""
    import torch

    c = attend_case(gpu, False, heads, kv, dim, 8, [5, 90, 33], "head", 11)
    run(attend_event(c))
    want = c["y"].clone()
    store = torch.zeros(2 * c["kp"].numel() + 3, dtype=torch.float16, device=gpu)
    for name, at in (("kp", 1), ("vp", c["kp"].numel() + 3)):
        t = store[at:at + c["kp"].numel()].view(c["kp"].shape)
        t.copy_(c[name])
        c[name] = t
    c["q"] = c["q"].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    c["y"] = torch.full((heads, dim, 3, 2), 5.0, device=gpu)[..., 1].permute(2, 0, 1)
    c["table"] = c["table"].t().contiguous().t()
    c["lengths"] = torch.stack([c["lengths"], c["lengths"] * 0 - 1], 1)[:, 0]
    run(attend_event(c))
    assert torch.equal(c["y"], want) and (c["y"]._base[..., 0] == 5.0).all()


# ---- logits -----------------------------------------------------------------------------------------


def logits_case(seed, card, rows, history, biases, mask, one_row=False):
    g = rng(seed)
    c = {"logits": (g.standard_normal((rows, card)) * 4).astype(np.float32)}
    r = 1 if one_row else rows
    if history:
        c["history"] = g.integers(-3, max(2, card // 3) + 3, (r, history)).astype(np.int32)
        c["history"][0, -1] = card  # past the vocabulary: ignored
        c["history_len"] = g.integers(-1, history + 2, r).astype(np.int32)
        c["repeat"], c["frequency"], c["presence"] = (g.uniform(0.5, 1.5, r).astype(np.float32) for _ in range(3))
    if biases:
        c["bias_ids"] = g.integers(-1, card + 1, (r, biases)).astype(np.int32)
        c["bias_ids"][:, -1] = c["bias_ids"][:, 0]
        c["bias"] = g.standard_normal((r, biases)).astype(np.float32)
    if mask:
        c["allowed"] = g.integers(-2**31, 2**31, (r, -(-card // 32))).astype(np.int32)
    return c


def logits_event(c, dev, y):
    return eh.OpLogitsAdjust(view(dev["logits"]), out(y), **{n: view(dev[n]) for n in c if n != "logits"})


@pytest.mark.parametrize("card,rows", [(1, 1), (31, 3), (4096, 2), (4097, 2), (50001, 5), (151936, 2)])
@pytest.mark.parametrize("history,biases,mask", [(0, 0, False), (1, 0, False), (700, 0, False), (0, 9, False), (0, 0, True), (5000, 40, True)])
@pytest.mark.parametrize("one_row", [False, True])
def test_logits_adjustment_is_the_definition(gpu, card, rows, history, biases, mask, one_row):
    import torch

    c = logits_case(card + history, card, rows, history, biases, mask, one_row)
    c["logits"][0, 0] = np.nan
    c["logits"][-1, -1] = -np.inf
    want = adjusted(**c)
    dev = {n: torch.from_numpy(v).to(gpu) for n, v in c.items()}
    y = torch.full((rows, card), 7.0, device=gpu)
    run(logits_event(c, dev, y))
    assert_bits_equal(y.cpu().numpy(), want, "apart")
    assert torch.equal(dev["logits"].view(torch.int32), torch.from_numpy(c["logits"]).to(gpu).view(torch.int32))
    run(logits_event(c, dev, dev["logits"]))
    assert_bits_equal(dev["logits"].cpu().numpy(), want, "in place")


@pytest.mark.parametrize("card,rows,history,biases,mask", [(151937, 15, 0, 0, False), (151937, 15, 700, 9, True), (2200001, 1, 70000, 66000, True)])
def test_logits_adjustment_of_many_logits(gpu, card, rows, history, biases, mask):
    """More logits than run at once in the shorter runs: apart, in place, and with a step of two."""
    import torch

    c = logits_case(card + rows, card, rows, history, biases, mask)
    want = adjusted(**c)
    dev = {n: torch.from_numpy(v).to(gpu) for n, v in c.items()}
    y = torch.full((rows, card), 7.0, device=gpu)
    run(logits_event(c, dev, y))
    assert_bits_equal(y.cpu().numpy(), want, "apart")
    y = torch.full((rows, 2 * card), 7.0, device=gpu)
    run(logits_event(c, dev, y[:, 1::2]))
    assert_bits_equal(y[:, 1::2].cpu().numpy(), want, "steps of two")
    assert (y[:, 0::2] == 7.0).all()
    two = torch.stack([dev["logits"], dev["logits"]], -1)[..., 0]
    run(logits_event(c, {**dev, "logits": two}, two))
    assert_bits_equal(two.cpu().numpy(), want, "in place, steps of two")
    run(logits_event(c, dev, dev["logits"]))
    assert_bits_equal(dev["logits"].cpu().numpy(), want, "in place")


def test_logits_adjustment_of_a_history_past_16_bits(gpu):
    """Counts and entry numbers that do not fit half a word."""
    import torch

    c = logits_case(9, 5003, 2, 70000, 66000, False)
    c["history"][0, :69000] = 77  # one token, 69000 times over
    c["history_len"][:] = 70000
    want = adjusted(**c)
    dev = {n: torch.from_numpy(v).to(gpu) for n, v in c.items()}
    y = torch.empty(2, 5003, device=gpu)
    run(logits_event(c, dev, y))
    assert_bits_equal(y.cpu().numpy(), want, "long history")


def test_logits_adjustment_strides(gpu):
    import torch

    c = logits_case(8, 5003, 3, 64, 5, True)
    want = adjusted(**c)
    dev = {n: torch.from_numpy(v).to(gpu) for n, v in c.items()}
    spread = {n: torch.stack([t, t * 0 - 9], -1)[..., 0] for n, t in dev.items()}
    y = torch.full((3, 2 * 5003 + 1), 3.0, device=gpu)
    run(logits_event(c, spread, y[:, 1::2]))
    assert_bits_equal(y[:, 1::2].cpu().numpy(), want, "steps of two")
    assert (y[:, 0::2] == 3.0).all()
    for at in range(4):  # rows that start anywhere, each inside a longer one
        y = torch.full((3, 5003 + at + 2), 3.0, device=gpu)
        run(logits_event(c, dev, y[:, at:at + 5003]))
        assert_bits_equal(y[:, at:at + 5003].cpu().numpy(), want, f"offset {at}")
        y[:, at:at + 5003] = 3.0
        assert (y == 3.0).all()
    y = torch.empty(5003, 3, device=gpu).t()
    run(logits_event(c, dev, y))
    assert_bits_equal(y.cpu().numpy(), want, "by columns")


# ---- together -----------------------------------------------------------------------------------------


class Step:
    """One token of three sequences through a layer and the head, as a serving program chains the events."""

    def __init__(self, gpu, hidden=512, heads=8, kv=2, dim=64, vocab=1000, page=8):
        import torch

        self.dim, self.page, seqs = dim, page, 3
        g = rng(12)
        up = lambda a: torch.from_numpy(a).to(gpu)  # noqa: E731
        self.rows = {"q": packed_rows(1, "q4_0", hidden, heads * dim), "k": packed_rows(2, "q4_0", hidden, kv * dim), "v": packed_rows(3, "q4_0", hidden, kv * dim),
                     "o": packed_rows(4, "q4_k", heads * dim, hidden), "head": packed_rows(5, "q4_k", hidden, vocab)}
        w = {n: packed(up(r), "q4_0" if n in "qkv" else "q4_k", heads * dim if n == "o" else hidden, len(r)) for n, r in self.rows.items()}
        self.x, self.gain = up(g.standard_normal((seqs, hidden)).astype(np.float32)), up(g.uniform(0.5, 1.5, hidden).astype(np.float32))
        self.kp, self.vp, _ = pools(gpu, True, 40, kv, page, dim, "token", 21)
        self.table = up(g.permutation(40)[:30].reshape(3, 10).astype(np.int32))
        self.lengths = up(np.array([1, 24, 61], np.int32))
        self.slots = up(np.zeros(seqs, np.int32))
        new = lambda *s: torch.zeros(*s, device=gpu)  # noqa: E731
        self.h, self.q, self.k, self.v, self.a = new(seqs, hidden), new(seqs, heads, dim), new(seqs, kv, dim), new(seqs, kv, dim), new(seqs, heads, dim)
        self.o, self.logits = new(seqs, hidden), new(seqs, vocab)
        self.best = torch.zeros(seqs, 1, dtype=torch.int32, device=gpu)
        self.history = up(g.integers(0, vocab, (seqs, 20)).astype(np.int32))
        self.repeat = up(np.full(1, 1.2, np.float32))
        self.allowed = up(g.integers(-2**31, 2**31, (1, -(-vocab // 32))).astype(np.int32))
        flat = lambda t: t.view(seqs, -1)  # noqa: E731
        self.events = [
            eh.OpRmsNormMul(view(self.x), view(self.gain), out(self.h), 1e-5),
            eh.OpMulMatQ4_0(w["q"], view(self.h), out(flat(self.q))),
            eh.OpMulMatQ4_0(w["k"], view(self.h), out(flat(self.k))),
            eh.OpMulMatQ4_0(w["v"], view(self.h), out(flat(self.v))),
            eh.OpPagedKvAppend(view(self.k), view(self.v), view(self.slots), out(self.kp), out(self.vp)),
            eh.OpPagedAttention(view(self.q), view(self.kp), view(self.vp), view(self.table), view(self.lengths), out(self.a), scale=dim ** -0.5),
            eh.OpMulMatQ4K(w["o"], view(flat(self.a)), out(self.o)),
            eh.OpAdd(view(self.x), view(self.o), out(self.o)),
            eh.OpMulMatQ4K(w["head"], view(self.o), out(self.logits)),
            eh.OpLogitsAdjust(view(self.logits), out(self.logits), history=view(self.history), repeat=view(self.repeat), allowed=view(self.allowed)),
            eh.OpArgmaxRows(view(self.logits), out(self.best)),
        ]

    def place(self):
        """The slot of each sequence's newest token."""
        import torch

        last = self.lengths.long() - 1
        self.slots.copy_((self.table.gather(1, (last // self.page)[:, None])[:, 0].long() * self.page + last % self.page).to(torch.int32))

    def outputs(self):
        return [t.clone() for t in (self.a, self.o, self.logits, self.best, self.kp, self.vp)]


def test_a_decoder_step_through_all_of_them(gpu):
    """Each event's output against the formula on the inputs that it had, through three steps of a growing cache."""
    import torch

    st = Step(gpu)
    kernel = eh.Kernel(synchronous=False)
    for step in range(3):
        st.place()
        for e in st.events:
            assert kernel.process_event(e) == eh.Status.OK, eh.last_error()
        torch.cuda.synchronize()
        n = lambda t: t.cpu().numpy()  # noqa: E731
        for name, src, dst in (("q", st.h, st.q), ("k", st.h, st.k), ("v", st.h, st.v), ("o", st.a, None), ("head", st.o, None)):
            if dst is not None:
                within(n(dst).reshape(3, -1), *product("q4_0", st.rows[name], n(src).reshape(3, -1)), name)
        for s, slot in enumerate(st.slots.tolist()):
            assert torch.equal(st.kp[slot // st.page, :, slot % st.page], st.k[s].to(torch.bfloat16))
            assert torch.equal(st.vp[slot // st.page, :, slot % st.page], st.v[s].to(torch.bfloat16))
        check_attention({"q": st.q, "kp": st.kp, "vp": st.vp, "table": st.table, "lengths": st.lengths, "y": st.a})
        want, tol = product("q4_k", st.rows["o"], n(st.a).reshape(3, -1))
        within(n(st.o), want + n(st.x), tol + 2.0**-23 * np.abs(want + n(st.x)), "o")
        raw, tol = product("q4_k", st.rows["head"], n(st.o))
        masked = np.isneginf(n(st.logits))
        plain = adjusted(raw.astype(np.float32), history=n(st.history), repeat=n(st.repeat), allowed=n(st.allowed))
        assert np.array_equal(masked, np.isneginf(plain))
        # a penalty scales an error by at most 1.2, or turns a logit within tol of zero
        within(np.where(masked, 0, n(st.logits)), np.where(masked, 0, plain), 1.5 * tol + 2.0**-22 * np.abs(raw), "logits")
        assert np.array_equal(n(st.best)[:, 0], n(st.logits).argmax(1))
        st.lengths += 1


def test_a_captured_step_follows_its_cache(gpu):
    """The step captured once and replayed: lengths, slots and pages are read when it runs."""
    import torch

    eager, graphed = Step(gpu), Step(gpu)
    side = torch.cuda.Stream()
    kernel = eh.Kernel(side.cuda_stream, synchronous=False)
    with torch.cuda.stream(side):  # sizes the stream's workspace
        graphed.place()
        kept = graphed.kp.clone(), graphed.vp.clone()
        for e in graphed.events:
            assert kernel.process_event(e) == eh.Status.OK, eh.last_error()
        side.synchronize()
        graphed.kp.copy_(kept[0])
        graphed.vp.copy_(kept[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for e in graphed.events:
            assert kernel.process_event(e) == eh.Status.OK, eh.last_error()
    plain = eh.Kernel(synchronous=False)
    for step in range(4):
        for st in (eager, graphed):
            st.place()
        for e in eager.events:
            assert plain.process_event(e) == eh.Status.OK
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager.outputs(), graphed.outputs()):
            assert torch.equal(a, b), step
        for st in (eager, graphed):
            st.lengths += 1
            st.x.mul_(1.01)


def test_streams_do_not_share_scratch(gpu):
    """Two streams at once, each with its own sequences and products."""
    import torch

    streams = [torch.cuda.Stream() for _ in range(2)]
    cases = [attend_case(gpu, False, 8, 2, 128, 16, [900, 3, 2500], "token", 40 + i) for i in range(2)]
    weights = [inputs(60 + i, "q4_k", 1024, 300, 12) for i in range(2)]
    dev = [(torch.from_numpy(r).to(gpu), torch.from_numpy(x).to(gpu), torch.empty(12, 300, device=gpu)) for r, x in weights]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, c, (w, x, y) in zip(streams, cases, dev):
            k = eh.Kernel(s.cuda_stream, synchronous=False)
            assert k.process_event(attend_event(c)) == k.process_event(eh.OpMulMatQ4K(packed(w, "q4_k", 1024, 300), view(x), out(y))) == eh.Status.OK
    torch.cuda.synchronize()
    for c, (r, x), (_, _, y) in zip(cases, weights, dev):
        check_attention(c)
        within(y.cpu().numpy(), *product("q4_k", r, x), "stream")


def test_a_capture_needs_its_scratch_beforehand(gpu):
    """Under capture a call whose scratch must grow is refused, and nothing of it is recorded; a reserve ahead lets it in."""
    import ctypes

    import torch

    handle = ctypes.c_void_p()  # a stream of its own: one of torch's pool may have scratch already
    assert eh.load().emel_stream_create(ctypes.byref(handle)) == eh.Status.OK
    stream = torch.cuda.ExternalStream(handle.value)
    kernel = eh.Kernel(stream.cuda_stream, synchronous=False)
    c = attend_case(gpu, False, 8, 2, 64, 16, [700, 90], "token", 21)
    rows, x = inputs(61, "q4_k", 1024, 300, 9)
    w, x_dev, y = torch.from_numpy(rows).to(gpu), torch.from_numpy(x).to(gpu), torch.full((9, 300), 7.0, device=gpu)
    events = attend_event(c), eh.OpMulMatQ4K(packed(w, "q4_k", 1024, 300), view(x_dev), out(y))
    c["y"].fill_(7.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        assert [kernel.process_event(e) for e in events] == [eh.Status.STREAM_CAPTURE] * 2
        x_dev.mul_(1.0)  # a graph of no nodes is no test of one
    graph.replay()
    torch.cuda.synchronize()
    assert (c["y"] == 7.0).all() and (y == 7.0).all()
    assert eh.stream_reserve(32 << 20, 1 << 20, stream.cuda_stream) == eh.Status.OK
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        assert [kernel.process_event(e) for e in events] == [eh.Status.OK] * 2
    for _ in range(3):
        c["y"].fill_(7.0)
        y.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        check_attention(c)
        within(y.cpu().numpy(), *product("q4_k", rows, x), "captured")
    del graph
    assert eh.load().emel_stream_destroy(handle) == eh.Status.OK
