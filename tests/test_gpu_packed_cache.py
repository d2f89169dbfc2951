"""GPU: the paged cache in packed rows: quantised as it is written, read back, and attended over."""
import numpy as np
import pytest

import emel_hip as eh
from decode_reference import attention, out, view
from helpers import rng
from packed_cache_reference import SIZE, decode, encode, pages_view, pool_tensors, random_rows
from rope_reference import rope

pytestmark = pytest.mark.gpu

KINDS = [("q8_0", "q8_0"), ("q8_0", "q4_0"), ("q4_0", "q8_0"), ("q4_0", "q4_0")]
ORDERS = ["head", "token", "both", "apart"]


def run(event, stream=None):
    status = eh.Kernel(stream).process_event(event)
    assert status == eh.Status.OK, eh.last_error()


def within(got, want, tol, what):
    got = np.asarray(got, np.float64)
    off = np.abs(got - want)
    assert got.shape == want.shape
    ok = (off <= tol) | (np.isnan(got) & np.isnan(want)) | (got == want)
    assert ok.all(), f"{what}: {int((~ok).sum())} outside; worst {np.nanmax(off / np.maximum(tol, 1e-300)):.3g} of the tolerance"


def up(gpu, a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).to(gpu)


# ---- written ------------------------------------------------------------------------------------


def append(gpu, kinds, k, v, slots, kp, vp, dim):
    run(eh.OpPagedKvAppend(view(k), view(v), view(up(gpu, slots)), pages_view(kp, kinds[0], dim, True), pages_view(vp, kinds[1], dim, True)))


def values(seed, shape):
    """Rows of many sizes: normal ones, an outlier each, zeros, subnormal scales, and values around every tie."""
    g = rng(seed)
    x = (g.standard_normal(shape) * np.exp(2 * g.standard_normal(shape[:-1] + (1,)))).astype(np.float32)
    flat = x.reshape(-1, shape[-1])
    flat[::5, 3] *= 50
    flat[1::9] *= np.float32(2.0**-22)
    flat[2::9] = 0
    flat[3::9] = np.round(flat[3::9])
    flat[4::9] *= np.float32(1e6)
    flat[5::9, : 32] = np.linspace(-8, 7.5, 32, dtype=np.float32)  # halves of a scale of one
    flat[6::9, 1::2] = -flat[6::9, ::2]  # pairs of opposite signs
    return x


@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("kv,page,dim,tokens", [(1, 1, 32, 1), (2, 16, 64, 5), (3, 7, 96, 100), (8, 16, 128, 64), (1, 64, 256, 700), (2, 24, 160, 2500), (1, 5, 1056, 30)])
def test_append_stores_each_token_and_nothing_else(gpu, kinds, order, kv, page, dim, tokens):
    import torch

    pages = tokens // page + 3
    kp, vp, store = pool_tensors(gpu, kinds, pages, kv, page, dim, order)
    g = rng(tokens + dim)
    k, v = values(dim, (tokens, kv, dim)), values(dim + 1, (tokens, kv, dim))
    slots = g.permutation(pages * page)[:tokens].astype(np.int32)
    slots[::7] = -1
    slots[3::11] = pages * page + 5
    if tokens > 4:
        slots[tokens - 1] = slots[1]  # the later token is stored
        k[2, 0, 5], v[2, -1, dim - 1], v[4, 0, 0] = np.inf, np.nan, -np.inf
    before = store.clone()
    append(gpu, kinds, up(gpu, k), up(gpu, v), slots, kp, vp, dim)
    stored = {s: t for t, s in enumerate(slots.tolist()) if 0 <= s < pages * page}
    for pool, kind, src in ((kp, kinds[0], k), (vp, kinds[1], v)):
        ids = list(stored)
        if ids:
            at = torch.tensor(ids, device=gpu)
            got = pool[at // page, :, at % page].cpu().numpy()
            assert np.array_equal(got, encode(kind, src[[stored[s] for s in ids]]))
            pool[at // page, :, at % page] = 0xAA
    assert torch.equal(store, before)  # every other slot, and what lies between


@pytest.mark.parametrize("kinds", KINDS)
def test_append_at_every_tie(gpu, kinds):
    """Every half of every scale, and the f32 values next to it, for scales over f16's whole range, subnormal ones too."""
    g = rng(17)
    d = np.abs(np.concatenate([np.arange(1, 60).astype(np.uint16).view(np.float16), g.integers(1, 0x7BFF, 900).astype(np.uint16).view(np.float16)])).astype(np.float64)
    k, v = (np.zeros((2 * len(d), 1, 128), np.float32) for _ in range(2))
    for x, kind in ((k, kinds[0]), (v, kinds[1])):
        end = 127 if kind == "q8_0" else 8
        halves = rng(18).integers(-end, end, (len(x), 1, 127)) + 0.5
        sign = np.repeat([1.0, -1.0], len(d))[:, None, None]
        near = (halves * np.concatenate([d, d])[:, None, None]).astype(np.float32)  # exact: 19 bits
        near = np.where(g.random(near.shape) < 1 / 3, near, np.nextafter(near, np.where(g.random(near.shape) < 0.5, np.float32(np.inf), np.float32(-np.inf))))
        x[..., 1:] = near
        x[..., 0::32] = (sign * end) * np.concatenate([d, d])[:, None, None]
    kp, vp, _ = pool_tensors(gpu, kinds, len(k), 1, 1, 128, "head")
    append(gpu, kinds, up(gpu, k), up(gpu, v), np.arange(len(k), dtype=np.int32), kp, vp, 128)
    for pool, kind, x in ((kp, kinds[0], k), (vp, kinds[1], v)):
        assert np.array_equal(pool.cpu().numpy()[:, 0, 0], encode(kind, x)[:, 0])


@pytest.mark.parametrize("kinds", KINDS[1:3])
def test_append_strides(gpu, kinds):
    import torch

    k, v = values(3, (9, 2, 64)), values(4, (9, 2, 64))
    kt, vt = up(gpu, k), up(gpu, v)
    slots = np.arange(9, dtype=np.int32)[::-1].copy()
    for a, b in ((kt.permute(2, 1, 0).contiguous().permute(2, 1, 0), vt), (torch.cat([kt[..., :1], kt], 2)[..., 1:], torch.cat([vt[:, :, :3], vt], 2)[..., 3:]),
                 (torch.stack([kt, kt], 3)[..., 0], vt.transpose(0, 1).contiguous().transpose(0, 1))):
        kp, vp, _ = pool_tensors(gpu, kinds, 3, 2, 4, 64, "apart")
        append(gpu, kinds, a, b, slots, kp, vp, 64)
        for pool, kind, x in ((kp, kinds[0], k), (vp, kinds[1], v)):
            at = torch.from_numpy(slots).to(gpu).long()
            assert np.array_equal(pool[at // 4, :, at % 4].cpu().numpy(), encode(kind, x))


@pytest.mark.parametrize("tokens", [2, 300, 5000, (1 << 17) + 1000])
def test_append_of_one_slot_named_by_all(gpu, tokens):
    import torch

    kp, vp, _ = pool_tensors(gpu, KINDS[1], 4, 1, 8, 32, "token")
    k = (torch.arange(tokens, device=gpu, dtype=torch.float32)[:, None, None] * torch.ones(1, 1, 32, device=gpu)).contiguous()
    append(gpu, KINDS[1], k, -k, np.full(tokens, 9, np.int32), kp, vp, 32)
    last = np.full((1, 32), tokens - 1, np.float32)
    assert np.array_equal(kp[1, :, 1].cpu().numpy(), encode("q8_0", last)) and np.array_equal(vp[1, :, 1].cpu().numpy(), encode("q4_0", -last))


# ---- read back ----------------------------------------------------------------------------------


@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("kv,page,dim,tokens", [(1, 1, 32, 1), (2, 16, 64, 5), (3, 7, 96, 100), (8, 16, 128, 64), (1, 64, 256, 2100), (1, 5, 1056, 30)])
def test_read_gives_each_slots_values(gpu, kinds, order, kv, page, dim, tokens):
    import torch

    pages = 40
    kp, vp, store = pool_tensors(gpu, kinds, pages, kv, page, dim, order, seed=dim)
    before = store.clone()
    slots = rng(tokens).integers(0, pages * page, tokens).astype(np.int32)  # some more than once
    slots[1::7], slots[4::9] = -3, pages * page
    k, v = (torch.full((tokens, kv, dim), 7.0, device=gpu) for _ in range(2))
    run(eh.OpPagedKvRead(pages_view(kp, kinds[0], dim), pages_view(vp, kinds[1], dim), view(up(gpu, slots)), out(k), out(v)))
    live = (slots >= 0) & (slots < pages * page)
    at = torch.from_numpy(slots[live]).to(gpu).long()
    for got, pool, kind in ((k, kp, kinds[0]), (v, vp, kinds[1])):
        got = got.cpu().numpy()
        assert np.array_equal(got[live].astype(np.float64), decode(kind, pool[at // page, :, at % page].cpu().numpy()))
        assert (got[~live] == 7.0).all()
    assert torch.equal(store, before)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("dim", [1, 20, 64, 136])
def test_read_of_halves(gpu, bf16, dim):
    import torch

    kind = torch.bfloat16 if bf16 else torch.float16
    kp, vp = (torch.randn(6, 4, 3, dim + 1, device=gpu).to(kind)[..., 1:].transpose(1, 2) for _ in range(2))
    kp[2, 0, 1, 0] = float("nan")
    vp[2, 1, 1, 0] = float("inf")
    slots = np.array([9, 0, -1, 23, 9, 24], np.int32)
    k, v = (torch.full((6, 3, dim), 7.0, device=gpu) for _ in range(2))
    run(eh.OpPagedKvRead(view(kp), view(vp), view(up(gpu, slots)), out(k), out(v)))
    for got, pool in ((k, kp), (v, vp)):
        want = torch.stack([pool[s // 4, :, s % 4].float() if 0 <= s < 24 else torch.full((3, dim), 7.0, device=gpu) for s in slots.tolist()])
        assert torch.equal(torch.nan_to_num(got, nan=-5.0), torch.nan_to_num(want, nan=-5.0))


@pytest.mark.parametrize("kinds", KINDS[1:3])
def test_read_strides_and_scales_that_are_not_finite(gpu, kinds):
    import torch

    kp, vp, _ = pool_tensors(gpu, kinds, 5, 2, 4, 64, "token", seed=3)
    for pool in (kp, vp):  # of slot 6: an infinite scale, and a NaN
        pool[1, 0, 2, -2:] = torch.tensor([0x00, 0xFC], dtype=torch.uint8, device=gpu)
        pool[1, 1, 2, -4:-2] = torch.tensor([0x01, 0x7C], dtype=torch.uint8, device=gpu)
    slots = np.array([6, 19, 3], np.int32)
    both = torch.full((3, 4, 64), 7.0, device=gpu)  # keys and values of a token side by side
    wide = torch.full((2, 64, 7), 7.0, device=gpu)
    for k, v in ((both[:, :2], both[:, 2:]), (wide[..., 1:4].permute(2, 0, 1), wide[..., 4:].permute(2, 0, 1))):
        if k.stride(2) != 1:
            v = torch.full((3, 2, 129), 7.0, device=gpu)[..., 1::2]
        run(eh.OpPagedKvRead(pages_view(kp, kinds[0], 64), pages_view(vp, kinds[1], 64), view(up(gpu, slots)), out(k), out(v)))
        for got, pool, kind in ((k, kp, kinds[0]), (v, vp, kinds[1])):
            want = decode(kind, np.stack([pool[s // 4, :, s % 4].cpu().numpy() for s in slots]))
            assert np.isnan(want[0, 0, 32:]).all() and np.isnan(want[0, 1, :32]).all()
            assert np.array_equal(got.cpu().numpy().astype(np.float64), want, equal_nan=True)
    assert (wide[..., 0] == 7.0).all() and (wide[..., 4:] == 7.0).all()


# ---- attended over ------------------------------------------------------------------------------


def attend_case(gpu, kinds, heads, kv, dim, page, lengths, order, seed, spare=2, size=2.0):
    import torch

    most = max(1, max(-(-n // page) for n in lengths)) + 1
    pages = len(lengths) * most + spare
    kp, vp, store = pool_tensors(gpu, kinds, pages, kv, page, dim, order, seed)
    g = rng(seed + 9)
    table = g.permutation(pages)[: len(lengths) * most].reshape(len(lengths), most).astype(np.int32)
    q = (g.standard_normal((len(lengths), heads, dim)) * size).astype(np.float32)
    return {"kinds": kinds, "dim": dim, "q": up(gpu, q), "kp": kp, "vp": vp, "store": store, "table": up(gpu, table),
            "lengths": torch.tensor(lengths, dtype=torch.int32, device=gpu), "y": torch.full(q.shape, 5.0, device=gpu)}


def attend_event(c, **more):
    more.setdefault("scale", c["dim"] ** -0.5)
    return eh.OpPagedAttention(view(c["q"]), pages_view(c["kp"], c["kinds"][0], c["dim"]), pages_view(c["vp"], c["kinds"][1], c["dim"]), view(c["table"]),
                               view(c["lengths"]), out(c["y"]), **more)


def cached(c, s, window=0):
    import torch

    n, page = int(c["lengths"][s]), c["kp"].shape[2]
    at = torch.arange(max(0, n - window) if window else 0, n, device=c["q"].device)
    ids = c["table"][s].long()[at // page]
    return tuple(decode(kind, p[ids, :, at % page].cpu().numpy()) for kind, p in zip(c["kinds"], (c["kp"], c["vp"])))


def tolerance(c, v, tol):
    """attention()'s, and what a weight times its block's scale loses as two halves: 2^-22 of itself, which is within that,
    or 2^-35 of the block's largest such product, of n tokens with numbers up to the format's end.  In blocks of random
    numbers the largest value is an eighth of that end or more."""
    big = 8 * np.abs(v).reshape(*v.shape[:2], -1, 32).max((0, 3))  # [kv, block]
    share = np.repeat(np.repeat(big, 32, 1), c["q"].shape[1] // len(big), 0)
    return tol + share * len(v) * 2.0**-35


def check_attention(c, window=0, cap=0.0, scale=None, skip=()):
    got, dim = c["y"].cpu().numpy(), c["dim"]
    for s, n in enumerate(c["lengths"].tolist()):
        if s in skip:
            continue
        if n == 0:
            assert (got[s] == 0).all(), f"sequence {s} of length 0"
            continue
        k, v = cached(c, s, window)
        want, tol = attention(c["q"][s].double().cpu().numpy(), k, v, dim ** -0.5 if scale is None else scale, cap)
        within(got[s], want, tolerance(c, v, tol), f"sequence {s} of length {n}")


@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 32), (4, 4, 64), (8, 2, 96), (32, 8, 128), (5, 1, 160), (40, 2, 64), (16, 1, 256), (6, 2, 192), (17, 1, 224), (7, 7, 128)])
@pytest.mark.parametrize("page,order", [(16, "token"), (1, "head"), (24, "both"), (64, "apart")])
def test_attention_matches_the_formula(gpu, kinds, heads, kv, dim, page, order):
    lengths = [1, 0, 15, 16, 17, 63, 64, 65, 129, 700]
    c = attend_case(gpu, kinds, heads, kv, dim, page, lengths, order, heads + dim)
    run(attend_event(c))
    check_attention(c)
    first = c["y"].clone()
    c["y"].fill_(-1)
    run(attend_event(c))
    assert (first == c["y"]).all()


@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("dim", range(32, 257, 32))
@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 9, 16])
def test_attention_of_every_width_and_group(gpu, kinds, dim, group):
    c = attend_case(gpu, kinds, 2 * group, 2, dim, 16, [1, 40, 300, 0, 515], "token", dim + group)
    run(attend_event(c))
    check_attention(c)


@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("window,cap,scale", [(1, 0.0, 0.1), (33, 0.0, 0.2), (128, 30.0, 0.3), (1000, 5.0, -0.2), (10**9, 0.0, 0.0), (0, 50.0, 2.0)])
def test_attention_windows_caps_and_scales(gpu, kinds, window, cap, scale):
    c = attend_case(gpu, kinds, 6, 2, 128, 16, [1, 5, 130, 1200, 0, 2049], "token", 7)
    run(attend_event(c, window=window, soft_cap=cap, scale=scale))
    check_attention(c, window, cap, scale)


@pytest.mark.parametrize("kinds", [KINDS[0], KINDS[3]])
@pytest.mark.parametrize("seqs,low,high,heads,kv,dim", [(1, 9000, 9000, 8, 2, 128), (70, 1, 300, 4, 1, 64), (300, 3, 40, 8, 2, 64), (2, 3000, 5000, 8, 8, 256), (3, 500, 3000, 32, 32, 64), (2, 700, 1500, 48, 48, 128), (1, 1, 1, 64, 64, 32), (1, 60000, 60000, 4, 1, 64), (1, 50000, 50000, 16, 1, 96)])
def test_attention_of_long_and_many_sequences(gpu, kinds, seqs, low, high, heads, kv, dim):
    lengths = rng(seqs).integers(low, high + 1, seqs).tolist()
    c = attend_case(gpu, kinds, heads, kv, dim, 16, lengths, "token", seqs)
    run(attend_event(c))
    check_attention(c, skip=set(range(40, seqs)))


@pytest.mark.parametrize("kinds", KINDS)
def test_attention_reads_nothing_behind_a_sequence(gpu, kinds):
    """What lies behind a length, or before a window, does not count: NaN scales, pages outside the pool, another's tokens."""
    import torch

    lengths = [5, 40, 129, 0]
    c = attend_case(gpu, kinds, 4, 2, 64, 16, lengths, "head", 31)
    run(attend_event(c, window=37))
    want = c["y"].clone()
    nan = torch.tensor([0x00, 0x7E], dtype=torch.uint8, device=gpu)
    for s, n in enumerate(lengths):
        pages = c["table"][s].tolist()
        for j in list(range(n, len(pages) * 16)) + list(range(0, max(0, n - 37))):
            for pool in (c["kp"], c["vp"]):
                pool[pages[j // 16], :, j % 16, -4:] = torch.cat([nan, nan])
        c["table"][s, -(-n // 16) if n else 0:] = 10**6
    c["y"].fill_(5.0)
    run(attend_event(c, window=37))
    assert torch.equal(c["y"], want)


@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 1)])
def test_attention_blocks_of_very_different_scales(gpu, kinds, heads, kv):
    """Values' scales spread over f16's whole range between blocks and along the tokens, zeros among them."""
    import torch

    c = attend_case(gpu, kinds, heads, kv, 128, 16, [3, 200, 1000], "token", 41)
    pages = c["vp"].shape[0]
    g = rng(42)
    d = (np.exp2(g.uniform(-24, 12, (pages, kv, 16, 4))) * np.exp2(np.array([0.0, -12, -12, 2]))).astype(np.float16)
    d[g.random(d.shape) < 0.1] = 0
    d[:, :, :, 2] = 0
    c["vp"][..., -8:] = up(gpu, d.view(np.uint8).reshape(pages, kv, 16, 8))
    run(attend_event(c))
    check_attention(c)
    assert (c["y"][..., 64:96] == 0).all()
    assert torch.isfinite(c["y"]).all()


@pytest.mark.parametrize("kinds", KINDS)
def test_attention_scales_that_are_not_finite(gpu, kinds):
    """A NaN block of a key makes its head NaN, one of a value its 32 dims, at any distance; infinite scales are NaN."""
    import torch

    c = attend_case(gpu, kinds, 4, 2, 128, 16, [300, 300, 300], "token", 51)
    at = lambda s, j: (int(c["table"][s, j // 16]), j % 16)  # noqa: E731
    inf, nan = (torch.tensor(b, dtype=torch.uint8, device=gpu) for b in ([0x00, 0x7C], [0x34, 0x7E]))
    page, tok = at(0, 250)
    c["kp"][page, 0, tok, -4:-2] = inf
    page, tok = at(1, 17)
    c["vp"][page, 1, tok, -8:-6] = nan
    page, tok = at(2, 299)
    c["vp"][page, 1, tok, -2:] = inf
    run(attend_event(c))
    with np.errstate(invalid="ignore"):
        check_attention(c)
    y = c["y"].cpu().numpy()
    assert np.isnan(y[0, :2]).all() and np.isfinite(y[0, 2:]).all()
    assert np.isnan(y[1, 2:, :32]).all() and np.isfinite(y[1, 2:, 32:]).all() and np.isfinite(y[1, :2]).all()
    assert np.isnan(y[2, 2:, 96:]).all() and np.isfinite(y[2, 2:, :96]).all()


def test_attention_of_queries_that_are_not_finite(gpu):
    """A NaN or an infinity in q: its own head is as the formula, the others stay; with a cap infinite scores are finite."""
    for kinds in KINDS:
        c = attend_case(gpu, kinds, 4, 2, 64, 16, [200, 3000], "token", 61)
        c["kp"][..., 0] = 0x11  # no number of value 0's is 0
        c["q"][0, 1, 7], c["q"][1, 2, 0] = float("nan"), float("inf")
        for cap in (0.0, 20.0):
            run(attend_event(c, soft_cap=cap))
            with np.errstate(invalid="ignore"):
                check_attention(c, cap=cap)
            y = c["y"].cpu().numpy()
            assert np.isnan(y[0, 1]).all() and np.isfinite(y[0, [0, 2, 3]]).all() and np.isfinite(y[1, [0, 1, 3]]).all()


@pytest.mark.parametrize("size", [1e-30, 1e-10, 1e4, 1e18])
def test_attention_of_queries_of_any_size(gpu, size):
    c = attend_case(gpu, KINDS[3], 4, 2, 64, 16, [1, 100, 700], "token", 71, size=size)
    run(attend_event(c, scale=0.1 / size))
    check_attention(c, scale=float(np.float32(0.1 / size)))


@pytest.mark.parametrize("kinds", [KINDS[1], KINDS[3]])
def test_attention_refuses_to_read_outside_the_pool(gpu, kinds):
    import torch

    c = attend_case(gpu, kinds, 4, 2, 64, 16, [40, 40, 40, 40, 40], "token", 81)
    pages = c["kp"].shape[0]
    c["table"][0, 1], c["table"][1, 2] = -1, pages
    c["lengths"][2], c["lengths"][3] = -7, c["table"].shape[1] * 16 + 1
    run(attend_event(c))
    assert torch.isnan(c["y"][:4]).all()
    check_attention(c, skip={0, 1, 2, 3})


@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("heads,kv,dim", [(6, 2, 64), (20, 1, 96)])
def test_attention_strides(gpu, kinds, heads, kv, dim):
    import torch

    c = attend_case(gpu, kinds, heads, kv, dim, 16, [9, 150, 700], "apart", 91)
    run(attend_event(c))
    want = c["y"].clone()
    check_attention(c)
    wide = torch.full((3, heads, 2 * dim + 1), 5.0, device=gpu)
    c["y"] = wide[..., 1::2]
    c["q"] = torch.stack([c["q"], c["q"] + 9], 3)[..., 0].transpose(0, 1).contiguous().transpose(0, 1)
    c["table"] = c["table"].t().contiguous().t()
    c["lengths"] = torch.stack([c["lengths"], c["lengths"] * 0], 1)[:, 0]
    run(attend_event(c))
    assert torch.equal(c["y"], want) and (wide[..., ::2] == 5.0).all()


@pytest.mark.parametrize("kinds", [KINDS[0], KINDS[3]])
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 32), (8, 2, 128), (16, 1, 256)])
def test_attention_counts_every_position_once(gpu, kinds, heads, kv, dim):
    """Equal scores: the mean of whole numbers, each weight's product exact, so the result is but for the last division."""
    lengths = [1, 31, 32, 33, 127, 128, 129, 1000, 2047]
    c = attend_case(gpu, kinds, heads, kv, dim, 16, lengths, "token", 95)
    c["q"].zero_()
    blocks = dim // 32
    one = np.full((c["vp"].shape[0], kv, 16, blocks), 0.5, np.float16)
    c["vp"][..., -2 * blocks:] = up(gpu, one.view(np.uint8).reshape(*one.shape[:3], -1))
    run(attend_event(c))
    got = c["y"].cpu().numpy()
    for s, n in enumerate(lengths):
        _, v = cached(c, s)
        mean = np.repeat(v.sum(0), heads // kv, 0) / n
        assert (np.abs(got[s] - mean) <= np.abs(mean) * 2.0**-22).all(), n


def test_a_cache_past_32_bit_offsets(gpu):
    """Pages behind 2^33 bytes of a pool: appended to, read back and attended over."""
    import torch

    kv, dim, page = 4, 128, 64
    row = dim // 32 * SIZE["q8_0"]
    pages = 2**33 // (kv * page * row) + 40
    kp, vp = (torch.zeros(pages, kv, page, row, dtype=torch.uint8, device=gpu) for _ in range(2))
    tokens = 300
    k, v = values(1, (tokens, kv, dim)), values(2, (tokens, kv, dim))
    ids = np.concatenate([[3], pages - 1 - np.arange(6)])[: -(-tokens // page)]
    at = np.arange(tokens)
    slots = (ids[at // page] * page + at % page).astype(np.int32)
    append(gpu, ("q8_0", "q8_0"), up(gpu, k), up(gpu, v), slots, kp, vp, dim)
    kb, vb = torch.zeros(tokens, kv, dim, device=gpu), torch.zeros(tokens, kv, dim, device=gpu)
    run(eh.OpPagedKvRead(pages_view(kp, "q8_0", dim), pages_view(vp, "q8_0", dim), view(up(gpu, slots)), out(kb), out(vb)))
    for got, x in ((kb, k), (vb, v)):
        assert np.array_equal(got.cpu().numpy().astype(np.float64), decode("q8_0", encode("q8_0", x)))
    c = {"kinds": ("q8_0", "q8_0"), "dim": dim, "q": up(gpu, (rng(5).standard_normal((1, 8, dim)) * 0.1).astype(np.float32)), "kp": kp, "vp": vp,
         "table": up(gpu, ids[None].astype(np.int32)), "lengths": torch.tensor([tokens], dtype=torch.int32, device=gpu), "y": torch.zeros(1, 8, dim, device=gpu)}
    run(attend_event(c, scale=1e-6))
    check_attention(c, scale=1e-6)


# ---- together ------------------------------------------------------------------------------------


class Layer:
    """A decoder layer's new tokens into a packed cache and out of it: positions, quantised keys and values, attention."""

    def __init__(self, gpu, kinds, seed=5):
        import torch

        g = rng(seed)
        self.kinds, self.seqs, self.heads, self.kv, self.dim, self.page = kinds, 3, 8, 2, 128, 16
        new = lambda n: up(gpu, g.standard_normal((self.seqs, n, self.dim)).astype(np.float32))  # noqa: E731
        self.q, self.k, self.v = new(self.heads), new(self.kv), new(self.kv)
        self.kp, self.vp, self.store = pool_tensors(gpu, kinds, 40, self.kv, self.page, self.dim, "token", seed)
        self.table = up(gpu, g.permutation(40)[:30].reshape(3, 10).astype(np.int32))
        self.lengths = up(gpu, np.array([1, 24, 61], np.int32))
        self.slots, self.positions = torch.zeros(3, dtype=torch.int32, device=gpu), torch.zeros(3, 3, dtype=torch.int32, device=gpu)
        self.qr, self.kr, self.y = torch.zeros_like(self.q), torch.zeros_like(self.k), torch.zeros_like(self.q)
        self.kb, self.vb = torch.zeros_like(self.k), torch.zeros_like(self.v)
        view_of = lambda i, mut=False: pages_view((self.kp, self.vp)[i], kinds[i], self.dim, mut)  # noqa: E731
        self.events = [
            eh.OpRope(view(self.q), out(self.qr), view(self.positions), [16, 24, 24], k=view(self.k), k_out=out(self.kr), base=1e6),
            eh.OpPagedKvAppend(view(self.kr), view(self.v), view(self.slots), view_of(0, True), view_of(1, True)),
            eh.OpPagedAttention(view(self.qr), view_of(0), view_of(1), view(self.table), view(self.lengths), out(self.y), scale=self.dim ** -0.5),
            eh.OpPagedKvRead(view_of(0), view_of(1), view(self.slots), out(self.kb), out(self.vb)),
        ]

    def place(self, step):
        """Slots and positions of each sequence's newest token."""
        import torch

        last = self.lengths.long() - 1
        self.slots.copy_((self.table.gather(1, (last // self.page)[:, None])[:, 0].long() * self.page + last % self.page).to(torch.int32))
        self.positions.copy_(torch.stack([self.lengths + 1000, self.lengths + step, self.lengths * 2]))

    def outputs(self):
        return [t.clone() for t in (self.qr, self.kr, self.y, self.kb, self.vb, self.store)]


@pytest.mark.parametrize("kinds", KINDS)
def test_a_layers_step_through_all_of_them(gpu, kinds):
    import torch

    st = Layer(gpu, kinds)
    kernel = eh.Kernel(synchronous=False)
    n = lambda t: t.cpu().numpy()  # noqa: E731
    for step in range(3):
        st.place(step)
        for e in st.events:
            assert kernel.process_event(e) == eh.Status.OK, eh.last_error()
        torch.cuda.synchronize()
        within(n(st.qr), *rope(n(st.q), n(st.positions), [16, 24, 24], base=1e6), "q")
        within(n(st.kr), *rope(n(st.k), n(st.positions), [16, 24, 24], base=1e6), "k")
        for got, kind, x in ((st.kb, kinds[0], st.kr), (st.vb, kinds[1], st.v)):
            assert np.array_equal(n(got).astype(np.float64), decode(kind, encode(kind, n(x))))
        check_attention({"kinds": kinds, "dim": st.dim, "q": st.qr, "kp": st.kp, "vp": st.vp, "table": st.table, "lengths": st.lengths, "y": st.y})
        st.lengths += 1


@pytest.mark.parametrize("kinds", [KINDS[1], KINDS[3]])
def test_a_captured_layer_follows_its_cache(gpu, kinds):
    """Captured once and replayed: positions, slots, lengths and pages are read when it runs."""
    import torch

    eager, graphed = Layer(gpu, kinds), Layer(gpu, kinds)
    side = torch.cuda.Stream()
    kernel = eh.Kernel(side.cuda_stream, synchronous=False)
    with torch.cuda.stream(side):  # sizes the stream's workspace
        graphed.place(0)
        kept = graphed.store.clone()
        for e in graphed.events:
            assert kernel.process_event(e) == eh.Status.OK, eh.last_error()
        side.synchronize()
        graphed.store.copy_(kept)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for e in graphed.events:
            assert kernel.process_event(e) == eh.Status.OK, eh.last_error()
    plain = eh.Kernel(synchronous=False)
    for step in range(4):
        for st in (eager, graphed):
            st.place(step)
        for e in eager.events:
            assert plain.process_event(e) == eh.Status.OK
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager.outputs(), graphed.outputs()):
            assert torch.equal(a, b), step
        for st in (eager, graphed):
            st.lengths += 1
            st.k.mul_(1.1)


def test_streams_do_not_share_scratch(gpu):
    import torch

    streams = [torch.cuda.Stream() for _ in range(2)]
    cases = [attend_case(gpu, KINDS[3 * i], 8, 2, 128, 16, [900, 3, 2500], "token", 40 + i) for i in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, c in zip(streams, cases):
            assert eh.Kernel(s.cuda_stream, synchronous=False).process_event(attend_event(c)) == eh.Status.OK
    torch.cuda.synchronize()
    for c in cases:
        check_attention(c)


def test_scratch_does_not_grow_under_capture(gpu):
    """Refused where the call's scratch would grow; a reserve ahead lets it in."""
    import ctypes

    import torch

    handle = ctypes.c_void_p()  # one of torch's streams may have scratch already
    assert eh.load().emel_stream_create(ctypes.byref(handle)) == eh.Status.OK
    stream = torch.cuda.ExternalStream(handle.value)
    kernel = eh.Kernel(stream.cuda_stream, synchronous=False)
    c = attend_case(gpu, KINDS[0], 8, 2, 128, 16, [900, 3], "token", 44)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        c["q"].mul_(1.0)
        assert kernel.process_event(attend_event(c)) == eh.Status.STREAM_CAPTURE
    assert eh.stream_reserve(32 << 20, 1 << 20, stream.cuda_stream) == eh.Status.OK
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        assert kernel.process_event(attend_event(c)) == eh.Status.OK
    for _ in range(3):
        c["y"].fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        check_attention(c)
    del graph
    assert eh.load().emel_stream_destroy(handle) == eh.Status.OK


def test_two_host_threads_on_one_stream(gpu):
    import threading

    import torch

    stream = torch.cuda.Stream()
    cases = [attend_case(gpu, KINDS[i], 8, 2, 64 * i, 16, [700, 40, 1500], "token", 50 + i) for i in (1, 2, 3)]
    torch.cuda.synchronize()
    got = []

    def work(c):
        kernel = eh.Kernel(stream.cuda_stream, synchronous=False)
        got.append([kernel.process_event(attend_event(c)) for _ in range(20)])

    threads = [threading.Thread(target=work, args=(c,)) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert got == [[eh.Status.OK] * 20] * 3
    for c in cases:
        check_attention(c)
