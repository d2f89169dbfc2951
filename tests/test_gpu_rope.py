"""GPU: rotary positions of several axes against their formula in 64 bits."""
from decimal import Decimal, localcontext

import numpy as np
import pytest

import emel_hip as eh
from decode_reference import out, view
from helpers import rng
from rope_reference import rope

pytestmark = pytest.mark.gpu


def run(event, stream=None):
    status = eh.Kernel(stream).process_event(event)
    assert status == eh.Status.OK, eh.last_error()


def within(got, want, tol, what):
    got = np.asarray(got, np.float64)
    off = np.abs(got - want)
    ok = (off <= tol) | (np.isnan(got) & np.isnan(want)) | (got == want)
    assert ok.all(), f"{what}: {int((~ok).sum())} outside; worst {np.nanmax(off / np.maximum(tol, 1e-300)):.3g} of the tolerance"


def arrays(seed, tokens, heads, kv, dim, axes, far=5000):
    g = rng(seed)
    q, k = g.standard_normal((tokens, heads, dim)).astype(np.float32), g.standard_normal((tokens, kv, dim)).astype(np.float32)
    return q, k, g.integers(-far // 8, far, (axes, tokens)).astype(np.int32)


def turned(gpu, q, k, pos, sections, place=False, factors=None, own=False, **kw):
    import torch

    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(gpu)  # noqa: E731
    qt, kt, pt = t(q), t(k), t(pos)
    qo, ko = (qt, kt) if place else (torch.full_like(qt, 7.0), torch.full_like(kt, 7.0))
    run(eh.OpRope(view(qt), out(qo), view(pt), sections, k=view(kt), k_out=out(ko), factors=None if factors is None else view(t(factors)), own_frequencies=own, **kw))
    if not place:
        assert np.array_equal(qt.cpu().numpy(), q, equal_nan=True) and np.array_equal(kt.cpu().numpy(), k)
    return qo.cpu().numpy(), ko.cpu().numpy()


SHAPES = [(2, [1]), (6, [1, 1]), (32, [16]), (64, [8, 12, 12]), (80, [20, 20]), (80, [13]), (128, [16, 24, 24]), (128, [16, 16, 16]), (130, [40, 1, 2, 22]), (256, [64, 64]),
          (256, [0, 100, 0, 0]), (1100, [100, 200, 250])]


@pytest.mark.parametrize("dim,sections", SHAPES)
@pytest.mark.parametrize("tokens,heads,kv", [(1, 1, 1), (1, 32, 8), (5, 7, 1), (67, 3, 3), (700, 4, 1)])
@pytest.mark.parametrize("adjacent,in_turn,own", [(False, False, False), (True, False, True), (False, True, False), (True, True, True)])
def test_matches_the_formula(gpu, dim, sections, tokens, heads, kv, adjacent, in_turn, own):
    q, k, pos = arrays(dim + tokens, tokens, heads, kv, dim, len(sections))
    kw = dict(adjacent=adjacent, in_turn=in_turn, own=own)
    for got, x in zip(turned(gpu, q, k, pos, sections, **kw), (q, k)):
        within(got, *rope(x, pos, sections, **kw), f"{dim} {sections} {tokens}")


@pytest.mark.parametrize("dim,sections", SHAPES)
@pytest.mark.parametrize("adjacent", [False, True])
def test_in_place_factors_scale_and_magnitude(gpu, dim, sections, adjacent):
    q, k, pos = arrays(dim, 33, 5, 2, dim, len(sections))
    kw = dict(adjacent=adjacent, base=5e5, scale=0.37, magnitude=1.2, factors=rng(3).uniform(0.5, 8.0, sum(sections)).astype(np.float32))
    for got, x in zip(turned(gpu, q, k, pos, sections, place=True, **kw), (q, k)):
        within(got, *rope(x, pos, sections, **kw), f"{dim} {sections}")


@pytest.mark.parametrize("far", [2**20, 2**31 - 1])
def test_far_positions(gpu, far):
    q, k, pos = arrays(1, 50, 2, 1, 64, 2, far)
    pos[0, :4] = 2**31 - 1, -2**31, 0, -1
    for got, x in zip(turned(gpu, q, k, pos, [16, 16], base=1e6), (q, k)):
        within(got, *rope(x, pos, [16, 16], base=1e6), "far")


@pytest.mark.parametrize("dim,sections", [(80, [20, 13]), (96, [16, 16, 8])])
@pytest.mark.parametrize("adjacent,in_turn,own", [(False, True, False), (True, False, True)])
def test_backward_is_the_gradient(gpu, dim, sections, adjacent, in_turn, own):
    """<w, rope(x + e u) - rope(x - e u)> / 2e by the formula in 64 bits is <backward(w), u>, and so is autograd's."""
    import torch

    q, k, pos = arrays(9, 21, 3, 1, dim, len(sections))
    kw = dict(adjacent=adjacent, in_turn=in_turn, own=own, magnitude=0.8)
    wq, wk, _ = arrays(10, 21, 3, 1, dim, 1)
    for grad, x, w in zip(turned(gpu, wq, wk, pos, sections, backward=True, **kw), (q, k), (wq, wk)):
        within(grad, *rope(w, pos, sections, backward=True, **kw), "backward")
        u = rng(11).standard_normal(x.shape)
        ahead, back = (rope(x.astype(np.float64) + e * u, pos, sections, **kw)[0] for e in (1e-3, -1e-3))
        size = (np.abs(w) * np.abs(u)).sum()
        assert abs((w * (ahead - back) / 2e-3).sum() - (grad * u).sum()) <= size * 2.0**-20
    assert torch.isfinite(torch.from_numpy(grad)).all()


@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("dim,sections", [(64, [10, 12]), (72, [9, 11, 5])])
def test_strides_and_buffers_side_by_side(gpu, adjacent, dim, sections):
    """Inputs by steps and by columns, outputs within larger buffers whose rest stays, and a fused projection in place."""
    import torch

    tokens, heads, kv = 9, 4, 2
    q, k, pos = arrays(4, tokens, heads, kv, dim, len(sections))
    (wq, tq), (wk, tk) = (rope(x, pos, sections, adjacent=adjacent) for x in (q, k))
    t = lambda a: torch.from_numpy(a).to(gpu)  # noqa: E731
    p2 = t(np.stack([pos.T, pos.T + 1], 2))[:, :, 0].t()  # axes side by side, a gap after each
    assert np.array_equal(p2.cpu().numpy(), pos)
    for qt, kt in ((t(q).transpose(0, 1).contiguous().transpose(0, 1), t(k).permute(2, 1, 0).contiguous().permute(2, 1, 0)),
                   (torch.stack([t(q), t(q) * 0], 3)[..., 0], torch.cat([t(k)[..., :1], t(k)], 2)[..., 1:])):
        qo, ko = torch.full((heads, tokens, dim + 1), 5.0, device=gpu), torch.full((tokens, kv, 2 * dim), 5.0, device=gpu)
        run(eh.OpRope(view(qt), out(qo[:, :, 1:].transpose(0, 1)), view(p2), sections, k=view(kt), k_out=out(ko[:, :, ::2]), adjacent=adjacent))
        within(qo[:, :, 1:].transpose(0, 1).cpu().numpy(), wq, tq, "q")
        within(ko[:, :, ::2].cpu().numpy(), wk, tk, "k")
        assert (qo[:, :, 0] == 5.0).all() and (ko[:, :, 1::2] == 5.0).all()
    fused = torch.cat([t(q), t(k), t(k)], 1)
    qf, kf = fused[:, :heads], fused[:, heads:heads + kv]
    run(eh.OpRope(view(qf), out(qf), view(p2), sections, k=view(kf), k_out=out(kf), adjacent=adjacent))
    within(qf.cpu().numpy(), wq, tq, "fused q")
    within(kf.cpu().numpy(), wk, tk, "fused k")
    assert torch.equal(fused[:, heads + kv:], t(k))


def test_infinities_and_nan_stay_in_their_pairs(gpu):
    q, k, pos = arrays(6, 5, 2, 1, 64, 1)
    q[1, 0, 3], q[2, 1, 40], q[3, 0, 60] = np.inf, np.nan, -np.inf
    pos[0, 1] = pos[0, 3] = 0  # a turn of zero: inf * 0
    got, _ = turned(gpu, q, k, pos, [30])
    with np.errstate(invalid="ignore"):
        want, tol = rope(q, pos, [30])
    assert (np.isnan(got) == np.isnan(want)).all() and (got[~np.isfinite(want)] == want[~np.isfinite(want)])[~np.isnan(want[~np.isfinite(want)])].all()
    fine = np.isfinite(want)
    within(got[fine], want[fine], tol[fine], "the others")


def test_a_captured_rotation_follows_its_positions(gpu):
    import torch

    q, k, pos = arrays(8, 64, 8, 2, 128, 3)
    qt, kt, pt = (torch.from_numpy(a).to(gpu) for a in (q, k, pos))
    qo, ko = torch.empty_like(qt), torch.empty_like(kt)
    event = eh.OpRope(view(qt), out(qo), view(pt), [16, 24, 24], k=view(kt), k_out=out(ko))
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run_async = eh.Kernel(side.cuda_stream, synchronous=False)
        assert run_async.process_event(event) == eh.Status.OK, eh.last_error()
    for turn in range(3):
        new = pos + 1000 * turn
        pt.copy_(torch.from_numpy(new))
        qo.fill_(0.0)
        graph.replay()
        torch.cuda.synchronize()
        within(qo.cpu().numpy(), *rope(q, new, [16, 24, 24]), f"replay {turn}")
        within(ko.cpu().numpy(), *rope(k, new, [16, 24, 24]), f"replay {turn}")


def test_more_values_than_32_bits_count(gpu):
    """Tokens behind 2^32 values of a buffer, most of which no call reads."""
    import torch

    dim, far = 64, 2**32 // 64 + 5
    store = torch.zeros(far + 3, 1, dim, device=gpu)
    q, k, pos = arrays(12, 2, 1, 1, dim, 1)
    rows = torch.tensor([1, far + 1], device=gpu)
    store[rows] = torch.from_numpy(q).to(gpu)
    x = store.as_strided((2, 1, dim), (far * dim, dim, 1), dim)
    assert np.array_equal(x.cpu().numpy(), q)
    run(eh.OpRope(view(x), out(x), view(torch.from_numpy(pos).to(gpu)), [32]))
    within(store[rows].cpu().numpy(), *rope(q, pos, [32]), "far rows")
    assert int((store != 0).sum()) <= 2 * dim


def reduced_angles(positions, pairs, base, scale, factors):
    """(angles [tokens, pairs], reduced to a turn, what they were), from 90 digits."""
    with localcontext() as ctx:
        ctx.prec = 90
        pi = 4 * (4 * arctan_of_inverse(5) - arctan_of_inverse(239))
        rate = -Decimal(float(np.float32(base))).ln() / pairs
        out, size = np.zeros((len(positions), pairs)), np.zeros((len(positions), pairs))
        for i in range(pairs):
            freq = (i * rate).exp() * Decimal(float(np.float32(scale))) / Decimal(float(factors[i]))
            for t, p in enumerate(positions):
                angle = int(p) * freq
                out[t, i], size[t, i] = float(angle % (2 * pi)), abs(float(angle))
    return out, size


def arctan_of_inverse(n):
    power, total, k = Decimal(1) / n, Decimal(0), 0
    while abs(power) > Decimal(10) ** -95:
        total += (power if k % 2 == 0 else -power) / (2 * k + 1)
        power, k = power / (n * n), k + 1
    return total


@pytest.mark.parametrize("base,scale", [(1e4, 2.0**12), (5e6, 2.0**20), (5e6, 2.0**30), (3e38, 2.0**115), (1e-30, 2.0**-100)])
@pytest.mark.parametrize("adjacent", [False, True])
def test_angles_keep_50_bits(gpu, base, scale, adjacent):
    """An angle is off by 2^-50 of itself: as cos and sin count turns of 2^30 and more, f32's roundings hide no more than that.
    They are off by 2^-23 each, and the products and the sum round by 2^-24 each: 2^-22 of |x| + |y|."""
    pairs = 32
    q, _, pos = arrays(14, 40, 1, 1, 2 * pairs, 1, 2**31 - 1)
    pos[0, :3] = 2**31 - 1, -2**31, 1
    factors = rng(15).uniform(0.5, 8.0, pairs).astype(np.float32)
    got, _ = turned(gpu, q, q, pos, [pairs], base=base, scale=scale, factors=factors, adjacent=adjacent)
    angle, size = reduced_angles(pos[0], pairs, base, scale, factors)
    first, second = (slice(0, None, 2), slice(1, None, 2)) if adjacent else (slice(0, pairs), slice(pairs, None))
    x, y = q[:, 0, first].astype(np.float64), q[:, 0, second].astype(np.float64)
    tol = (np.abs(x) + np.abs(y)) * (2.0**-22 + size * 2.0**-50)
    within(got[:, 0, first], x * np.cos(angle) - y * np.sin(angle), tol, "first")
    within(got[:, 0, second], x * np.sin(angle) + y * np.cos(angle), tol, "second")
