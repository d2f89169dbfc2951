"""GPU: attention over packed pages where scales and weights go apart: what a token of next to no weight has for scales, or one
of almost all weight lacks, costs the others' values nothing."""
import numpy as np
import pytest

from helpers import rng
from packed_cache_reference import decode
from test_gpu_packed_cache import KINDS, attend_case, attend_event, cached, run, up, within

pytestmark = pytest.mark.gpu

# one column a head, two, four and eight, with whole sets of blocks and without
SHAPES = [(4, 4, 128), (16, 2, 128), (32, 2, 128), (2, 2, 32), (3, 1, 64), (12, 1, 64), (4, 2, 96), (10, 2, 160), (2, 1, 224), (9, 1, 224), (2, 1, 256), (16, 2, 256), (24, 1, 256)]
TOP = {"q8_0": 127, "q4_0": 8}


def even(gpu, kinds, heads, kv, dim, lengths, seed, small):
    """Keys whose scores are within some 5 of one another, and values with scales around `small`."""
    c = attend_case(gpu, kinds, heads, kv, dim, 16, lengths, "token", seed)
    g = rng(seed + 1)
    pages, blocks = c["kp"].shape[0], dim // 32
    size = {"q8_0": 0.005, "q4_0": 0.08}[kinds[0]]
    c["kp"][..., -2 * blocks:] = up(gpu, np.full((pages, kv, 16, blocks), size, np.float16).view(np.uint8))
    d = (small * g.uniform(0.5, 2.0, (pages, kv, 16, blocks)) * g.choice([-1, 1], (pages, kv, 16, blocks))).astype(np.float16)
    c["vp"][..., -2 * blocks:] = up(gpu, d.view(np.uint8))
    c["q"][..., 0] = 8.0
    return c


def special(gpu, c, s, j, score, scale):
    """Token j of sequence s gets this score (scale dim^-0.5) under every head, and values with this scale."""
    page, tok = int(c["table"][s, j // 16]), j % 16
    c["kp"][page, :, tok] = key(gpu, c, score)
    c["vp"][page, :, tok, -c["dim"] // 16:] = up(gpu, np.full(c["dim"] // 32, scale, np.float16).view(np.uint8))


def key(gpu, c, score):
    """A key's row: the lowest number in front of the queries' 8, nothing else."""
    blocks, kind = c["dim"] // 32, c["kinds"][0]
    row = np.full(c["kp"].shape[-1] - 2 * blocks, 0x88 if kind == "q4_0" else 0, np.uint8)
    row[0] = 0x80 if kind == "q4_0" else 256 - TOP[kind]
    scales = np.zeros(blocks, np.float16)
    scales[0] = score * c["dim"]**0.5 / 8.0 / -TOP[kind]
    return up(gpu, np.concatenate([row, scales.view(np.uint8)]))


def formula(q, k, v, rows, kind, dim):
    """(out [heads, dim], tolerance): a score's error as attention()'s has it, token by token, so that one of no weight
    widens nothing; out = sum p v moves by sum p dz |v| + (sum p dz) (sum p |v|) with it, and by 2^-22 and the sum's n + 64
    steps of 2^-23; a weight by its block's scale by 2^-22 of itself, which the like of both hold, or by 2^-36 of
    the largest, each times its number."""
    heads, n, kv = len(q), *k.shape[:2]
    blocks = dim // 32
    d = np.abs(np.ascontiguousarray(rows[..., -2 * blocks:]).view(np.float16).astype(np.float64))  # [n, kv, blocks]
    out, tol = np.zeros((heads, dim)), np.zeros((heads, dim))
    for h in range(heads):
        at = h // (heads // kv)
        kk, vv = k[:, at], v[:, at]
        z = dim**-0.5 * (kk @ q[h])
        dz = dim**-0.5 * (np.abs(kk) @ np.abs(q[h])) * (dim + 4) * 2.0**-23 + (np.abs(z) + np.abs(z.max()) + 1) * 2.0**-21
        e = np.exp(z - z.max())
        p = e / e.sum()
        out[h] = p @ vv
        share = n * TOP[kind] * (p[:, None] * d[:, at]).max(0) * 2.0**-36
        tol[h] = (p * dz) @ np.abs(vv) + ((p @ dz) + (n + 64) * 2.0**-23) * (p @ np.abs(vv)) + np.repeat(share, 32) + 2.0**-110 * TOP[kind] * n
    return out, tol


def check(c):
    got = c["y"].cpu().numpy()
    assert np.isfinite(got).all()
    for s, n in enumerate(c["lengths"].tolist()):
        k, v = cached(c, s)
        ids = c["table"][s].long()[[j // 16 for j in range(n)]]
        rows = c["vp"][ids, :, [j % 16 for j in range(n)]].cpu().numpy()
        want, tol = formula(c["q"][s].double().cpu().numpy(), k, v, rows, c["kinds"][1], c["dim"])
        within(got[s], want, tol, f"sequence {s} of length {n}")


@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("score,scale,small", [(-100.0, 60000.0, 1e-6), (-40.0, 1000.0, 1e-4), (-15.0, 100.0, 1e-4), (-1000.0, 60000.0, 1e-3)])
def test_a_large_scale_of_little_weight(gpu, kinds, heads, kv, dim, score, scale, small):
    """One token whose values tower over the rest and whose weight is next to none, at the start, within and at the end."""
    lengths = [33, 300, 700, 129]
    c = even(gpu, kinds, heads, kv, dim, lengths, heads + dim, small)
    for s, j in enumerate((0, 150, 699, 128)):
        special(gpu, c, s, j, score, scale)
    run(attend_event(c))
    check(c)


@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("scale", [0.0, 6e-8, 1e-3])
def test_a_token_of_almost_all_weight(gpu, kinds, heads, kv, dim, scale):
    """A first token that takes all but some 2^-20 (or 2^-45) of the weight and has no values or small ones: the others' count as
    they are, relative to the largest product of a weight and a scale."""
    c = even(gpu, kinds, heads, kv, dim, [200, 31, 400, 160], heads + dim + 1, 0.5)
    for s, (j, score) in enumerate(((0, 14.0), (5, 30.0), (0, 31.0), (159, 20.0))):
        special(gpu, c, s, j, score, scale)
    run(attend_event(c))
    check(c)


@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
def test_weight_moves_from_large_scales_to_small_ones(gpu, kinds, heads, kv, dim):
    """Tokens with large scales lead until later ones, with scales far smaller, take all the weight."""
    c = even(gpu, kinds, heads, kv, dim, [500, 64, 900], heads + dim + 2, 1e-5)
    for s, (first, later) in enumerate(((0, 499), (1, 40), (7, 300))):
        special(gpu, c, s, first, 10.0, 1000.0)
        special(gpu, c, s, first + 33 if s != 1 else 20, 25.0, 0.5)
        special(gpu, c, s, later, 80.0, 2e-5)
    run(attend_event(c))
    check(c)


@pytest.mark.parametrize("kinds", [KINDS[0], KINDS[3]])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 128), (4, 1, 128), (2, 1, 224), (16, 1, 256)])
@pytest.mark.parametrize("empty", [False, True])
def test_a_token_with_all_the_weight_is_its_values(gpu, kinds, heads, kv, dim, empty):
    """Far into sequences of several steps a wave, where the others have e^-45 of its weight each: a result is the value but for the
    rounding of the weight's product (2^-24), of its halves (2^-23), of their sum, of the sum's inverse and of the last
    product (2^-24 each), so within 2^-21, whether or not the first block has values."""
    lengths = [7000] * 40
    c = even(gpu, kinds, heads, kv, dim, lengths, heads + dim + 3, 0.5)
    g = rng(heads + dim + 4)
    at = g.integers(1000, 7000, 40).tolist()
    places = [int(c["table"][s, j // 16]) for s, j in enumerate(at)], slice(None), [j % 16 for j in at]
    kept = c["kp"][places].clone()  # scores within 5 of 0
    c["kp"][:] = key(gpu, c, -50.0)
    c["kp"][places] = kept
    if empty:
        c["vp"][..., -dim // 16: 2 - dim // 16] = 0
    run(attend_event(c))
    got = c["y"].cpu().numpy().astype(np.float64)
    for s, j in enumerate(at):
        v = decode(kinds[1], c["vp"][int(c["table"][s, j // 16]), :, j % 16].cpu().numpy())
        want = np.repeat(v, heads // kv, 0)
        # the others' values: 127 at most
        within(got[s], want, np.abs(want) * 2.0**-21 + 7000 * 128 * 2.0**-57, f"sequence {s}")
