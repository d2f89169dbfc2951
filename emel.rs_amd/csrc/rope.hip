// rope.hip -- rotary positions of several axes, turned into queries and keys.
#include <utility>

#include "common.hpp"
#include "launch.hpp"

namespace emel {
namespace {

// Pair i of a head turns by position * frequency.  A workgroup works its pairs'
// frequencies out, in quarter turns a position and in 64 bits, then the cos and
// sin of a tile of tokens, one of each a thread, and walks the tile's heads with
// them.  In quarter turns the reduction of far positions is exact: t - rint(t).  An
// exponent e rate is up to 128 and would lose a frequency 2^-47 of itself by its rounding: what
// that and rate's own leave out goes in as a factor 1 - ln(2) rest.  With u = 2^-53 an angle is
// then off by exp2's 2 u, 0.6 u of 2 / pi, u each of the products with scale, exp2, that
// factor, the pair's factor and the position, and 0.2 u of rate + rest: 2^-50 of itself, and by
// f32's rounding of what is left of it.
//
// Bound by the bytes, 4 read and 4 written a value: 8001 tokens of 40 heads of 128
// 60 us (5.4 TB/s), 73 with every thread working out its own pairs' angles for all
// heads over again.

typedef v4f v4f_any __attribute__((aligned(4)));

// cos and sin of t quarter turns: their series on [-pi/4, pi/4] (the next
// terms are below 2^-28 of the result), then the quadrant.
__device__ __forceinline__ void quarter_turns(double t, float &c, float &s)
{
    const double q = __builtin_rint(t);
    const float x = static_cast<float>((t - q) * 1.5707963267948966);
    const float z = x * x;
    float ps = __builtin_fmaf(z, 2.75573192e-6f, -1.98412698e-4f);
    ps = __builtin_fmaf(z, ps, 8.33333333e-3f);
    ps = __builtin_fmaf(z, ps, -1.66666667e-1f);
    const float sx = __builtin_fmaf(x * z, ps, x);
    float pc = __builtin_fmaf(z, -2.75573192e-7f, 2.48015873e-5f);
    pc = __builtin_fmaf(z, pc, -1.38888889e-3f);
    pc = __builtin_fmaf(z, pc, 4.16666667e-2f);
    pc = __builtin_fmaf(z, pc, -0.5f);
    const float cx = __builtin_fmaf(z, pc, 1.0f);
    const uint32_t n = static_cast<uint32_t>(q - 4.0 * __builtin_floor(q * 0.25));
    const float a = n & 1 ? sx : cx, b = n & 1 ? cx : sx;
    c = (n + 1) & 2 ? -a : a;
    s = n & 2 ? -b : b;
}

struct RopePlan {
    FastDiv items;   // of a head in a workgroup
    FastDiv turning; // pairs of a workgroup's items
    uint32_t rot;    // items of a head that turn; the others copy
    uint32_t all;    // items of a head
    uint32_t per;    // heads of a step
    uint32_t steps;  // of a token
    uint32_t tile;   // tokens of a workgroup
    uint32_t groups; // workgroups that share a tile's steps
    bool stream;     // outputs that the dies' caches do not hold, stored past them (60 us, 64 through them)
};

constexpr uint32_t kRopeTurns = 1024;     // angles of a tile
constexpr uint32_t kRopeGrid = 1u << 22;  // tiles of a launch, and its workgroups: threads are counted in 32 bits

// An item: four pairs, or eight values behind the pairs that are copied; one
// pair and two values where VEC is false.
template <bool VEC, bool ADJ>
__global__ __launch_bounds__(kBlock) void k_rope(RopeArgs a, RopePlan pl)
{
    constexpr uint32_t W = VEC ? 4 : 1;
    __shared__ double freq[W * kBlock];
    __shared__ uint8_t axis[W * kBlock];
    __shared__ __attribute__((aligned(16))) float cosines[kRopeTurns], sines[kRopeTurns];
    const uint32_t tid = threadIdx.x, first = blockIdx.y * kBlock; // the workgroup's items from `first` on
    const uint32_t slot = pl.items.div(tid), local = tid - slot * pl.items.d, item = local + first;
    const bool mine = slot < pl.per && item < pl.all, turns = item < pl.rot;
    const uint32_t left = a.pairs > first * W ? a.pairs - first * W : 0, pairs = left < pl.items.d * W ? left : pl.items.d * W;
    const uint32_t tile = blockIdx.x / pl.groups, group = blockIdx.x - tile * pl.groups;
    const uint32_t token0 = tile * pl.tile, tokens = a.tokens - token0 < pl.tile ? a.tokens - token0 : pl.tile;
    const uint32_t heads = a.q.heads + a.k.heads;

    // the first values of the item's pairs and their second ones
    const uint32_t d0 = turns ? (ADJ ? 2 * W * item : W * item) : 2 * a.pairs + 2 * W * (item - pl.rot);
    const uint32_t d1 = !turns || ADJ ? d0 + W : d0 + a.pairs;
    struct Unit {
        const float *x;
        float *y;
        int64_t st;
        float lo[W], hi[W];
    };
    auto ask = [&](uint32_t t, uint32_t step) {
        Unit n = {};
        const uint32_t h = step * pl.per + slot;
        if (!mine || h >= heads) return n;
        const RopeTensor &r = h >= a.q.heads ? a.k : a.q;
        const int64_t head = h >= a.q.heads ? h - a.q.heads : h;
        n.x = r.x + head * r.x_st[1] + static_cast<int64_t>(token0 + t) * r.x_st[2];
        n.y = r.y + head * r.y_st[1] + static_cast<int64_t>(token0 + t) * r.y_st[2];
        n.st = r.y_st[0];
        if constexpr (VEC) {
            const v4f p = *reinterpret_cast<const v4f_any *>(n.x + d0), q = *reinterpret_cast<const v4f_any *>(n.x + d1);
            for (int w = 0; w < 4; ++w) {
                n.lo[w] = p[w];
                n.hi[w] = q[w];
            }
        } else {
            n.lo[0] = n.x[d0 * r.x_st[0]];
            n.hi[0] = d1 < a.dim ? n.x[d1 * r.x_st[0]] : 0.0f;
        }
        return n;
    };
    Unit next = ask(0, group);

    for (uint32_t j = tid; j < pairs; j += kBlock) {
        const uint32_t i = first * W + j;
        RopeRun r = a.runs[0];
        for (int n = 1; n < 4; ++n)
            if (i >= a.runs[n].start) r = a.runs[n];
        const uint32_t at = i - r.start, round = r.live == 1 ? at : r.live == 2 ? at / 2 : r.live == 3 ? at / 3 : at / 4;
        const uint32_t x = (r.axes >> (2 * (at - round * r.live))) & 3u;
        const double rate = x == 0 ? a.rate[0] : x == 1 ? a.rate[1] : x == 2 ? a.rate[2] : a.rate[3];
        const float rest = x == 0 ? a.rest[0] : x == 1 ? a.rest[1] : x == 2 ? a.rest[2] : a.rest[3];
        const double e = a.own ? r.round + round : i, by = e * rate, left = __builtin_fma(e, rate, -by) + e * rest;
        const double f = a.quarters * exp2(-by);
        axis[j] = static_cast<uint8_t>(x);
        freq[j] = __builtin_fma(f, -0.6931471805599453 * left, f);
        if (a.factors) freq[j] /= static_cast<double>(a.factors[static_cast<int64_t>(i) * a.factors_st]);
    }
    __syncthreads();
    for (uint32_t e = tid; e < tokens * pairs; e += kBlock) {
        const uint32_t t = pl.tile == 1 ? 0 : pl.turning.div(e), j = e - t * pairs;
        const int32_t p = a.pos[static_cast<int64_t>(token0 + t) * a.pos_st[0] + axis[j] * a.pos_st[1]];
        float c, s;
        quarter_turns(p * freq[j], c, s);
        cosines[e] = c * a.magnitude;
        sines[e] = s * (a.back ? -a.magnitude : a.magnitude);
    }
    __syncthreads();
    for (uint32_t t = 0, step = group; t < tokens;) {
        const Unit n = next;
        const uint32_t at = t * pairs + local * W; // of the item's angles
        step += pl.groups;
        if (step >= pl.steps) {
            step = group;
            ++t;
        }
        if (t < tokens) next = ask(t, step); // ahead of this one's stores
        if (!n.y || (!turns && n.x == n.y)) continue;
        float o0[W], o1[W], c[W], s[W];
        for (uint32_t w = 0; w < W; ++w) {
            c[w] = turns ? cosines[at + w] : 1.0f;
            s[w] = turns ? sines[at + w] : 0.0f;
        }
        for (uint32_t w = 0; w < W; ++w) {
            if (!turns) {
                o0[w] = n.lo[w];
                o1[w] = n.hi[w];
            } else if constexpr (VEC && ADJ) { // pairs 0, 1 in lo, 2, 3 in hi
                const float *v = w < 2 ? n.lo : n.hi;
                const float e = v[2 * (w % 2)], f = v[2 * (w % 2) + 1];
                float *o = w < 2 ? o0 : o1;
                o[2 * (w % 2)] = __builtin_fmaf(e, c[w], -(f * s[w]));
                o[2 * (w % 2) + 1] = __builtin_fmaf(e, s[w], f * c[w]);
            } else {
                o0[w] = __builtin_fmaf(n.lo[w], c[w], -(n.hi[w] * s[w]));
                o1[w] = __builtin_fmaf(n.lo[w], s[w], n.hi[w] * c[w]);
            }
        }
        if constexpr (VEC) {
            const v4f p = {o0[0], o0[1], o0[2], o0[3]}, q = {o1[0], o1[1], o1[2], o1[3]};
            if (pl.stream) {
                __builtin_nontemporal_store(p, reinterpret_cast<v4f_any *>(n.y + d0));
                __builtin_nontemporal_store(q, reinterpret_cast<v4f_any *>(n.y + d1));
            } else {
                *reinterpret_cast<v4f_any *>(n.y + d0) = p;
                *reinterpret_cast<v4f_any *>(n.y + d1) = q;
            }
        } else {
            n.y[d0 * n.st] = o0[0];
            if (d1 < a.dim) n.y[d1 * n.st] = o1[0];
        }
    }
}

template <bool VEC, bool ADJ>
hipError_t rope(const RopeArgs &a, hipStream_t stream)
{
    constexpr uint32_t W = VEC ? 4 : 1;
    RopePlan pl;
    pl.rot = (a.pairs + W - 1) / W;
    pl.all = pl.rot + (a.dim - 2 * a.pairs + 2 * W - 1) / (2 * W);
    const uint32_t items = pl.all < kBlock ? pl.all : kBlock, chunks = (pl.all + kBlock - 1) / kBlock;
    const uint32_t pairs = a.pairs < items * W ? a.pairs : items * W; // of a workgroup, at most
    pl.items = FastDiv(items);
    pl.per = kBlock / items;
    pl.steps = (a.q.heads + a.k.heads + pl.per - 1) / pl.per;
    // Tiles for some 8000 workgroups (8001 tokens of 40 heads of 128 60.1 us, 71.7 with
    // 2000), and no more angles than their places; heads of more items than a
    // workgroup has threads take a token at a time, as their last workgroup has fewer
    // pairs.  Few tokens' heads are shared out too.
    const uint32_t most = chunks > 1 ? 1 : kRopeTurns / pairs, want = a.tokens / 8192 + 1;
    pl.tile = want < most ? want : most;
    uint32_t tiles = (a.tokens + pl.tile - 1) / pl.tile;
    tiles = tiles < kRopeGrid ? tiles : kRopeGrid;
    pl.groups = tiles < 512 ? pl.steps : 1;
    if (pl.groups > kRopeGrid / tiles) pl.groups = kRopeGrid / tiles;
    pl.stream = static_cast<uint64_t>(a.tokens) * (a.q.heads + a.k.heads) * a.dim * 4 > uint64_t{32} << 20;
    pl.turning = FastDiv(pairs);
    RopeArgs b = a;
    const uint64_t part = static_cast<uint64_t>(tiles) * pl.tile;
    for (uint64_t t = 0; t < a.tokens; t += part) {
        b.tokens = static_cast<uint32_t>(a.tokens - t < part ? a.tokens - t : part);
        b.pos = a.pos + static_cast<int64_t>(t) * a.pos_st[0];
        for (auto [to, from] : {std::pair<RopeTensor *, const RopeTensor *>{&b.q, &a.q}, {&b.k, &a.k}}) {
            to->x = from->x + static_cast<int64_t>(t) * from->x_st[2];
            to->y = from->y + static_cast<int64_t>(t) * from->y_st[2];
        }
        const uint32_t grid = (b.tokens + pl.tile - 1) / pl.tile * pl.groups;
        k_rope<VEC, ADJ><<<dim3(grid, chunks), kBlock, 0, stream>>>(b, pl);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

} // namespace

hipError_t launch_rope(const RopeArgs &a, hipStream_t stream)
{
    auto unit = [](const RopeTensor &t) { return t.heads == 0 || (t.x_st[0] == 1 && t.y_st[0] == 1); };
    const bool vec = a.pairs % 4 == 0 && (a.dim - 2 * a.pairs) % 8 == 0 && unit(a.q) && unit(a.k);
    if (vec) return a.adjacent ? rope<true, true>(a, stream) : rope<true, false>(a, stream);
    return a.adjacent ? rope<false, true>(a, stream) : rope<false, false>(a, stream);
}

} // namespace emel
