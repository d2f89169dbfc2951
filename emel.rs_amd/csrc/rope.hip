// rope.hip -- rotary positions of several axes, turned into queries and keys.
#include "common.hpp"
#include "launch.hpp"

namespace emel {
namespace {

// Pair i of a head turns by position * frequency.  A thread keeps its pairs'
// frequencies, in quarter turns a position and in 64 bits, and walks tokens
// and heads; a token's angles serve all of its heads.  In quarter turns the
// reduction of far positions is exact: t - rint(t), whose rounding is 2^-53 of t,
// so an angle is off by 2^-52 of itself and by f32's rounding of what is left.
//
// Bound by the bytes, 4 read and 4 written a value.

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
    uint32_t rot;    // items of a head that turn; the others copy
    uint32_t all;    // items of a head
    uint32_t per;    // heads of a step
    uint32_t steps;  // of a token
    uint64_t units, run; // token steps: all, and of a workgroup
};

// An item: four pairs, or eight values behind the pairs that are copied; one
// pair and two values where VEC is false.
template <bool VEC, bool ADJ>
__global__ __launch_bounds__(kBlock) void k_rope(RopeArgs a, RopePlan pl)
{
    constexpr uint32_t W = VEC ? 4 : 1;
    const uint32_t slot = pl.items.div(threadIdx.x);
    const uint32_t item = threadIdx.x - slot * pl.items.d + blockIdx.y * kBlock;
    if (slot >= pl.per || item >= pl.all) return;
    const bool turns = item < pl.rot;
    const uint32_t heads = a.q.heads + a.k.heads;

    double freq[W];
    uint32_t axis[W];
    if (turns) {
        for (uint32_t w = 0; w < W; ++w) {
            const uint32_t i = item * W + w;
            RopeRun r = a.runs[0];
            for (int n = 1; n < 4; ++n)
                if (i >= a.runs[n].start) r = a.runs[n];
            const uint32_t at = i - r.start, round = r.live == 1 ? at : r.live == 2 ? at / 2 : r.live == 3 ? at / 3 : at / 4;
            axis[w] = (r.axes >> (2 * (at - round * r.live))) & 3u;
            const double j = a.own ? r.round + round : i;
            const double rate = axis[w] == 0 ? a.rate[0] : axis[w] == 1 ? a.rate[1] : axis[w] == 2 ? a.rate[2] : a.rate[3];
            freq[w] = a.quarters * exp2(-j * rate);
            if (a.factors) freq[w] /= static_cast<double>(a.factors[static_cast<int64_t>(i) * a.factors_st]);
        }
    }
    uint64_t u = blockIdx.x * pl.run;
    const uint64_t end = u + pl.run < pl.units ? u + pl.run : pl.units;
    uint64_t token = u / pl.steps;
    uint32_t step = static_cast<uint32_t>(u - token * pl.steps);
    bool fresh = true;
    float c[W], s[W];
    for (; u < end; ++u) {
        const uint32_t h = step * pl.per + slot;
        const bool live = h < heads;
        const bool is_k = h >= a.q.heads;
        const RopeTensor &t = is_k ? a.k : a.q;
        const int64_t head = is_k ? h - a.q.heads : h;
        const float *x = t.x + head * t.x_st[1] + static_cast<int64_t>(token) * t.x_st[2];
        float *y = t.y + head * t.y_st[1] + static_cast<int64_t>(token) * t.y_st[2];
        // the first values of the item's pairs and their second ones
        const uint32_t d0 = turns ? (ADJ ? 2 * W * item : W * item) : 2 * a.pairs + 2 * W * (item - pl.rot);
        const uint32_t d1 = !turns || ADJ ? d0 + W : d0 + a.pairs;
        float lo[W], hi[W];
        if (live) {
            if constexpr (VEC) {
                const v4f p = *reinterpret_cast<const v4f_any *>(x + d0), r = *reinterpret_cast<const v4f_any *>(x + d1);
                for (int w = 0; w < 4; ++w) {
                    lo[w] = p[w];
                    hi[w] = r[w];
                }
            } else {
                lo[0] = x[d0 * t.x_st[0]];
                hi[0] = d1 < a.dim ? x[d1 * t.x_st[0]] : 0.0f;
            }
        }
        if (turns && fresh) {
            int32_t p[W];
            for (uint32_t w = 0; w < W; ++w) p[w] = a.pos[static_cast<int64_t>(token) * a.pos_st[0] + axis[w] * a.pos_st[1]];
            for (uint32_t w = 0; w < W; ++w) {
                quarter_turns(p[w] * freq[w], c[w], s[w]);
                c[w] *= a.magnitude;
                s[w] *= a.back ? -a.magnitude : a.magnitude;
            }
        }
        if (live) {
            float o0[W], o1[W];
            for (uint32_t w = 0; w < W; ++w) {
                if (!turns) {
                    o0[w] = lo[w];
                    o1[w] = hi[w];
                } else if constexpr (VEC && ADJ) { // pairs 0, 1 in lo, 2, 3 in hi
                    const float *v = w < 2 ? lo : hi;
                    const float e = v[2 * (w % 2)], f = v[2 * (w % 2) + 1];
                    float *o = w < 2 ? o0 : o1;
                    o[2 * (w % 2)] = __builtin_fmaf(e, c[w], -(f * s[w]));
                    o[2 * (w % 2) + 1] = __builtin_fmaf(e, s[w], f * c[w]);
                } else {
                    o0[w] = __builtin_fmaf(lo[w], c[w], -(hi[w] * s[w]));
                    o1[w] = __builtin_fmaf(lo[w], s[w], hi[w] * c[w]);
                }
            }
            if (turns || x != y) {
                if constexpr (VEC) {
                    *reinterpret_cast<v4f_any *>(y + d0) = v4f{o0[0], o0[1], o0[2], o0[3]};
                    *reinterpret_cast<v4f_any *>(y + d1) = v4f{o1[0], o1[1], o1[2], o1[3]};
                } else {
                    y[d0 * t.y_st[0]] = o0[0];
                    if (d1 < a.dim) y[d1 * t.y_st[0]] = o1[0];
                }
            }
        }
        fresh = ++step == pl.steps;
        if (fresh) {
            step = 0;
            ++token;
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
    pl.items = FastDiv(items);
    pl.per = kBlock / items;
    pl.steps = (a.q.heads + a.k.heads + pl.per - 1) / pl.per;
    pl.units = static_cast<uint64_t>(a.tokens) * pl.steps;
    const uint64_t most = 2048;
    pl.run = (pl.units + most - 1) / most;
    const uint32_t grid = static_cast<uint32_t>((pl.units + pl.run - 1) / pl.run);
    k_rope<VEC, ADJ><<<dim3(grid, chunks), kBlock, 0, stream>>>(a, pl);
    return hipGetLastError();
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
