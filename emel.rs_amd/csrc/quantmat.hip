// quantmat.hip -- products of packed 4-bit weights with f32 columns:
//   y[r, c] = sum over k of W[r, k] x[k, c],
// W[r, k] = (q - 8) d for Q4_0 (blocks of 32 values: an f16 d, 16 bytes of
// nibbles, the low ones first) and d sc q - dmin m for Q4_K (blocks of 256:
// f16 d and dmin, eight 6-bit sc and m, 128 bytes of nibbles).
//
// Bound by the weights' bytes for the few columns of a decode step, if what is
// done per weight stays small.  So the scales stay out of the inner product:
// a 32-value group's nibbles are exact as f16 integers, and one 16x16x32
// matrix instruction multiplies a group of 16 rows with up to 16 columns; the
// scale then goes once into each group's f32 result.  x is f32, so a column
// goes in as two halves, hi + lo, scaled by a power of two that brings its largest
// value to [2^14, 2^15): 22 bits of every value down to 2^-16 of that, and
// 2^-40 of it below.  Nibble-half products are exact, sums are f32.
// A nibble becomes a half by and-or into 1024's mantissa and one packed
// subtraction (or a packed fma for the high nibbles): 9 instructions for 8
// weights, and about 5 more a group for lanes' exchange and scales.
//
// Lane (j, g) of a wave works for row j of a tile of 16 rows.  Q4_0: it loads
// the whole of every fourth block, and the four lanes of a row exchange so
// that each instruction sees one block.  Q4_K: a block's nibbles are read 16
// bytes a lane, two swaps make sub-blocks of them.  The order of values within a group
// is whatever that gives; x is laid out in the same order.  The waves of a
// workgroup share a tile's k range and add up through LDS.
//
// hi + lo breaks 0 * inf and inf - inf, and a scale that is infinite times a
// sum is not the sum of its products: an output that is not finite is
// computed again as the formula stands, by the whole wave.
#include "common.hpp"
#include "launch.hpp"
#include "libm_replica.hpp"

namespace emel {
namespace {

constexpr int kQmWaves = 8;
constexpr int kQmBlock = kQmWaves * kWave;
constexpr uint32_t kQmLds = 64 * 1024; // of laid-out columns: two workgroups fit a compute unit

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef u4 u4_any __attribute__((aligned(1))); // packed rows may start at any byte
typedef v4f v4f_any __attribute__((aligned(4)));

// Per format: values of a unit (what a wave takes at a time), its bytes.
template <bool Q4K>
constexpr uint32_t kUnit = Q4K ? 256 : 128;

// Columns as the matrix instruction reads them, in 16-byte pieces of 8 halves.
// Column c of a group of 16 sits at [32-value group][part][c][lane row g]; Q4_K
// adds each column's group sums (for the minima) at [unit][c][part].
template <bool Q4K>
struct XLayout {
    uint32_t units, n; // n: columns laid out
    __host__ __device__ uint32_t groups() const { return units * (kUnit<Q4K> / 32); }
    __device__ uint32_t at(uint32_t group, uint32_t part, uint32_t c, uint32_t g) const { return ((group * 2 + part) * n + c) * 4 + g; }
    __device__ uint32_t sum_at(uint32_t unit, uint32_t c, uint32_t part) const { return groups() * n * 8 + (unit * n + c) * 2 + part; }
    __host__ __device__ uint64_t pieces() const { return static_cast<uint64_t>(groups()) * n * 8 + (Q4K ? units * n * 2 : 0); }
};

// Where the eight values of lane row g lie in their group: four from first
// and four from second, dealt out evens before odds as the nibbles fall.
template <bool Q4K>
__device__ __forceinline__ void value_places(uint32_t g, uint32_t &first, uint32_t &second)
{
    first = Q4K ? 16 * (g & 1) + 8 * (g >> 1) : 4 * g;
    second = Q4K ? first + 4 : 16 + 4 * g;
}

__device__ __forceinline__ uint32_t pack(_Float16 a, _Float16 b)
{
    return __builtin_bit_cast(uint16_t, a) | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, b)) << 16;
}

// The power of two that brings the largest finite magnitude into [2^14, 2^15), and its inverse.
__device__ __forceinline__ void column_scale(float top, float &up, float &down)
{
    int e = static_cast<int>((__builtin_bit_cast(uint32_t, top) >> 23) & 255u) - 127;
    e = top == 0.0f || e == 128 ? 0 : e < -110 ? -110 : e;
    up = __builtin_bit_cast(float, static_cast<uint32_t>(127 + 14 - e) << 23);
    down = __builtin_bit_cast(float, static_cast<uint32_t>(127 - 14 + e) << 23);
}

// Lays out a column's eight values of (group, g): x points at the column.
template <bool Q4K>
__device__ __forceinline__ void lay_out(const QMatArgs &a, const XLayout<Q4K> &lay, const float *x, float up, uint32_t group, uint32_t g, uint32_t c, u4 *to)
{
    uint32_t p[2];
    value_places<Q4K>(g, p[0], p[1]);
    float v[8];
    const uint32_t k0 = group * 32;
    if (k0 >= a.k) {
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    } else if (a.x_st[0] == 1) {
        const v4f lo = *reinterpret_cast<const v4f_any *>(x + k0 + p[0]), hi = *reinterpret_cast<const v4f_any *>(x + k0 + p[1]);
        for (int i = 0; i < 4; ++i) {
            v[i] = lo[i] * up;
            v[4 + i] = hi[i] * up;
        }
    } else {
        for (int i = 0; i < 8; ++i) v[i] = x[static_cast<int64_t>(k0 + p[i / 4] + i % 4) * a.x_st[0]] * up;
    }
    // Q4_0 halves: evens and odds of both fours; Q4_K: of each four
    constexpr int order[2][8] = {{0, 2, 4, 6, 1, 3, 5, 7}, {0, 2, 1, 3, 4, 6, 5, 7}};
    u4 hi, lo;
    for (int i = 0; i < 4; ++i) {
        const float x0 = v[order[Q4K][2 * i]], x1 = v[order[Q4K][2 * i + 1]];
        const _Float16 h0 = static_cast<_Float16>(x0), h1 = static_cast<_Float16>(x1);
        hi[i] = pack(h0, h1);
        lo[i] = pack(static_cast<_Float16>(x0 - static_cast<float>(h0)), static_cast<_Float16>(x1 - static_cast<float>(h1)));
    }
    to[lay.at(group, 0, c, g)] = hi;
    to[lay.at(group, 1, c, g)] = lo;
    if constexpr (Q4K) { // the group's sum over its four lanes, by 2^-6 within f16's range
        float s = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        s += __shfl_xor(s, 1, kWave);
        s += __shfl_xor(s, 2, kWave);
        s *= 0.015625f;
        const _Float16 h = static_cast<_Float16>(s);
        if (g < 2) {
            _Float16 *sums = reinterpret_cast<_Float16 *>(to + lay.sum_at(group / 8, c, g));
            sums[group % 8] = g == 0 ? h : static_cast<_Float16>(s - static_cast<float>(h));
        }
    }
}

// One column of a workgroup's threads: its scale, then its pieces.  All threads
// call it; top needs a float per wave.
template <bool Q4K, int THREADS>
__device__ __forceinline__ float lay_out_column(const QMatArgs &a, const XLayout<Q4K> &lay, uint32_t col, uint32_t c, u4 *to, float *top)
{
    const float *x = a.x + static_cast<int64_t>(col) * a.x_st[1];
    float m = 0.0f;
    if (a.x_st[0] == 1)
        for (uint32_t k = threadIdx.x * 4; k < a.k; k += THREADS * 4) {
            const v4f v = *reinterpret_cast<const v4f_any *>(x + k);
            for (int i = 0; i < 4; ++i) m = __builtin_fmaxf(m, __builtin_fabsf(v[i]));
        }
    else
        for (uint32_t k = threadIdx.x; k < a.k; k += THREADS) m = __builtin_fmaxf(m, __builtin_fabsf(x[static_cast<int64_t>(k) * a.x_st[0]]));
    m = wave_max_dpp(m);
    if (threadIdx.x % kWave == 0) top[threadIdx.x / kWave] = m;
    __syncthreads();
    for (int w = 0; w < THREADS / kWave; ++w) m = __builtin_fmaxf(m, top[w]);
    float up, down;
    column_scale(m, up, down);
    for (uint32_t i = threadIdx.x; i < lay.groups() * 4; i += THREADS) lay_out<Q4K>(a, lay, x, up, i / 4, i % 4, c, to);
    return down;
}

__device__ __forceinline__ float half_value(uint32_t h) { return hw_fp16_to_f32(static_cast<uint16_t>(h)); }

// W[r, k] x[k] over a whole row by one wave, product by product.
template <bool Q4K>
__device__ __forceinline__ float walk_row(const unsigned char *row, const float *x, int64_t st, uint32_t k)
{
    float sum = 0.0f;
#pragma unroll 1
    for (uint32_t g = threadIdx.x % kWave; g < k / 32; g += kWave) {
        const unsigned char *b = row + static_cast<uint64_t>(Q4K ? g / 8 * 144 : g * 18);
        const unsigned j = g % 8;
        float d = half_value(b[0] | b[1] << 8), off = 0.0f;
        if constexpr (Q4K) {
            const unsigned char *s = b + 4;
            const unsigned sc = j < 4 ? s[j] & 63u : (s[j + 4] & 15u) | ((s[j - 4] >> 6) << 4);
            const unsigned mn = j < 4 ? s[j + 4] & 63u : (s[j + 4] >> 4) | ((s[j] >> 6) << 4);
            off = half_value(b[2] | b[3] << 8) * static_cast<float>(mn);
            d *= static_cast<float>(sc);
        }
        const unsigned char *q = b + (Q4K ? 16 + 32 * (j / 2) : 2);
#pragma unroll 1
        for (unsigned i = 0; i < 32; ++i) {
            const unsigned v = Q4K ? (j % 2 ? q[i] >> 4 : q[i] & 15u) : (i < 16 ? q[i] & 15u : q[i - 16] >> 4);
            const float w = Q4K ? d * static_cast<float>(v) - off : (static_cast<float>(v) - 8.0f) * d;
            sum += w * x[static_cast<int64_t>(g * 32 + i) * st];
        }
    }
    return wave_sum(sum);
}

// Packed bytes of one unit as lane (j, g) loads them.
template <bool Q4K>
struct Raw;
template <>
struct Raw<false> {
    u4 q;
    uint32_t d;
};
template <>
struct Raw<true> {
    u4 head, q[2];
};

__device__ __forceinline__ u4 load16(const unsigned char *p) { return *reinterpret_cast<const u4_any *>(p); }

__device__ __forceinline__ void load_unit(Raw<false> &r, const unsigned char *row, uint32_t unit, uint32_t g, uint32_t blocks)
{
    const uint32_t b = unit * 4 + g;
    const unsigned char *p = row + static_cast<uint64_t>(b < blocks ? b : blocks - 1) * 18;
    uint16_t d;
    __builtin_memcpy(&d, p, 2);
    r.d = b < blocks ? d : 0; // past the row: nothing times zeros
    r.q = load16(p + 2);
}
__device__ __forceinline__ void load_unit(Raw<true> &r, const unsigned char *row, uint32_t unit, uint32_t g, uint32_t)
{
    const unsigned char *p = row + static_cast<uint64_t>(unit) * 144;
    r.head = load16(p);
    r.q[0] = load16(p + 16 + 16 * g);
    r.q[1] = load16(p + 80 + 16 * g);
}

__device__ __forceinline__ void swap16(uint32_t &a, uint32_t &b)
{
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}
__device__ __forceinline__ void swap32(uint32_t &a, uint32_t &b)
{
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}

// Two nibbles, in bits 0-3 (or 4-7) of a word's halves, as halves minus `off`.
__device__ __forceinline__ uint32_t low_nibbles(uint32_t u, _Float16 off)
{
    const v2h v = __builtin_bit_cast(v2h, (u & 0x000F000Fu) | 0x64006400u);
    return __builtin_bit_cast(uint32_t, v - v2h{static_cast<_Float16>(1024.0f + off), static_cast<_Float16>(1024.0f + off)});
}
__device__ __forceinline__ uint32_t high_nibbles(uint32_t u, _Float16 off)
{
    const v2h v = __builtin_bit_cast(v2h, (u & 0x00F000F0u) | 0x64006400u);
    const v2h s = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
    const v2h o = {static_cast<_Float16>(-64.0f - off), static_cast<_Float16>(-64.0f - off)};
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(v, s, o));
}

__device__ __forceinline__ v4f mfma(u4 x, u4 w, v4f c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, w), c, 0, 0, 0);
}

// acc[r] (column 4 r + g of row j) += this unit's products.
template <int NR>
__device__ __forceinline__ void do_unit(Raw<false> r, const XLayout<false> &lay, const u4 *xs, uint32_t unit, uint32_t c, uint32_t g, float *acc)
{
    uint32_t w[4] = {r.q[0], r.q[1], r.q[2], r.q[3]}; // word t of block g ...
    swap32(w[0], w[2]);
    swap32(w[1], w[3]);
    swap16(w[0], w[1]);
    swap16(w[2], w[3]); // ... to word g of block t
    uint32_t d[4];
    d[0] = d[2] = __builtin_bit_cast(uint32_t, half_value(r.d));
    swap32(d[0], d[2]);
    d[1] = d[0];
    d[3] = d[2];
    swap16(d[0], d[1]);
    swap16(d[2], d[3]); // every lane of the row: block t's scale
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const uint32_t u = w[t], v = u >> 8;
        const u4 q = {low_nibbles(u, 8.0f), high_nibbles(u, 8.0f), low_nibbles(v, 8.0f), high_nibbles(v, 8.0f)};
        const uint32_t group = unit * 4 + t;
        const v4f s = mfma(xs[lay.at(group, 0, c, g)], q, mfma(xs[lay.at(group, 1, c, g)], q, v4f{0.0f, 0.0f, 0.0f, 0.0f}));
        const float f = __builtin_bit_cast(float, d[t]);
        for (int i = 0; i < NR; ++i) acc[i] = __builtin_fmaf(f, s[i], acc[i]);
    }
}

template <int NR>
__device__ __forceinline__ void do_unit(Raw<true> r, const XLayout<true> &lay, const u4 *xs, uint32_t unit, uint32_t c, uint32_t g, float *acc)
{
    const uint32_t h0 = r.head[0], s0 = r.head[1], s1 = r.head[2], s2 = r.head[3];
    const uint32_t sc[2] = {s0 & 0x3f3f3f3fu, (s2 & 0x0f0f0f0fu) | ((s0 >> 2) & 0x30303030u)};
    const uint32_t mn[2] = {s1 & 0x3f3f3f3fu, ((s2 >> 4) & 0x0f0f0f0fu) | ((s1 >> 2) & 0x30303030u)};
    const float d = half_value(h0 & 0xffffu), dmin = half_value(h0 >> 16) * -64.0f;
    float t[NR];
    for (int i = 0; i < NR; ++i) t[i] = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t w[4] = {r.q[h][0], r.q[h][1], r.q[h][2], r.q[h][3]};
        swap32(w[0], w[2]); // words 0, 1: quarter 2 h of the block, words 2, 3: quarter 2 h + 1
        swap32(w[1], w[3]);
#pragma unroll
        for (int b = 0; b < 4; ++b) { // sub-block 4 h + b
            const uint32_t u = w[b / 2 * 2], v = w[b / 2 * 2 + 1];
            const u4 q = b % 2 ? u4{high_nibbles(u, 0.0f), high_nibbles(u >> 8, 0.0f), high_nibbles(v, 0.0f), high_nibbles(v >> 8, 0.0f)}
                               : u4{low_nibbles(u, 0.0f), low_nibbles(u >> 8, 0.0f), low_nibbles(v, 0.0f), low_nibbles(v >> 8, 0.0f)};
            const uint32_t group = unit * 8 + 4 * h + b;
            const v4f s = mfma(xs[lay.at(group, 0, c, g)], q, mfma(xs[lay.at(group, 1, c, g)], q, v4f{0.0f, 0.0f, 0.0f, 0.0f}));
            const float f = static_cast<float>((sc[h] >> (8 * b)) & 255u);
            for (int i = 0; i < NR; ++i) t[i] = __builtin_fmaf(f, s[i], t[i]);
        }
    }
    // the minima: their products with the groups' sums, hi for lane row 0, lo for 1
    const u4 sums = xs[lay.sum_at(unit, c, g & 1)], none = {0, 0, 0, 0};
    u4 m;
    for (int i = 0; i < 4; ++i) { // bytes 2 i and 2 i + 1 into 1024's mantissa
        const v2h v = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, mn[i / 2], i % 2 ? 0x07030702u : 0x05010400u));
        m[i] = __builtin_bit_cast(uint32_t, v - v2h{static_cast<_Float16>(1024.0f), static_cast<_Float16>(1024.0f)});
    }
    const v4f s = mfma(g < 2 ? sums : none, m, v4f{0.0f, 0.0f, 0.0f, 0.0f});
    for (int i = 0; i < NR; ++i) acc[i] = __builtin_fmaf(d, t[i], __builtin_fmaf(dmin, s[i], acc[i]));
}

struct QmPlan {
    uint32_t tiles;    // of 16 rows
    uint32_t kw;       // waves along k; the others take further tiles
    uint32_t groups;   // of 16 columns
    uint64_t x_pieces; // workspace pieces of a group (0: columns are laid out in LDS)
};

// Lays out a column a workgroup in the workspace, and leaves its scale behind the pieces.
template <bool Q4K>
__global__ __launch_bounds__(kQmBlock) void k_qm_columns(QMatArgs a, QmPlan pl)
{
    __shared__ float top[kQmWaves];
    for (uint32_t col = blockIdx.x; col < a.n; col += gridDim.x) {
        const uint32_t group = col / 16, n = a.n - group * 16 < 16 ? a.n - group * 16 : 16;
        const XLayout<Q4K> lay{(a.k + kUnit<Q4K> - 1) / kUnit<Q4K>, n};
        u4 *to = static_cast<u4 *>(a.workspace) + group * pl.x_pieces;
        __syncthreads(); // top of the column before
        const float down = lay_out_column<Q4K, kQmBlock>(a, lay, col, col % 16, to, top);
        if (threadIdx.x == 0) reinterpret_cast<float *>(static_cast<u4 *>(a.workspace) + pl.groups * pl.x_pieces)[col] = down;
    }
}

// NR: a quarter of the columns, rounded up.  LDS: columns laid out here, else read from the workspace.
template <bool Q4K, int NR, bool LDS>
__global__ __launch_bounds__(kQmBlock, 2) void k_qm(QMatArgs a, QmPlan pl)
{
    constexpr int U = Q4K ? 2 : 4; // units in flight
    extern __shared__ u4 laid[];
    __shared__ float top[kQmWaves], downs[16];
    __shared__ float part[2][kQmWaves][NR][kWave];
    const uint32_t tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave), j = lane % 16, g = lane / 16;
    const uint32_t c0 = blockIdx.y * 16, n = a.n - c0 < 16 ? a.n - c0 : 16;
    const XLayout<Q4K> lay{(a.k + kUnit<Q4K> - 1) / kUnit<Q4K>, n};
    const uint32_t kw = pl.kw, tw = kQmWaves / kw, wk = wave % kw, wt = wave / kw;
    const uint32_t u0 = static_cast<uint32_t>(static_cast<uint64_t>(lay.units) * wk / kw);
    const uint32_t u1 = static_cast<uint32_t>(static_cast<uint64_t>(lay.units) * (wk + 1) / kw);
    const uint32_t blocks = a.k / 32;
    const uint64_t row_bytes = Q4K ? static_cast<uint64_t>(a.k / 256) * 144 : static_cast<uint64_t>(blocks) * 18;
    const unsigned char *w = static_cast<const unsigned char *>(a.w);
    auto row_of = [&](uint32_t tile) { // of this wave's tile; past the last one, rows that are read and dropped
        const uint64_t r = (static_cast<uint64_t>(tile) + wt) * 16 + j;
        return w + (r < a.m ? r : a.m - 1) * row_bytes;
    };
    // the first weights are on their way while the columns are laid out
    uint32_t tile = blockIdx.x * tw;
    const unsigned char *row = row_of(tile);
    Raw<Q4K> raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
        if (u0 + i < u1) load_unit(raw[i], row, u0 + i, g, blocks);
    const u4 *xs;
    if constexpr (LDS) {
        for (uint32_t c = 0; c < n; ++c) {
            if (c) __syncthreads();
            const float down = lay_out_column<Q4K, kQmBlock>(a, lay, c0 + c, c, laid, top);
            if (tid == 0) downs[c] = down;
        }
        xs = laid;
    } else {
        xs = static_cast<const u4 *>(a.workspace) + blockIdx.y * pl.x_pieces;
        const float *d = reinterpret_cast<const float *>(static_cast<const u4 *>(a.workspace) + pl.groups * pl.x_pieces) + c0;
        if (tid < n) downs[tid] = d[tid];
    }
    __syncthreads();
    // slot j of the instruction's 16 columns is column 4 (j % 4) + j / 4, so
    // that result i of lane row g is column 4 i + g; the slots past n repeat
    uint32_t c = (j % 4) * 4 + j / 4;
    c = c < n ? c : n - 1;
    uint32_t turn = 0;
    for (; tile < pl.tiles; tile += gridDim.x * tw, turn ^= 1) {
        float acc[NR];
        for (int i = 0; i < NR; ++i) acc[i] = 0.0f;
        const unsigned char *next = row_of(tile + gridDim.x * tw);
        for (uint32_t u = u0; u < u1; u += U) {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (u + i < u1) do_unit<NR>(raw[i], lay, xs, u + i, c, g, acc);
                // the slot's next unit: of this tile, or of the next one
                if (u + i + U < u1) load_unit(raw[i], row, u + i + U, g, blocks);
                else if (u + U >= u1 && u0 + i < u1) load_unit(raw[i], next, u0 + i, g, blocks);
            }
        }
        row = next;
        for (int i = 0; i < NR; ++i) part[turn][wave][i][lane] = acc[i];
        __syncthreads();
        for (uint32_t e = wave; e < tw * NR; e += kQmWaves) { // a wave per tile and quarter of columns
            const uint32_t t = e / NR, i = e % NR, col = 4 * i + g;
            float v = 0.0f;
            for (uint32_t s = 0; s < kw; ++s) v += part[turn][t * kw + s][i][lane];
            const uint64_t r = (static_cast<uint64_t>(tile) + t) * 16 + j;
            const bool live = r < a.m && col < n;
            v *= live ? downs[col] : 0.0f;
            uint64_t odd = __ballot(live && !(__builtin_fabsf(v) < __builtin_inff()));
            while (__builtin_expect(odd != 0, 0)) {
                const int l = __builtin_ctzll(odd);
                odd &= odd - 1;
                const uint64_t rr = (static_cast<uint64_t>(tile) + t) * 16 + l % 16;
                const float f = walk_row<Q4K>(w + rr * row_bytes, a.x + static_cast<int64_t>(c0 + 4 * i + l / 16) * a.x_st[1], a.x_st[0], a.k);
                if (lane == static_cast<uint32_t>(l)) v = f;
            }
            if (live) a.y[static_cast<int64_t>(r) * a.y_st[0] + static_cast<int64_t>(c0 + col) * a.y_st[1]] = v;
        }
    }
}

template <bool Q4K>
QmPlan qm_plan(const QMatArgs &a)
{
    QmPlan pl;
    const uint32_t units = (a.k + kUnit<Q4K> - 1) / kUnit<Q4K>;
    pl.tiles = static_cast<uint32_t>((static_cast<uint64_t>(a.m) + 15) / 16);
    pl.kw = units >= 16 ? 8 : units >= 8 ? 4 : units >= 4 ? 2 : 1;
    pl.groups = (a.n + 15) / 16;
    const XLayout<Q4K> lay{units, a.n < 16 ? a.n : 16};
    pl.x_pieces = pl.groups == 1 && lay.pieces() * 16 <= kQmLds ? 0 : lay.pieces();
    return pl;
}

template <bool Q4K, int NR>
void qm_launch(const QMatArgs &a, const QmPlan &pl, hipStream_t stream)
{
    static const uint32_t cus = [] {
        int dev = 0, n = 0;
        if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
            n = 256;
        return static_cast<uint32_t>(n);
    }();
    const uint32_t tw = kQmWaves / pl.kw, wgs = (pl.tiles + tw - 1) / tw;
    const dim3 grid(wgs < 2 * cus ? wgs : 2 * cus, pl.groups);
    if (pl.x_pieces) {
        k_qm_columns<Q4K><<<a.n < 65536 ? a.n : 65536, kQmBlock, 0, stream>>>(a, pl);
        k_qm<Q4K, NR, false><<<grid, kQmBlock, 0, stream>>>(a, pl);
    } else {
        const XLayout<Q4K> lay{(a.k + kUnit<Q4K> - 1) / kUnit<Q4K>, a.n};
        k_qm<Q4K, NR, true><<<grid, kQmBlock, static_cast<uint32_t>(lay.pieces() * 16), stream>>>(a, pl);
    }
}

template <bool Q4K>
hipError_t qm_run(const QMatArgs &a, hipStream_t stream)
{
    const QmPlan pl = qm_plan<Q4K>(a);
    switch ((a.n + 3) / 4) {
    case 1: qm_launch<Q4K, 1>(a, pl, stream); break;
    case 2: qm_launch<Q4K, 2>(a, pl, stream); break;
    case 3: qm_launch<Q4K, 3>(a, pl, stream); break;
    default: qm_launch<Q4K, 4>(a, pl, stream); break;
    }
    return hipGetLastError();
}

} // namespace

uint64_t quant_mat_workspace_bytes(const QMatArgs &a)
{
    const QmPlan pl = a.q4k ? qm_plan<true>(a) : qm_plan<false>(a);
    return pl.x_pieces ? pl.groups * pl.x_pieces * 16 + static_cast<uint64_t>(a.n) * 4 : 0;
}

hipError_t launch_quant_mat(const QMatArgs &a, hipStream_t stream)
{
    return a.q4k ? qm_run<true>(a, stream) : qm_run<false>(a, stream);
}

} // namespace emel
