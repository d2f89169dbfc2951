// quantmat.hip -- products of packed 4-bit weights with f32 columns:
//   y[r, c] = sum over k of W[r, k] x[k, c],
// W[r, k] = (q - 8) d for Q4_0 (blocks of 32 values: an f16 d, 16 bytes of
// nibbles, the low ones first) and d sc q - dmin m for Q4_K (blocks of 256:
// f16 d and dmin, eight 6-bit sc and m, 128 bytes of nibbles).
//
// Bound by the weights' bytes for the few columns of a decode step, if what is
// done per weight stays small.  So scales and minima stay out of the inner
// product: a matrix instruction multiplies a 32-value group of 16 rows with the columns,
// nibbles as integers, and the group's scale goes once into its result.  x is
// f32 and is not to lose by it; two ways, by the number of columns:
//
// k_qm_digits, up to four columns where they fit LDS.  Each column's run of 256 values is a
// fixed-point number of 30 bits and a sign, scaled by a power of two to its largest
// value, and cut into four signed bytes.  The 16 columns of the 8-bit
// instruction then hold 4 digits x 4 columns, and one instruction a group does
// them all, exactly, in integers.  Eight weights cost three or four
// instructions of unpacking, a group one LDS read, and a conversion and an fma
// a column.  A value is off by 2^-30 of the largest of its 256 at most (by 2^-127
// where that is below 2^-97: the scale stays a normal number).  While most of
// the run is within 2^-9 of its largest, that is less than f32's rounding of
// a sum of such products.  It is not where a few values stand far above the
// rest and meet small or zero weights (10^4 times: 5e-6 of the result), so a
// workgroup that finds two runs side by side of whose nonzero values more than
// a quarter is below 2^-9 of their run's largest lays out what the digits left
// over, as four more of them, goes through its tiles again and adds that: 60
// bits, at twice the time (one column of 4096x4096 9.2 us).  To look for such
// runs costs 0.2 us there.
// One column of 4096x4096 5.6 us (a launch, the layout, one round of loads),
// three of 4096x151936 78 us: 4.5 TB/s.
//
// k_qm_halves, all others.  Each column's run of 256 values goes in as two
// halves each, hi + lo, scaled by a power of two that brings its largest value to
// [2^14, 2^15): 22 bits of every value down to 2^-16 of that, and 2^-40 of it
// below.  The 16 columns of the f16 instruction are 16 columns, two
// instructions a group.  A workgroup lays a chunk of k, up to four units, of 16
// columns out in LDS and takes a run of tiles through it, a tile a wave,
// without another barrier; k_qm_sum adds up the chunks.  (Columns laid out by a
// kernel of their own and staged by half units, each workgroup over all of k:
// 15 columns of 4096x11008 20.7 us against 15.5, 16 of 4096x40000 56 against 35.)  A nibble
// becomes a half by and-or into 1024's mantissa and a packed subtraction (as a
// subnormal half it would need neither, but the instruction drops as many
// low bits of its sum as such a factor has leading zeros: 1e-5 off).
// Of 15.5 us of 4096x11008 about 9.6 are the launch and the weights (25 MB from
// the L2 and the Infinity Cache), 2.3 the columns' layout, 2 to 3 the
// matrix instructions and what surrounds them, 2 to 3 k_qm_sum.
//
// Sums are f32, and their order depends on the sizes alone.
//
// Lane (j, g) of a wave works for row j of a tile of 16 rows.  It loads a
// fourth of the row's 256-value unit, whole blocks of Q4_0 or 16 bytes of each
// half of a Q4_K block, and the four lanes of a row exchange words so that each
// instruction sees one group.  The order of values within a group is whatever
// that gives; x is laid out in the same order.  As digits, the waves of a
// workgroup share a tile's k range and add up through LDS.
//
// Neither digits nor halves hold infinities: an output that is not finite is
// computed again as the formula stands, by the whole wave, but where its column
// holds a NaN: then it is one (a slot of a batch that nobody filled would make
// 15 columns of 4096x11008 216 us instead of 15.5, and so makes it 21).
#include <type_traits>

#include "common.hpp"
#include "launch.hpp"
#include "libm_replica.hpp"

namespace emel {
namespace {

constexpr int kQmWaves = 8;
constexpr int kQmBlock = kQmWaves * kWave;
constexpr uint32_t kQmUnit = 256;      // values that a wave takes of a row at a time: eight groups
constexpr uint32_t kQmLds = 80 * 1024, kQmLdsAlone = 110 * 1024; // of a workgroup: two fit a compute unit, or one

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef u4 u4_byte __attribute__((aligned(1))); // packed rows may start at any byte
typedef u4 u4_word __attribute__((aligned(4)));
typedef v4f v4f_any __attribute__((aligned(4)));

// Where the eight values of lane row g lie in their group: four from first
// and four from second, dealt out as the nibbles fall.
template <bool Q4K>
__device__ __forceinline__ void value_places(uint32_t g, uint32_t &first, uint32_t &second)
{
    first = Q4K ? 16 * (g & 1) + 8 * (g >> 1) : 4 * g;
    second = Q4K ? first + 4 : 16 + 4 * g;
}

// Eight values of (group, g) of a column, times up; zeros past the column.
template <bool Q4K>
__device__ __forceinline__ void load_values(const QMatArgs &a, const float *x, uint32_t group, uint32_t g, float v[8])
{
    uint32_t p[2];
    value_places<Q4K>(g, p[0], p[1]);
    const uint32_t k0 = group * 32;
    if (k0 >= a.k) {
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    } else if (a.x_st[0] == 1) {
        const v4f lo = *reinterpret_cast<const v4f_any *>(x + k0 + p[0]), hi = *reinterpret_cast<const v4f_any *>(x + k0 + p[1]);
        for (int i = 0; i < 4; ++i) {
            v[i] = lo[i];
            v[4 + i] = hi[i];
        }
    } else {
        for (int i = 0; i < 8; ++i) v[i] = x[static_cast<int64_t>(k0 + p[i / 4] + i % 4) * a.x_st[0]];
    }
}

template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v)
{
    return __builtin_bit_cast(float, dpp32<CTRL>(__builtin_bit_cast(uint32_t, v)));
}

// Scales the eight values of each lane of a half wave, 256 in all, by the power
// of two that brings the largest to [2^TOP, 2^(TOP + 1)); returns its inverse,
// or NaN where a value is not finite (an output that meets it is computed again).
template <int TOP>
__device__ __forceinline__ float scale_unit(float v[8])
{
    float top = 0.0f, zero = 0.0f;
    for (int e = 0; e < 8; ++e) {
        top = __builtin_fmaxf(top, __builtin_fabsf(v[e]));
        zero = __builtin_fmaf(v[e], 0.0f, zero); // NaN from an infinity or NaN
    }
    top = __builtin_fmaxf(top, dpp_f32<kDppXor1>(top));
    top = __builtin_fmaxf(top, dpp_f32<kDppXor2>(top));
    top = __builtin_fmaxf(top, dpp_f32<kDppHalfMirror>(top));
    top = __builtin_fmaxf(top, dpp_f32<kDppMirror>(top));
    top = __builtin_fmaxf(top, __shfl_xor(top, 16, kWave));
    const uint64_t odd = __ballot(!(zero == 0.0f)) >> (threadIdx.x & 32);
    constexpr int least = TOP - 126; // the power stays a normal number
    int e = static_cast<int>((__builtin_bit_cast(uint32_t, top) >> 23) & 255u) - 127;
    e = e == 128 ? 0 : e < least ? least : e;
    const float up = __builtin_bit_cast(float, static_cast<uint32_t>(127 + TOP - e) << 23);
    for (int i = 0; i < 8; ++i) v[i] *= up;
    return static_cast<uint32_t>(odd) ? __builtin_nanf("") : __builtin_bit_cast(float, static_cast<uint32_t>(127 - TOP + e) << 23);
}

// ---- columns as digits ---------------------------------------------------------------

// In LDS, eight bytes each: digit d of unit u's group t at [u][t][d][column][lane
// row], its group sums behind all of those at [u][d][column], and the units'
// scales as floats behind all at [u][column].
template <int N>
struct Digits {
    static constexpr uint32_t kUnit = 8 * 4 * N * 4;
    static __host__ __device__ uint32_t sums(uint32_t units) { return units * kUnit; }
    static __host__ __device__ uint32_t scales(uint32_t units) { return units * (kUnit + 4 * N); }
    static __host__ __device__ uint64_t bytes(uint64_t units) { return units * ((kUnit + 4 * N) * 8 + N * 4); }
};

// The four signed bytes d0 + 2^8 d1 + 2^16 d2 + 2^24 d3 of v, |v| < 2^30;
// LEFT: of 2^30 times what they leave of v.
template <bool LEFT>
__device__ __forceinline__ uint32_t digits_of(float v)
{
    float n = __builtin_rintf(v);
    if constexpr (LEFT) n = __builtin_rintf((v - n) * 0x1p30f);
    return (static_cast<uint32_t>(static_cast<int>(n)) + 0x00808080u) ^ 0x00808080u;
}

// Whether more than a quarter of the nonzero values of a wave's two units, as
// scale_unit<29> leaves them, are below 2^21.
__device__ __forceinline__ bool units_wide(const float v[8])
{
    const uint32_t all = 8 * __builtin_popcountll(__ballot(true));
    uint32_t small = 0, zero = 0;
    for (int i = 0; i < 8; ++i) small += __builtin_popcountll(__ballot(__builtin_fabsf(v[i]) < 0x1p21f));
    if (__builtin_expect(4 * small <= all, 1)) return false;
    for (int i = 0; i < 8; ++i) zero += __builtin_popcountll(__ballot(v[i] == 0.0f));
    return 4 * (small - zero) > all - zero;
}

// Byte b of four words, as word b.
__device__ __forceinline__ void bytes4(const uint32_t t[4], uint32_t out[4])
{
    const uint32_t a = __builtin_amdgcn_perm(t[1], t[0], 0x05010400u), b = __builtin_amdgcn_perm(t[3], t[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(t[1], t[0], 0x07030602u), d = __builtin_amdgcn_perm(t[3], t[2], 0x07030602u);
    out[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    out[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    out[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    out[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// Returns whether units of this wave's are wide.
template <bool Q4K, int N, bool LEFT>
__device__ __forceinline__ bool lay_out_digits(const QMatArgs &a, uint32_t units, u2 *to, uint32_t tid)
{
    bool wide = false;
    // A unit of a column per half wave: group i / 4 % 8, lane row i % 4.  Four
    // of them at a time, so that their loads overlap (LEFT is rare: one).
    constexpr uint32_t B = LEFT ? 1 : 4;
    const uint32_t run = units * 32, all = run * a.n;
    for (uint32_t i0 = tid; i0 < all; i0 += B * kQmBlock) {
        float v[B][8];
#pragma unroll
        for (uint32_t b = 0; b < B; ++b) {
            const uint32_t i = i0 + b * kQmBlock, c = N == 1 ? 0 : i / run, k = i - c * run;
            if (i < all) load_values<Q4K>(a, a.x + static_cast<int64_t>(c) * a.x_st[1], k / 4, k % 4, v[b]);
        }
#pragma unroll
        for (uint32_t b = 0; b < B; ++b) {
            const uint32_t i = i0 + b * kQmBlock, c = N == 1 ? 0 : i / run, k = i - c * run;
            if (i >= all) break;
            const uint32_t unit = k / 32, t = k / 4 % 8, g = k % 4;
            const float down = scale_unit<29>(v[b]);
            if constexpr (!LEFT) wide |= units_wide(v[b]);
            if (k % 32 == 0) reinterpret_cast<float *>(to + Digits<N>::scales(units))[unit * N + c] = down;
            uint32_t w[2][4], d[2][4];
            for (int q = 0; q < 8; ++q) w[q / 4][q % 4] = digits_of<LEFT>(v[b][q]);
            bytes4(w[0], d[0]);
            bytes4(w[1], d[1]);
            for (uint32_t q = 0; q < 4; ++q) to[unit * Digits<N>::kUnit + ((t * 4 + q) * N + c) * 4 + g] = u2{d[0][q], d[1][q]};
            if constexpr (Q4K) { // sums of 32 values, by 2^-5
                float sum = ((v[b][0] + v[b][1]) + (v[b][2] + v[b][3])) + ((v[b][4] + v[b][5]) + (v[b][6] + v[b][7]));
                sum += dpp_f32<kDppXor1>(sum);
                sum += dpp_f32<kDppXor2>(sum);
                const uint32_t s = digits_of<LEFT>(sum * 0.03125f);
                // lane row g writes digit g
                reinterpret_cast<unsigned char *>(to + Digits<N>::sums(units) + (unit * 4 + g) * N + c)[t] = static_cast<unsigned char>(s >> (8 * g));
            }
        }
    }
    return wide;
}

// ---- columns as halves -----------------------------------------------------------------

// In LDS, 16 bytes of 8 halves each, 16 columns side by side: unit u's group t
// at [u][t][part][column][lane row], and behind all units, at [u][column][part],
// the eight groups' sums (parts 2 and 3 are zeros), and behind those the
// units' scales, column 4 i + g at [u][g][i].
constexpr uint32_t kHalvesUnit = 8 * 2 * 16 * 4;
constexpr uint32_t kHalvesBytes = (kHalvesUnit + 16 * 4 + 4) * 16; // of a unit
constexpr uint32_t halves_at(uint32_t t, uint32_t part) { return (t * 2 + part) * 16 * 4; }

__device__ __forceinline__ uint32_t pack(_Float16 a, _Float16 b)
{
    return __builtin_bit_cast(uint16_t, a) | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, b)) << 16;
}

// Column c's unit, by a half wave: lane i % 32 holds its (group, lane row).
template <bool Q4K>
__device__ __forceinline__ void lay_out_halves(float v[8], uint32_t units, uint32_t unit, uint32_t i, uint32_t c, u4 *to)
{
    const uint32_t t = i / 4, g = i % 4;
    const float down = scale_unit<14>(v);
    u4 *sums = to + units * kHalvesUnit;
    if (i == 0) reinterpret_cast<float *>(sums + units * (16 * 4))[unit * 16 + c % 4 * 4 + c / 4] = down;
    if constexpr (Q4K) { // the group's sum over its four lanes, by 2^-6 within f16's range
        float sum = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        sum += dpp_f32<kDppXor1>(sum);
        sum += dpp_f32<kDppXor2>(sum);
        sum *= 0.015625f;
        const _Float16 h = static_cast<_Float16>(sum);
        reinterpret_cast<_Float16 *>(sums + (unit * 16 + c) * 4 + g)[t] =
            g == 0 ? h : g == 1 ? static_cast<_Float16>(sum - static_cast<float>(h)) : static_cast<_Float16>(0.0f);
    }
    // Q4_0 halves: evens and odds of both fours; Q4_K: of each four
    constexpr int order[2][8] = {{0, 2, 4, 6, 1, 3, 5, 7}, {0, 2, 1, 3, 4, 6, 5, 7}};
    u4 hi, lo;
    for (int q = 0; q < 4; ++q) {
        const float x0 = v[order[Q4K][2 * q]], x1 = v[order[Q4K][2 * q + 1]];
        const _Float16 h0 = static_cast<_Float16>(x0), h1 = static_cast<_Float16>(x1);
        hi[q] = pack(h0, h1);
        lo[q] = pack(static_cast<_Float16>(x0 - static_cast<float>(h0)), static_cast<_Float16>(x1 - static_cast<float>(h1)));
    }
    u4 *at = to + unit * kHalvesUnit + c * 4 + g;
    at[halves_at(t, 0)] = hi;
    at[halves_at(t, 1)] = lo;
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

// Whether a column holds a NaN, which makes all of its outputs NaN: by one wave.
__device__ __forceinline__ bool column_nan(const float *x, int64_t st, uint32_t k)
{
    bool nan = false;
#pragma unroll 4
    for (uint32_t i = threadIdx.x % kWave; i < k; i += kWave) nan |= __builtin_isnan(x[static_cast<int64_t>(i) * st]);
    return __any(nan);
}

// Packed bytes of one unit as lane (j, g) loads them: two Q4_0 blocks (d in
// word 0's low and word 4's high half, nibbles between and behind), or a Q4_K
// block's head and its lane's 16 bytes of both halves.
template <bool Q4K>
struct Raw;
template <>
struct Raw<false> {
    u4 a, b;
    uint32_t c;
};
template <>
struct Raw<true> {
    u4 head, q[2];
};

// WORDS: rows start at multiples of four bytes and hold whole pairs of blocks.
template <bool WORDS>
__device__ __forceinline__ void load_unit(Raw<false> &r, const unsigned char *row, uint32_t unit, uint32_t g, uint32_t blocks)
{
    const uint32_t b = unit * 8 + 2 * g;
    if constexpr (WORDS) {
        const unsigned char *p = row + static_cast<uint64_t>(b < blocks ? b : blocks - 2) * 18;
        r.a = *reinterpret_cast<const u4_word *>(p);
        r.b = *reinterpret_cast<const u4_word *>(p + 16);
        r.c = *reinterpret_cast<const uint32_t *>(p + 32);
    } else { // a block at a time, put together as above
        const unsigned char *p = row + static_cast<uint64_t>(b < blocks ? b : blocks - 1) * 18;
        const unsigned char *s = row + static_cast<uint64_t>(b + 1 < blocks ? b + 1 : blocks - 1) * 18;
        uint16_t last, d;
        __builtin_memcpy(&last, p + 16, 2);
        __builtin_memcpy(&d, s, 2);
        r.a = *reinterpret_cast<const u4_byte *>(p);
        const u4 q = *reinterpret_cast<const u4_byte *>(s + 2);
        r.b = u4{last | static_cast<uint32_t>(d) << 16, q[0], q[1], q[2]};
        r.c = q[3];
    }
}
template <bool WORDS>
__device__ __forceinline__ void load_unit(Raw<true> &r, const unsigned char *row, uint32_t unit, uint32_t g, uint32_t)
{
    typedef std::conditional_t<WORDS, u4_word, u4_byte> piece;
    const unsigned char *p = row + static_cast<uint64_t>(unit) * 144;
    r.head = *reinterpret_cast<const piece *>(p);
    r.q[0] = *reinterpret_cast<const piece *>(p + 16 + 16 * g);
    r.q[1] = *reinterpret_cast<const piece *>(p + 80 + 16 * g);
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
// Word t of lane row g to word g of lane row t.
__device__ __forceinline__ void transpose(uint32_t w[4])
{
    swap32(w[0], w[2]);
    swap32(w[1], w[3]);
    swap16(w[0], w[1]);
    swap16(w[2], w[3]);
}

// ---- a unit made ready: words and scales of its eight groups ----------------------------

template <bool Q4K>
struct Unit;

template <>
struct Unit<false> {
    uint32_t w[2][4]; // even and odd blocks
    uint32_t d[4];    // eight halves

    __device__ __forceinline__ Unit(const Raw<false> &r, uint32_t unit, uint32_t g, uint32_t blocks)
    {
        const uint32_t x[9] = {r.a[0], r.a[1], r.a[2], r.a[3], r.b[0], r.b[1], r.b[2], r.b[3], r.c};
        for (int i = 0; i < 4; ++i) {
            w[0][i] = __builtin_amdgcn_alignbit(x[i + 1], x[i], 16);
            w[1][i] = x[5 + i];
        }
        transpose(w[0]);
        transpose(w[1]);
        uint32_t p = (x[0] & 0xffffu) | (x[4] & 0xffff0000u);
        if (__builtin_expect((unit + 1) * 8 > blocks, 0)) { // past the row: nothing times zeros
            const uint32_t b = unit * 8 + 2 * g;
            p = b + 1 < blocks ? p : b < blocks ? p & 0xffffu : 0u;
        }
        d[0] = d[2] = p; // every lane of the row: all scales
        swap32(d[0], d[2]);
        d[1] = d[0];
        d[3] = d[2];
        swap16(d[0], d[1]);
        swap16(d[2], d[3]);
    }
    __device__ __forceinline__ float scale(int t) const { return half_value(t % 2 ? d[t / 2] >> 16 : d[t / 2] & 0xffffu); }
    // 16 (q - 8) as signed bytes: values 0-3 and 4-7 of the lane
    __device__ __forceinline__ u2 bytes(int t) const
    {
        const uint32_t u = w[t % 2][t / 2] ^ 0x88888888u;
        return u2{(u << 4) & 0xF0F0F0F0u, u & 0xF0F0F0F0u};
    }
    __device__ __forceinline__ u4 halves(int t) const; // q - 8
};

template <>
struct Unit<true> {
    uint32_t w[2][4];
    uint32_t sc[2], mn[2];
    float d, dmin;

    __device__ __forceinline__ Unit(const Raw<true> &r, uint32_t, uint32_t, uint32_t)
    {
        const uint32_t h0 = r.head[0], s0 = r.head[1], s1 = r.head[2], s2 = r.head[3];
        sc[0] = s0 & 0x3f3f3f3fu;
        sc[1] = (s2 & 0x0f0f0f0fu) | ((s0 >> 2) & 0x30303030u);
        mn[0] = s1 & 0x3f3f3f3fu;
        mn[1] = ((s2 >> 4) & 0x0f0f0f0fu) | ((s1 >> 2) & 0x30303030u);
        d = half_value(h0 & 0xffffu);
        dmin = half_value(h0 >> 16);
        for (int h = 0; h < 2; ++h) {
            for (int i = 0; i < 4; ++i) w[h][i] = r.q[h][i];
            swap32(w[h][0], w[h][2]); // words 0, 1: quarter 2 h of the block, words 2, 3: quarter 2 h + 1
            swap32(w[h][1], w[h][3]);
        }
    }
    __device__ __forceinline__ float scale(int t) const { return static_cast<float>((sc[t / 4] >> (8 * (t % 4))) & 255u); }
    __device__ __forceinline__ u2 bytes(int t) const // q
    {
        const uint32_t u = w[t / 4][t / 2 % 2 * 2], v = w[t / 4][t / 2 % 2 * 2 + 1], s = t % 2 * 4;
        return u2{(u >> s) & 0x0F0F0F0Fu, (v >> s) & 0x0F0F0F0Fu};
    }
    __device__ __forceinline__ u4 halves(int t) const; // q
    __device__ __forceinline__ u4 minima() const       // as halves
    {
        u4 m;
        for (int i = 0; i < 4; ++i) { // two bytes into 1024's mantissa
            const v2h v = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, mn[i / 2], i % 2 ? 0x07030702u : 0x07010700u));
            m[i] = __builtin_bit_cast(uint32_t, v - v2h{static_cast<_Float16>(1024.0f), static_cast<_Float16>(1024.0f)});
        }
        return m;
    }
};

// Two nibbles, in bits 0-3 (or 4-7) of a word's halves, as halves minus `off`.
__device__ __forceinline__ uint32_t low_nibbles(uint32_t u, _Float16 off)
{
    const v2h v = __builtin_bit_cast(v2h, (u & 0x000F000Fu) | 0x64006400u);
    const _Float16 o = static_cast<_Float16>(1024.0f) + off;
    return __builtin_bit_cast(uint32_t, v - v2h{o, o});
}
__device__ __forceinline__ uint32_t high_nibbles(uint32_t u, _Float16 off)
{
    const v2h v = __builtin_bit_cast(v2h, (u & 0x00F000F0u) | 0x64006400u);
    const _Float16 s = static_cast<_Float16>(0.0625f), o = static_cast<_Float16>(-64.0f) - off;
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(v, v2h{s, s}, v2h{o, o}));
}
__device__ __forceinline__ u4 Unit<false>::halves(int t) const
{
    const uint32_t u = w[t % 2][t / 2], v = u >> 8;
    return u4{low_nibbles(u, 8.0f), high_nibbles(u, 8.0f), low_nibbles(v, 8.0f), high_nibbles(v, 8.0f)};
}
__device__ __forceinline__ u4 Unit<true>::halves(int t) const
{
    const uint32_t u = w[t / 4][t / 2 % 2 * 2], v = w[t / 4][t / 2 % 2 * 2 + 1];
    return t % 2 ? u4{high_nibbles(u, 0.0f), high_nibbles(u >> 8, 0.0f), high_nibbles(v, 0.0f), high_nibbles(v >> 8, 0.0f)}
                 : u4{low_nibbles(u, 0.0f), low_nibbles(u >> 8, 0.0f), low_nibbles(v, 0.0f), low_nibbles(v >> 8, 0.0f)};
}

__device__ __forceinline__ v4i mfma(u2 x, u2 w)
{
    return __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, x), __builtin_bit_cast(long, w), v4i{0, 0, 0, 0}, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma(u4 x, u4 w, v4f c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, w), c, 0, 0, 0);
}

// acc[i] (digit g of column i, of row j) += a unit's products.
template <bool Q4K, int N>
__device__ __forceinline__ void digits_unit(const Raw<Q4K> &raw, const u2 *xs, const u2 *sums, const float *scales, uint32_t unit, uint32_t g, uint32_t blocks, float (&acc)[N])
{
    const Unit<Q4K> un(raw, unit, g, blocks);
    float part[N];
    for (int i = 0; i < N; ++i) part[i] = 0.0f;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        const v4i p = mfma(xs[t * 4 * N * 4], un.bytes(t));
        const float f = un.scale(t);
        for (int i = 0; i < N; ++i) part[i] = __builtin_fmaf(f, static_cast<float>(p[i]), part[i]);
    }
    if constexpr (Q4K) {
        const v4i p = mfma(*sums, g == 0 ? u2{un.mn[0], un.mn[1]} : u2{0u, 0u});
        for (int i = 0; i < N; ++i) part[i] = __builtin_fmaf(un.d, part[i], (un.dmin * -32.0f) * static_cast<float>(p[i]));
    }
    for (int i = 0; i < N; ++i) acc[i] = __builtin_fmaf(scales[i], part[i], acc[i]);
}

struct QmPlan {
    uint32_t units;  // of k
    uint32_t tiles;  // of 16 rows
    uint32_t kw;     // digits: waves along k; the others take further tiles
    bool words;      // load_unit's
    uint32_t groups; // halves: of 16 columns
    uint32_t chunks; // parts of k
    uint32_t parts;  // workgroups of a chunk, each with a run of tiles
};

// A wave's share: units [u0, u1) of its rows.
struct QmShare {
    uint32_t kw, tw, wt, u0, u1, blocks;
    uint64_t row_bytes;
    __device__ __forceinline__ QmShare(const QMatArgs &a, const QmPlan &pl, uint32_t wave, bool q4k)
    {
        kw = pl.kw;
        tw = kQmWaves / kw; // both powers of two
        wt = wave / kw;
        const uint32_t wk = wave % kw;
        u0 = static_cast<uint32_t>(static_cast<uint64_t>(pl.units) * wk / kw);
        u1 = static_cast<uint32_t>(static_cast<uint64_t>(pl.units) * (wk + 1) / kw);
        blocks = a.k / 32;
        row_bytes = q4k ? static_cast<uint64_t>(a.k / 256) * 144 : static_cast<uint64_t>(blocks) * 18;
    }
};

// Up to N <= 4 columns, as digits.
template <bool Q4K, int N, bool WORDS>
__global__ __launch_bounds__(kQmBlock, 4) void k_qm_digits(QMatArgs a, QmPlan pl)
{
    constexpr int U = 2; // units in flight
    extern __shared__ u2 laid[];
    __shared__ float part[2][kQmWaves][N][kWave];
    __shared__ uint32_t wides[kQmWaves];
    const uint32_t tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave), j = lane % 16, g = lane / 16;
    const QmShare sh(a, pl, wave, Q4K);
    const unsigned char *w = static_cast<const unsigned char *>(a.w);
    auto row_of = [&](uint32_t tile) { // of this wave's tile; past the last one, rows that are read and dropped
        const uint64_t at = (static_cast<uint64_t>(tile) + sh.wt) * 16 + j;
        return w + (at < a.m ? at : a.m - 1) * sh.row_bytes;
    };
    // the first weights are on their way while the columns are laid out
    const uint32_t step = gridDim.x * sh.tw;
    uint32_t tile = blockIdx.x * sh.tw;
    const unsigned char *row = row_of(tile);
    Raw<Q4K> raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
        if (sh.u0 + i < sh.u1) load_unit<WORDS>(raw[i], row, sh.u0 + i, g, sh.blocks);
    const bool wide = lay_out_digits<Q4K, N, false>(a, pl.units, laid, tid);
    if (lane == 0) wides[wave] = wide;
    __syncthreads();
    bool again = __any(wides[lane % kQmWaves]); // the digits left something over
    // slot j of the instruction's 16 columns is digit j / 4 of column j % 4 (the
    // ones past n repeat the last), so that result i of lane row g is digit g of column i
    const uint32_t c = j % 4 < a.n ? j % 4 : a.n - 1;
    const u2 *xs = laid + (j / 4 * N + c) * 4 + g, *sums = laid + Digits<N>::sums(pl.units) + j / 4 * N + c;
    const float *scales = reinterpret_cast<const float *>(laid + Digits<N>::scales(pl.units));
    float digit = __builtin_bit_cast(float, (127u + 8 * g) << 23) * (Q4K ? 1.0f : 0.0625f);
    uint32_t turn = 0;
    bool left = false; // the digits laid out are what the first ones left
    for (;; tile += step, turn ^= 1) {
        if (tile >= pl.tiles) {
            if (__builtin_expect(!again, 1)) break;
            again = false;
            left = true;
            digit *= 0x1p-30f;
            tile = blockIdx.x * sh.tw;
            __syncthreads(); // the first digits are read
            uint32_t thread = threadIdx.x;
            asm volatile("" : "+v"(thread)); // what the layout derives from it takes no registers ahead of here
            lay_out_digits<Q4K, N, true>(a, pl.units, laid, thread);
            __syncthreads();
            row = row_of(tile);
#pragma unroll
            for (int i = 0; i < U; ++i)
                if (sh.u0 + i < sh.u1) load_unit<WORDS>(raw[i], row, sh.u0 + i, g, sh.blocks);
        }
        float acc[N];
        for (int i = 0; i < N; ++i) acc[i] = 0.0f;
        const unsigned char *next = row_of(tile + step);
        for (uint32_t u = sh.u0; u < sh.u1; u += U) {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (u + i < sh.u1)
                    digits_unit<Q4K, N>(raw[i], xs + (u + i) * Digits<N>::kUnit, sums + (u + i) * 4 * N, scales + (u + i) * N, u + i, g, sh.blocks, acc);
                // the slot's next unit: of this tile, or of the next one
                const bool more = u + i + U < sh.u1;
                if (more || (u + U >= sh.u1 && sh.u0 + i < sh.u1))
                    load_unit<WORDS>(raw[i], more ? row : next, more ? u + i + U : sh.u0 + i, g, sh.blocks);
            }
        }
        row = next;
        for (int i = 0; i < N; ++i) part[turn][wave][i][lane] = acc[i] * digit;
        __syncthreads();
        for (uint32_t e = wave; e < sh.tw * N; e += kQmWaves) { // a wave per tile and column
            const uint32_t t = e / N, i = e % N;
            if (i >= a.n) continue;
            float v = 0.0f;
            for (uint32_t k = 0; k < sh.kw; ++k) v += part[turn][t * sh.kw + k][i][lane];
            // the digits' sum, the small ones first: lane rows 0 + 1, 2 + 3, then both
            uint32_t p0 = __builtin_bit_cast(uint32_t, v), p1 = p0;
            swap16(p0, p1);
            v = __builtin_bit_cast(float, p0) + __builtin_bit_cast(float, p1);
            p0 = p1 = __builtin_bit_cast(uint32_t, v);
            swap32(p0, p1);
            v = __builtin_bit_cast(float, p0) + __builtin_bit_cast(float, p1);
            const uint64_t r = (static_cast<uint64_t>(tile) + t) * 16 + j;
            const bool live = r < a.m && g == 0;
            uint64_t odd = __ballot(live && !(__builtin_fabsf(v) < __builtin_inff()));
            float *y = a.y + static_cast<int64_t>(r) * a.y_st[0] + static_cast<int64_t>(i) * a.y_st[1];
            if (__builtin_expect(left, 0) && live) v += *y; // this lane's own; one that is not finite is walked once more
            if (__builtin_expect(odd != 0, 0) && column_nan(a.x + static_cast<int64_t>(i) * a.x_st[1], a.x_st[0], a.k)) {
                odd = 0;
                v = __builtin_nanf("");
            }
            while (__builtin_expect(odd != 0, 0)) {
                const int l = __builtin_ctzll(odd);
                odd &= odd - 1;
                const float f = walk_row<Q4K>(w + (r - j + l) * sh.row_bytes, a.x + static_cast<int64_t>(i) * a.x_st[1], a.x_st[0], a.k);
                if (lane == static_cast<uint32_t>(l)) v = f;
            }
            if (live) *y = v;
        }
    }
}

// Up to 16 columns a workgroup, as halves.  NR: a quarter of them, rounded up.
template <bool Q4K, int NR, bool WORDS>
__global__ __launch_bounds__(kQmBlock, 4) void k_qm_halves(QMatArgs a, QmPlan pl)
{
    constexpr int U = 2; // units in flight
    extern __shared__ u4 pieces[];
    const uint32_t tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave), j = lane % 16, g = lane / 16;
    const uint32_t c0 = blockIdx.y * 16, n = a.n - c0 < 16 ? a.n - c0 : 16;
    const uint32_t chunk = blockIdx.x / pl.parts, part = blockIdx.x - chunk * pl.parts;
    const uint32_t u0 = static_cast<uint32_t>(static_cast<uint64_t>(pl.units) * chunk / pl.chunks);
    const uint32_t u1 = static_cast<uint32_t>(static_cast<uint64_t>(pl.units) * (chunk + 1) / pl.chunks), units = u1 - u0;
    const uint32_t end = static_cast<uint32_t>(static_cast<uint64_t>(pl.tiles) * (part + 1) / pl.parts);
    uint32_t tile = static_cast<uint32_t>(static_cast<uint64_t>(pl.tiles) * part / pl.parts) + wave;
    const uint32_t blocks = a.k / 32;
    const uint64_t row_bytes = Q4K ? static_cast<uint64_t>(a.k / 256) * 144 : static_cast<uint64_t>(blocks) * 18;
    const unsigned char *w = static_cast<const unsigned char *>(a.w);
    auto row_of = [&](uint32_t t) { // past the last one, rows that are read and dropped
        const uint64_t at = static_cast<uint64_t>(t) * 16 + j;
        return w + (at < a.m ? at : a.m - 1) * row_bytes;
    };
    // the first weights are on their way while the columns are laid out
    const unsigned char *row = row_of(tile);
    Raw<Q4K> raw[U];
#pragma unroll
    for (uint32_t i = 0; i < U; ++i)
        if (i < units) load_unit<WORDS>(raw[i], row, u0 + i, g, blocks);
    // a unit of a column per half wave, two at a time, so that their loads overlap
    const uint32_t i32 = lane % 32, halves = 2 * kQmWaves;
    for (uint32_t e0 = tid / 32; e0 < units * n; e0 += 2 * halves) {
        float v[2][8];
#pragma unroll
        for (uint32_t b = 0; b < 2; ++b) {
            const uint32_t e = e0 + b * halves, c = e / units, unit = e - c * units;
            if (e < units * n) load_values<Q4K>(a, a.x + static_cast<int64_t>(c0 + c) * a.x_st[1], (u0 + unit) * 8 + i32 / 4, i32 % 4, v[b]);
        }
#pragma unroll
        for (uint32_t b = 0; b < 2; ++b) {
            const uint32_t e = e0 + b * halves, c = e / units, unit = e - c * units;
            if (e < units * n) lay_out_halves<Q4K>(v[b], units, unit, i32, c, pieces);
        }
    }
    __syncthreads();
    // slot j of the instruction's 16 columns is column 4 (j % 4) + j / 4, so
    // that result i of lane row g is column 4 i + g; the slots past n repeat
    uint32_t c = (j % 4) * 4 + j / 4;
    c = c < n ? c : n - 1;
    const u4 *x = pieces + c * 4 + g, *sums = pieces + units * kHalvesUnit + c * 4 + g;
    const v4f *scales = reinterpret_cast<const v4f *>(pieces + units * (kHalvesUnit + 16 * 4)) + g;
    const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
    float *to = static_cast<float *>(a.workspace) + (static_cast<uint64_t>(blockIdx.y) * pl.chunks + chunk) * pl.tiles * (NR * kWave) + lane;
    for (; tile < end; tile += kQmWaves) {
        float acc[NR];
        for (int i = 0; i < NR; ++i) acc[i] = 0.0f;
        const unsigned char *next = row_of(tile + kQmWaves);
        for (uint32_t u = 0; u < units; u += U) {
#pragma unroll
            for (uint32_t i = 0; i < U; ++i) {
                if (u + i < units) {
                    const Unit<Q4K> un(raw[i], u0 + u + i, g, blocks);
                    const u4 *xs = x + (u + i) * kHalvesUnit;
                    float p[NR];
                    for (int q = 0; q < NR; ++q) p[q] = 0.0f;
#pragma unroll
                    for (int t = 0; t < 8; ++t) {
                        const u4 q = un.halves(t);
                        const v4f r = mfma(xs[halves_at(t, 0)], q, mfma(xs[halves_at(t, 1)], q, zero));
                        const float f = un.scale(t);
                        for (int k = 0; k < NR; ++k) p[k] = __builtin_fmaf(f, r[k], p[k]);
                    }
                    if constexpr (Q4K) {
                        const v4f r = mfma(sums[(u + i) * (16 * 4)], un.minima(), zero);
                        for (int k = 0; k < NR; ++k) p[k] = __builtin_fmaf(un.d, p[k], (un.dmin * -64.0f) * r[k]);
                    }
                    const v4f scale = scales[(u + i) * 4];
                    for (int k = 0; k < NR; ++k) acc[k] = __builtin_fmaf(scale[k], p[k], acc[k]);
                }
                // the slot's next unit: of this tile, or of the next one
                const bool more = u + i + U < units;
                if (more || (u + U >= units && i < units))
                    load_unit<WORDS>(raw[i], more ? row : next, u0 + (more ? u + i + U : i), g, blocks);
            }
        }
        row = next;
        for (int i = 0; i < NR; ++i) to[static_cast<uint64_t>(tile) * (NR * kWave) + i * kWave] = acc[i];
    }
}

// Adds up the chunks' parts, a wave per tile and quarter of columns.
template <bool Q4K, int NR>
__global__ __launch_bounds__(kBlock) void k_qm_sum(QMatArgs a, QmPlan pl)
{
    const uint32_t lane = threadIdx.x % kWave, j = lane % 16, g = lane / 16;
    const uint64_t run = static_cast<uint64_t>(pl.tiles) * NR, all = run * pl.groups;
    const uint64_t row_bytes = Q4K ? static_cast<uint64_t>(a.k / 256) * 144 : static_cast<uint64_t>(a.k / 32) * 18;
    const unsigned char *w = static_cast<const unsigned char *>(a.w);
    for (uint64_t e = static_cast<uint64_t>(blockIdx.x) * (kBlock / kWave) + threadIdx.x / kWave; e < all; e += static_cast<uint64_t>(gridDim.x) * (kBlock / kWave)) {
        const uint64_t group = e / run, at = e - group * run, tile = at / NR;
        const float *from = static_cast<const float *>(a.workspace) + (group * pl.chunks * run + at) * kWave + lane;
        float v = 0.0f;
        for (uint32_t k0 = 0; k0 < pl.chunks; k0 += 8) {
            float p[8];
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) p[k] = k0 + k < pl.chunks ? from[(k0 + k) * run * kWave] : 0.0f;
            for (int k = 0; k < 8; ++k) v += p[k];
        }
        const uint64_t r = tile * 16 + j, col = group * 16 + 4 * (at - tile * NR) + g;
        const bool live = r < a.m && col < a.n;
        uint64_t odd = __ballot(live && !(__builtin_fabsf(v) < __builtin_inff()));
        for (uint32_t q = 0; __builtin_expect(odd != 0, 0) && q < 4; ++q) { // a column of this wave's
            const uint64_t lanes = 0xffffull << (16 * q);
            if (!(odd & lanes) || !column_nan(a.x + static_cast<int64_t>(col - g + q) * a.x_st[1], a.x_st[0], a.k)) continue;
            odd &= ~lanes;
            if (g == q) v = __builtin_nanf("");
        }
        while (__builtin_expect(odd != 0, 0)) {
            const int l = __builtin_ctzll(odd);
            odd &= odd - 1;
            const float f = walk_row<Q4K>(w + (tile * 16 + l % 16) * row_bytes, a.x + static_cast<int64_t>(col - g + l / 16) * a.x_st[1], a.x_st[0], a.k);
            if (lane == static_cast<uint32_t>(l)) v = f;
        }
        if (live) a.y[static_cast<int64_t>(r) * a.y_st[0] + static_cast<int64_t>(col) * a.y_st[1]] = v;
    }
}

uint32_t qm_cus()
{
    static const uint32_t cus = [] {
        int dev = 0, n = 0;
        if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
            n = 256;
        return static_cast<uint32_t>(n);
    }();
    return cus;
}

// Columns that are laid out as digits: up to four whose digits and waves' sums
// let two workgroups share a compute unit, or one where there is no more than a
// tile to each; 0: as halves.  Every workgroup lays out all of k: 4 columns of
// 4096x4096 7.9 us against 9.4 as halves, of 4096x11008 18.7 (a workgroup a
// compute unit) against 13.1; 2 columns of 11008x4096 (97 KB) 11.3 against 15.0, 4 of
// 8192x4096 (149 KB) 12.3 against 11.9, of 8192x1024 11.2 against 8.9.
int qm_digits(const QMatArgs &a)
{
    if (a.n > 4) return 0;
    const uint64_t units = (static_cast<uint64_t>(a.k) + kQmUnit - 1) / kQmUnit;
    const uint64_t bytes[] = {Digits<1>::bytes(units), Digits<2>::bytes(units), Digits<3>::bytes(units), Digits<4>::bytes(units)};
    const uint64_t lds = bytes[a.n - 1] + a.n * (2 * kQmBlock * sizeof(float)) + kQmWaves * sizeof(uint32_t);
    return lds <= kQmLds || (lds <= kQmLdsAlone && a.m <= 16 * qm_cus()) ? static_cast<int>(a.n) : 0;
}

QmPlan qm_plan(const QMatArgs &a)
{
    QmPlan pl{};
    pl.units = (a.k + kQmUnit - 1) / kQmUnit;
    pl.tiles = static_cast<uint32_t>((static_cast<uint64_t>(a.m) + 15) / 16);
    pl.kw = pl.units >= 8 ? 8 : pl.units >= 4 ? 4 : pl.units >= 2 ? 2 : 1;
    pl.words = reinterpret_cast<uintptr_t>(a.w) % 4 == 0 && a.k % 64 == 0;
    pl.groups = (a.n + 15) / 16;
    // Halves, by sets of a tile a wave and chunk.  Four units (68 KB, two
    // workgroups a compute unit) write the fewest parts: 5 columns of
    // 4096x151936 99 us, 103 with two units.  Fewer sets go in chunks of two
    // units, to a workgroup a compute unit: 15 columns of 4096x11008 15.5 us, 16.3
    // with two workgroups, 17.3 with four units; and of one unit where those
    // leave compute units idle: 12 columns of 1024x2000 7.4 us, 8.3 with two units.
    const uint64_t sets = (static_cast<uint64_t>(pl.tiles) + kQmWaves - 1) / kQmWaves;
    auto work = [&](uint32_t chunk) { return sets * pl.groups * ((pl.units + chunk - 1) / chunk); };
    const bool large = work(4) >= 4 * qm_cus();
    const uint32_t chunk = large ? 4 : work(2) >= qm_cus() ? 2 : 1;
    pl.chunks = (pl.units + chunk - 1) / chunk;
    uint64_t parts = (large ? 2 : 1) * qm_cus() / (static_cast<uint64_t>(pl.chunks) * pl.groups);
    // In eights, a row's chunks run on one of the eight XCDs, whose L2 holds
    // the lines that two chunks share (15 columns of 4096x11008 in 88 parts
    // 17.1 us, in 86 18.5).
    if (parts > 8) parts = parts / 8 * 8;
    pl.parts = static_cast<uint32_t>(parts < 1 ? 1 : parts < sets ? parts : sets);
    return pl;
}

uint32_t qm_quarter(const QMatArgs &a) { return a.n > 12 ? 4 : (a.n + 3) / 4; }

// Workgroups for tiles taken `per` at a time: even shares of what runs at once.
uint32_t qm_grid(const QmPlan &pl, uint32_t per)
{
    const uint32_t wgs = (pl.tiles + per - 1) / per, most = 2 * qm_cus(), rounds = (wgs + most - 1) / most;
    return (wgs + rounds - 1) / rounds;
}

template <bool Q4K, int N>
void qm_run_digits(const QMatArgs &a, const QmPlan &pl, hipStream_t stream)
{
    const uint32_t grid = qm_grid(pl, kQmWaves / pl.kw), lds = static_cast<uint32_t>(Digits<N>::bytes(pl.units));
    if (pl.words) k_qm_digits<Q4K, N, true><<<grid, kQmBlock, lds, stream>>>(a, pl);
    else k_qm_digits<Q4K, N, false><<<grid, kQmBlock, lds, stream>>>(a, pl);
}

template <bool Q4K, int NR>
void qm_run_halves(const QMatArgs &a, const QmPlan &pl, hipStream_t stream)
{
    const dim3 grid(pl.chunks * pl.parts, pl.groups);
    const uint32_t lds = (pl.units + pl.chunks - 1) / pl.chunks * kHalvesBytes;
    if (pl.words) k_qm_halves<Q4K, NR, true><<<grid, kQmBlock, lds, stream>>>(a, pl);
    else k_qm_halves<Q4K, NR, false><<<grid, kQmBlock, lds, stream>>>(a, pl);
    const uint64_t sums = (static_cast<uint64_t>(pl.tiles) * NR * pl.groups + kBlock / kWave - 1) / (kBlock / kWave);
    k_qm_sum<Q4K, NR><<<static_cast<uint32_t>(sums < 65536 ? sums : 65536), kBlock, 0, stream>>>(a, pl);
}

template <bool Q4K>
void qm_run(const QMatArgs &a, const QmPlan &pl, hipStream_t stream)
{
    switch (qm_digits(a)) {
    case 1: return qm_run_digits<Q4K, 1>(a, pl, stream);
    case 2: return qm_run_digits<Q4K, 2>(a, pl, stream);
    case 3: return qm_run_digits<Q4K, 3>(a, pl, stream);
    case 4: return qm_run_digits<Q4K, 4>(a, pl, stream);
    }
    switch (qm_quarter(a)) {
    case 1: return qm_run_halves<Q4K, 1>(a, pl, stream);
    case 2: return qm_run_halves<Q4K, 2>(a, pl, stream);
    case 3: return qm_run_halves<Q4K, 3>(a, pl, stream);
    default: return qm_run_halves<Q4K, 4>(a, pl, stream);
    }
}

// Products run in parts of columns and rows whose partial sums take 256 MB of
// workspace at most: kilobytes, by tile, 16 columns and chunk of k.  Parts are
// of eight tiles, one a wave, or more, but where k is so long that
// the sums of fewer fill it (k past 2^25: 2^16 chunks of it are 64 MB a tile).
constexpr uint64_t kQmPartials = 1u << 18;

struct QmPart {
    uint32_t rows, columns;
};
QmPart qm_part(const QMatArgs &a)
{
    const QmPlan pl = qm_plan(a);
    if (qm_digits(a)) return {a.m, a.n};
    const uint64_t all = static_cast<uint64_t>(pl.chunks) * pl.tiles;
    uint64_t groups = all * pl.groups <= kQmPartials ? pl.groups : all < kQmPartials ? kQmPartials / all : 1;
    if (groups > 4096) groups = 4096; // within a grid's second axis
    uint64_t tiles = pl.tiles;
    if (all * groups > kQmPartials) { // one group: a tile and chunk take quarters of a kilobyte
        const uint64_t fit = kQmPartials * 4 / qm_quarter(a) / pl.chunks;
        tiles = pl.chunks * kQmWaves < kQmPartials ? kQmPartials / pl.chunks : fit < kQmWaves ? fit : kQmWaves;
    }
    const uint64_t rows = tiles * 16, columns = groups * 16;
    return {static_cast<uint32_t>(rows < a.m ? rows : a.m), static_cast<uint32_t>(columns < a.n ? columns : a.n)};
}

} // namespace

uint64_t quant_mat_workspace_bytes(const QMatArgs &a)
{
    const QmPart part = qm_part(a);
    uint64_t most = 0;
    for (const uint32_t m : {part.rows, a.m % part.rows}) // whole parts and what is left of them
        for (const uint32_t n : {part.columns, a.n % part.columns}) {
            QMatArgs b = a;
            b.m = m;
            b.n = n;
            if (m == 0 || n == 0 || qm_digits(b)) continue;
            const QmPlan pl = qm_plan(b);
            const uint64_t bytes = static_cast<uint64_t>(pl.chunks) * pl.tiles * pl.groups * qm_quarter(b) * kWave * sizeof(float);
            most = bytes > most ? bytes : most;
        }
    return most;
}

hipError_t launch_quant_mat(const QMatArgs &a, hipStream_t stream)
{
    const QmPart part = qm_part(a);
    const uint64_t row_bytes = static_cast<uint64_t>(a.k) / (a.q4k ? 256 : 32) * (a.q4k ? 144 : 18);
    QMatArgs b = a;
    for (uint64_t r = 0; r < a.m; r += part.rows) {
        b.m = static_cast<uint32_t>(a.m - r < part.rows ? a.m - r : part.rows);
        b.w = static_cast<const unsigned char *>(a.w) + r * row_bytes;
        for (uint64_t c = 0; c < a.n; c += part.columns) {
            b.n = static_cast<uint32_t>(a.n - c < part.columns ? a.n - c : part.columns);
            b.x = a.x + static_cast<int64_t>(c) * a.x_st[1];
            b.y = a.y + static_cast<int64_t>(r) * a.y_st[0] + static_cast<int64_t>(c) * a.y_st[1];
            const QmPlan pl = qm_plan(b);
            if (b.q4k) qm_run<true>(b, pl, stream);
            else qm_run<false>(b, pl, stream);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

} // namespace emel
