// paged_attn.hpp -- the attention of one new token per sequence over a paged
// cache: the kernel that paged.hip builds for halves, and a source for each pair of
// types for packed rows.
#pragma once

#include "paged.hpp"

namespace emel {
namespace {

// ---- attention of one new token per sequence ------------------------------------------
//
// A row is one (sequence, cache head, group of up to 16 of its query heads);
// its positions are cut into units of kPaUnit tokens, and all units of all
// rows, sequence after sequence, are dealt out in equal runs to the grid's
// workgroups, so ragged batches and single long sequences both fill the chip.
// A workgroup's run falls into segments, one per row it touches.  Of a
// segment's units each of the four waves takes 32 tokens:
//   scores   S[token, head] = K q^T on 16x16x32 matrix instructions: a lane's
//            operand is 8 consecutive halves of its token, as loaded.  q is
//            f32: it goes in as several halves (below), so a score is as
//            exact as f32 sums are.
//   softmax  a lane then holds 8 scores of one head; running maximum m, sum l.
//   values   out^T[dim, head] = V^T P^T: the instruction's inner index is the
//            token, in any order that both operands share.  Lane (c, g) loads
//            the VW dims from VW c on of tokens 4g .. 4g+3 of both 16-token
//            tiles; 16-bit permutes of its own registers turn them into operands,
//            and its scores are the other operand where they stand.
// The weights P, and q, go in as halves that add up to f32's 24 bits for bf16
// (three) and 22 for f16 (hi + lo): a third f16 half would be half as many
// instructions again for less than f32's sums over a head's dims or a sequence's
// tokens lose.  f16's are scaled so that the largest is near 2^14: lo keeps its 11 bits down
// to 2^-16 of that, and 2^-39 of it below, where lo is subnormal (hi is from
// 2^-28 on).  A subnormal factor also costs the instruction low bits: halves of
// the cache below 2^-14 count to about 2^-38 of what they are multiplied by.
// A wave's (m, l, out) are joined through LDS, a row's segments of several
// workgroups through the workspace by the last of them to finish: stores and
// loads at agent scope and an arrival counter, as in reduce.hip.  The order
// of every sum depends on the lengths alone.
//
// Long caches are bound by HBM: 64 sequences of 90 to 9000 tokens with 32/8 heads of
// 128 take 106 us (4.9 TB/s), two of 40001 to 60001 with 32/32 heads 274 us (6.0 TB/s).  A
// single sequence of 4001 tokens takes 13 us, most of it latency: lengths,
// page ids, K and V one after the other, then the join (about 5 us).
//
// Splitting a factor into parts breaks 0 * inf and inf - inf.  A wave whose
// results are not all finite walks its tokens again one by one in f32, as the
// formula stands, and takes those (but for heads whose query holds a NaN: one
// slot of a batch that nobody filled made 64 sequences of 3000 tokens 3.9 ms
// instead of 142 us, and does no more).  So does one whose sums pass 2^97, which
// bf16's range allows: their weighted mean is finite where the sums of this wave or of
// the row's waves together are not.  The walk takes bf16 values by 2^-34, and a maximum
// 34 above its own, which is what the joins weigh a part by.

// Packed rows go the same way with their whole numbers as f16 halves, which are exact:
//   scores   a block's products with q, two halves a value, times the block's
//            scale in f32, added up over the blocks.
//   values   out^T[dim, head] = N^T (w d)^T: a weight by the scale of its token's block
//            is one f32 factor, cut into hi + lo.  Each column has a power of two for
//            each set of blocks (`raised`: its exponent, which out keeps until the end) that
//            holds the largest such factor so far between 2^11 and 2^15: one is off by 2^-22
//            of itself, or 2^-36 of that largest where lo is subnormal, whatever scales tokens
//            of next to no weight have.  The power is 2^94 at most, so that factors stay in
//            f32's range: beside weights whose scales are 0 one is off by 2^-118 of the
//            largest weight.
// A 32-token step of a head of 128 in Q4_0 is some 400 vector instructions, most of
// them numbers made halves, and 32 matrix ones for 4.6 KB: what bounds short and middle
// rows (64 sequences of 90 to 9000 tokens, 32/8 heads of 128: 54.8 us, 148 MB, 2.7
// TB/s).  A token's rows are scattered over its page besides: 64 of 8000 take 175 us with
// a token's heads in a row, 133 with a head's tokens in a row; over the same pages for
// all, which the caches hold, 120 and 112.  Long rows in
// Q8_0 are bound by HBM (two of 40001 to 60001 with 32/32 heads: 164 us, 870 MB, 5.3
// TB/s).  One sequence of 4001 takes 12.4 us, as with halves: latency.
// A row's end runs once a workgroup, from cold: loops that were unrolled, 42 KB of code
// with the rest, made the last workgroups of rows take 10 to 15 us longer than the 22 KB here.

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

template <bool BF16>
__device__ __forceinline__ v4f mfma32(u4 a, u4 b, v4f c)
{
    if constexpr (BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// Parts of an f32 factor: bf16 takes its 24 bits as three truncated eights,
// f16 its upper 22 as two elevens (the caller scales it into f16's range).
template <bool BF16>
constexpr int kParts = BF16 ? 3 : 2;

template <bool BF16>
__device__ __forceinline__ void split(float x, uint32_t part[3])
{
    if constexpr (BF16) {
        const uint32_t b = __builtin_bit_cast(uint32_t, x);
        part[0] = b >> 16;
        const float r = x - __builtin_bit_cast(float, b & 0xffff0000u);
        const uint32_t rb = __builtin_bit_cast(uint32_t, r);
        part[1] = rb >> 16;
        part[2] = __builtin_bit_cast(uint32_t, r - __builtin_bit_cast(float, rb & 0xffff0000u)) >> 16;
    } else {
        const _Float16 hi = static_cast<_Float16>(x);
        part[0] = __builtin_bit_cast(uint16_t, hi);
        part[1] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(x - static_cast<float>(hi)));
    }
}

// ---- packed rows: whole numbers as halves --------------------------------------------------
//
// 1024 + n is the half whose low bits are n: a mask gives it, one packed sum
// takes 1024 (and 8 or 128) away, exactly.  A nibble that stands four bits up is
// 1024 + 16 n, which the same instruction divides by 16.

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

// `magic` is twice the half 1024.

__device__ __forceinline__ uint32_t pk_low(uint32_t x, float less, uint32_t magic)
{
    const _Float16 l = static_cast<_Float16>(less);
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, x | magic) - v2h{l, l});
}
__device__ __forceinline__ uint32_t pk_high(uint32_t x, uint32_t magic)
{
    const v2h y = __builtin_bit_cast(v2h, x | magic), part = {0.0625f16, 0.0625f16}, less = {-72.0f16, -72.0f16};
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(y, part, less));
}

// An eight of Q4_0, and of Q8_0, in order.
__device__ __forceinline__ u4 pk_halves4(uint32_t w, uint32_t magic)
{
    const uint32_t s = w >> 8;
    return u4{pk_low(w & 0x000f000fu, 1032.0f, magic), pk_high(w & 0x00f000f0u, magic), pk_low(s & 0x000f000fu, 1032.0f, magic),
              pk_high(s & 0x00f000f0u, magic)};
}
__device__ __forceinline__ u4 pk_halves8(uint32_t w0, uint32_t w1, uint32_t magic)
{
    w0 ^= 0x80808080u;
    w1 ^= 0x80808080u;
    return u4{pk_low(__builtin_amdgcn_perm(0, w0, 0x0c010c00u), 1152.0f, magic), pk_low(__builtin_amdgcn_perm(0, w0, 0x0c030c02u), 1152.0f, magic),
              pk_low(__builtin_amdgcn_perm(0, w1, 0x0c010c00u), 1152.0f, magic), pk_low(__builtin_amdgcn_perm(0, w1, 0x0c030c02u), 1152.0f, magic)};
}

// One value of two tokens: the byte that `pick` takes of each, and of Q4_0 its j-th nibble.
__device__ __forceinline__ uint32_t pk_pair4(uint32_t a, uint32_t b, uint32_t pick, int j, uint32_t magic)
{
    const uint32_t x = __builtin_amdgcn_perm(b, a, pick);
    return j ? pk_high(x & 0x00f000f0u, magic) : pk_low(x & 0x000f000fu, 1032.0f, magic);
}
__device__ __forceinline__ uint32_t pk_pair8(uint32_t a, uint32_t b, uint32_t pick, uint32_t magic)
{
    return pk_low(__builtin_amdgcn_perm(b, a, pick) ^ 0x00800080u, 1152.0f, magic);
}

// Value d of a packed row.
template <bool Q4>
__device__ __forceinline__ float pk_value(const uint16_t *row, uint32_t blocks, uint32_t d)
{
    const uint8_t *bytes = reinterpret_cast<const uint8_t *>(row);
    const uint32_t block = d / 32, unit = d % 32 / 8 * blocks + block, i = d % 8;
    const float scale = pk_scale(row[(Q4 ? 8 : 16) * blocks + block]);
    if constexpr (Q4) return static_cast<float>(static_cast<int>((bytes[4 * unit + i / 4 + i % 2 * 2] >> (i / 2 % 2 * 4)) & 15) - 8) * scale;
    else return static_cast<float>(static_cast<int8_t>(bytes[8 * unit + i])) * scale;
}

// max / sum over the four 16-lane rows of a wave: every lane gets the result
// of the lanes that share its low four bits.
template <class F>
__device__ __forceinline__ float rows16(float v, F f)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto p = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    const uint32_t p0 = p[0], p1 = p[1];
    const uint32_t c = __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(float, p0), __builtin_bit_cast(float, p1)));
    const auto q = __builtin_amdgcn_permlane32_swap(c, c, false, false);
    const uint32_t q0 = q[0], q1 = q[1];
    return f(__builtin_bit_cast(float, q0), __builtin_bit_cast(float, q1));
}

// Inclusive sum over the lanes up to each: within rows of 16 by shifts, then
// each row's last lane to the rows behind it.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_or_zero(uint32_t v)
{
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v)
{
    v += dpp_or_zero<0x111, 0xF>(v); // row_shr 1, 2, 4, 8
    v += dpp_or_zero<0x112, 0xF>(v);
    v += dpp_or_zero<0x114, 0xF>(v);
    v += dpp_or_zero<0x118, 0xF>(v);
    v += dpp_or_zero<0x142, 0xA>(v); // row_bcast 15 into rows 1 and 3
    v += dpp_or_zero<0x143, 0xC>(v); // row_bcast 31 into rows 2 and 3
    return v;
}

struct PaSeq {
    uint32_t first, tokens, units;
    bool bad;
};

__device__ __forceinline__ int32_t pa_len(const PagedAttnArgs &a, uint32_t s)
{
    return a.lengths[static_cast<int64_t>(s) * a.lengths_st];
}

__device__ __forceinline__ PaSeq pa_seq(const PagedAttnArgs &a, int32_t len)
{
    PaSeq q;
    q.bad = len < 0 || static_cast<uint64_t>(len) > static_cast<uint64_t>(a.max_pages) * a.page;
    const uint32_t n = q.bad ? 0u : static_cast<uint32_t>(len);
    q.first = a.window && n > a.window ? n - a.window : 0u;
    q.tokens = n - q.first;
    q.units = q.tokens ? (q.tokens + kPaUnit - 1) / kPaUnit : 1u; // a row without tokens still has an output
    return q;
}

__device__ __forceinline__ void pa_store(float *p, float v)
{
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float pa_load(const float *p)
{
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void pa_store2(float *p, float x, float y)
{
    const uint64_t v = __builtin_bit_cast(uint32_t, x) | static_cast<uint64_t>(__builtin_bit_cast(uint32_t, y)) << 32;
    __hip_atomic_store(reinterpret_cast<uint64_t *>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 pa_load2(const float *p)
{
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return __builtin_bit_cast(float2, v);
}

// tanh to a few units in the last place: its series to x^9 below 1/4 (the next term is
// 2^-27 of x), 1 - 2 / (e^2x + 1) above.
__device__ __forceinline__ float pa_tanh(float x)
{
    const float s = x * x;
    const float p = x - x * s * (0.333333343f - s * (0.133333340f - s * (0.0539682545f - s * 0.0218694881f)));
    const float e = 1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * 2.88539008177792681472f) + 1.0f);
    return __builtin_fabsf(x) < 0.25f ? p : e;
}

// 2^(m - ref) of a part whose maximum is m, in a whole whose maximum is ref.
__device__ __forceinline__ float pa_weight(float m, float ref)
{
    return __builtin_amdgcn_exp2f(m - (ref == -__builtin_inff() ? 0.0f : ref));
}

// ---- the end of a packed segment -------------------------------------------------------------
//
// The waves' parts joined into the result, or into this workgroup's slot of the
// workspace and by the last workgroup of the row from all slots, as the halves'
// rows end; a slot is the heads' maxima, their sums and values.

struct PaEnd {
    bool empty, whole;
    uint32_t heads, h0, s, w0, lane_row, pieces; // w0: the row's first bundle
};

__device__ __forceinline__ void pa_ends(const PagedAttnArgs &a, const PaPlan &pl, const PaEnd &n, float *slot, float *joined,
                                        const float *wm, const float *wl, uint32_t *last, uint32_t tid)
{
    constexpr uint32_t kWaves = kBlock / kWave;
    const uint32_t dim = a.dim, pitch = dim + 4, all = n.heads, cells = all * dim;
    float *out = a.y + static_cast<int64_t>(n.h0) * a.y_st[1] + static_cast<int64_t>(n.s) * a.y_st[2];
    auto put = [&](uint32_t h, uint32_t d, float x, float y) {
        float *o = out + static_cast<int64_t>(d) * a.y_st[0] + static_cast<int64_t>(h) * a.y_st[1];
        o[0] = x;
        o[a.y_st[0]] = y;
    };
    // the waves' maximum and sum of a head, and each wave's weight
    auto join = [&](uint32_t h, float f[kWaves], float &sum) {
        float top = wm[h];
        for (uint32_t w = 1; w < kWaves; ++w) top = __builtin_fmaxf(top, wm[w * 16 + h]);
        sum = 0.0f;
        for (uint32_t w = 0; w < kWaves; ++w) {
            f[w] = pa_weight(wm[w * 16 + h], top);
            sum += wl[w * 16 + h] * f[w];
        }
        return top;
    };
    for (uint32_t e = 2 * tid; e < cells; e += 2 * kBlock) {
        const uint32_t h = pl.dim.div(e), d = e - h * dim;
        float f[kWaves], sum, x = 0.0f, y = 0.0f;
        join(h, f, sum);
        for (uint32_t w = 0; w < kWaves; ++w) {
            const float *from = joined + (w * all + h) * pitch + d;
            x += from[0] * f[w];
            y += from[1] * f[w];
        }
        if (!n.whole) pa_store2(slot + 2 * kPaLead + e, x, y);
        else if (n.empty) put(h, d, 0.0f, 0.0f);
        else put(h, d, x * (1.0f / sum), y * (1.0f / sum));
    }
    if (__builtin_expect(n.whole, 0)) return;
    if (tid < all) {
        float f[kWaves], sum;
        pa_store(slot + tid, join(tid, f, sum));
        pa_store(slot + kPaLead + tid, sum);
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
        uint32_t *arrived = pl.arrived + static_cast<size_t>(n.w0 * pl.side + n.lane_row) * kPaLine;
        *last = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n.pieces - 1;
        if (*last) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!*last) return;
    // Short code, as a row's last workgroup is the only one that runs it: what it
    // would take longest for is instructions that no cache holds.
    const uint32_t pieces = n.pieces;
    const size_t stride = static_cast<size_t>(2) * pl.side * pl.slot;
    const float *from = pl.parts + static_cast<size_t>(2 * (n.w0 * pl.side + n.lane_row)) * pl.slot;
    auto piece = [&](uint32_t p) { return from + p * stride + (p == 0 ? pl.slot : 0); };
    float *jl = joined, *weight = joined + kPaLead; // each head's sum, [piece][head]
    constexpr uint32_t kAtOnce = 16;
    float2 v[kAtOnce] = {};
    auto ask = [&](uint32_t p0, uint32_t e) {
#pragma unroll
        for (uint32_t i = 0; i < kAtOnce; ++i)
            if (p0 + i < pieces) v[i] = pa_load2(piece(p0 + i) + 2 * kPaLead + e);
    };
    // The first loads of everything go out together: the thread's first pair,
    // maxima and sums (16 threads a head).
    if (2 * tid < cells) ask(0, 2 * tid);
    const uint32_t h1 = tid / 16 < all ? tid / 16 : 0, i1 = tid % 16;
    float pm[4], ps[4], top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t p = i1 + 16 * i;
        pm[i] = p < pieces ? pa_load(piece(p) + h1) : -__builtin_inff();
        ps[i] = p < pieces ? pa_load(piece(p) + kPaLead + h1) : 0.0f;
        top = __builtin_fmaxf(top, pm[i]);
    }
#pragma unroll 1
    for (uint32_t p = i1 + 64; p < pieces; p += 16) top = __builtin_fmaxf(top, pa_load(piece(p) + h1));
    for (int d = 8; d > 0; d >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, d, 16));
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const float f = pa_weight(pm[i], top);
        sum += ps[i] * f;
        if (i1 + 16 * i < pieces) weight[(i1 + 16 * i) * all + h1] = f;
    }
#pragma unroll 1
    for (uint32_t p = i1 + 64; p < pieces; p += 16) {
        const float f = pa_weight(pa_load(piece(p) + h1), top);
        sum += pa_load(piece(p) + kPaLead + h1) * f;
        weight[p * all + h1] = f;
    }
    for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 16);
    if (i1 == 0 && tid / 16 < all) jl[h1] = sum;
    __syncthreads();
#pragma unroll 1
    for (uint32_t e = 2 * tid; e < cells; e += 2 * kBlock) {
        const uint32_t h = pl.dim.div(e);
        const float *f = weight + h;
        float x = 0.0f, y = 0.0f;
#pragma unroll 1
        for (uint32_t p0 = 0; p0 < pieces; p0 += kAtOnce) {
            if (p0 > 0 || e != 2 * tid) ask(p0, e);
#pragma unroll
            for (uint32_t i = 0; i < kAtOnce; ++i, f += all)
                if (p0 + i < pieces) {
                    x += v[i].x * *f;
                    y += v[i].y * *f;
                }
        }
        const float scale = 1.0f / jl[h];
        put(h, e - h * dim, n.empty ? 0.0f : x * scale, n.empty ? 0.0f : y * scale);
    }
}

// KS: 32-dim steps of a score; VW: dims of a lane's values (4, 8, 12 or 16; 2
// KS of packed pages).
// FOLD: of packed pages, the columns of a product that a head takes (1, 2, 4 or
// 8, with 16 columns for all heads of a row); 0 of halves.  Column p of a head stands for every
// block b with b % FOLD == p.  Its query is 0 in the other blocks, so what the
// products of a set of FOLD consecutive blocks add up in it is one block's part of a
// score, to be scaled by that block; a head's columns are added last.  Its weights
// are by the scales of its own block of a set, and of the rows of a set's values only
// those of that block count, the others are never looked at.  A lane so scales and splits
// 8 weights a set and step, not a block and step, and its rows may be of any of a set's
// blocks: it loads what lies side by side.  All of that costs as many matrix instructions
// as FOLD 1 does.
template <PaPages PAGES, int KS, int VW, int FOLD = 0>
__global__ __launch_bounds__(kBlock, pa_per_cu(KS, FOLD)) void k_pa_attn(PagedAttnArgs a, PaPlan pl)
{
    constexpr bool BF16 = PAGES == PaPages::Bf16, PACKED = PAGES > PaPages::Bf16;
    constexpr int P = kParts<BF16>;
    constexpr int kWaves = kBlock / kWave;
    constexpr bool K4 = PAGES >= PaPages::Q4Q8, V4 = PAGES == PaPages::Q8Q4 || PAGES == PaPages::Q4Q4;
    constexpr int KI = K4 ? 8 : 16, VI = V4 ? 8 : 16; // packed: halves of a block's whole numbers
    constexpr int kAcc = PACKED ? 2 * KS : VW;
    constexpr bool kEarly = PACKED && KS <= 4 && FOLD >= KS;
    constexpr int F = PACKED ? FOLD : 1, kSets = PACKED ? (KS + F - 1) / F : 1;
    // packed: blocks of set e; words that a lane loads of a token's, and of those before
    constexpr auto blocks_of = [](int e) { return e < KS / F ? F : KS - e * F; };
    constexpr auto words_of = [](int n) { return V4 ? (n + 3) / 4 : (n + 1) / 2; };
    constexpr int kWords = PACKED ? KS / F * words_of(F) + (KS % F ? words_of(KS % F) : 0) : 1;
    constexpr float kLift = BF16 ? 0.0f : 14.0f;
    constexpr int kRaise = 94;
    // [wave][head of the group][dim]; packed: before that the score operands, by
    // planes of 64 lanes and a zero
    extern __shared__ __attribute__((aligned(16))) float joined[];
    __shared__ u4 qop[PACKED ? 1 : KS * P * kWave]; // score operands, lane after lane
    constexpr uint32_t kPlane = kWave + 1;
    __shared__ int64_t off[kWaves][2][32];       // a step's tokens in the key and value pools
    __shared__ float scales[PACKED ? kWaves : 1][2][PACKED ? KS : 1][32]; // packed: of their blocks
    __shared__ float wm[kWaves][16], wl[kWaves][16], jl[16];
    __shared__ uint32_t scan[kWaves], found[2];
    __shared__ uint32_t last;
    const uint32_t thread = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(thread / kWave);
    const uint32_t dim = a.dim, pitch = dim + 4; // of a head in joined

    // Rows of a few units are mostly set-up, which more workgroups hide; long
    // ones stream best with two a compute unit (64 sequences of 90 to 9000
    // tokens 106 us, 113 with three; 640 of 100 tokens 90 us, 77 with three).
    // Packed rows are unpacked as much as loaded, and take all.
    auto share_of = [&](uint32_t units) { return !PACKED && units > 4 * a.seqs ? pl.few : pl.grid; };
    // This workgroup's run of units, and the sequence it starts in.  A row's
    // set-up and end cost about a unit: it counts as one more, but where there
    // is no more than a unit to a workgroup (that would only part the rows).
    // Packed rows are short, and a token's heads share cache lines: `side` rows
    // go to as many workgroups of one die, which walk the same tokens at one time
    // (blocks are dealt to eight dies in turn).  `block` counts such bundles.
    const uint32_t turn = blockIdx.x / kDies, lane_row = PACKED ? turn % pl.side : 0;
    const uint32_t block = PACKED ? turn / pl.side * kDies + blockIdx.x % kDies : blockIdx.x;
    const uint32_t rows = PACKED ? pl.rows / pl.side : pl.rows;
    const uint32_t first_lane = thread % kWave;
    uint32_t total, run, cur, base; // base: the sequence's first unit
    uint32_t more = 0; // packed: workgroups that take a unit above `run`, the first ones
    uint32_t s, setup;
    int32_t s_len;
    if (__builtin_expect(a.seqs <= kWave, 1)) { // every wave for itself: a sequence per first_lane
        const int32_t len = first_lane < a.seqs ? pa_len(a, first_lane) : 0;
        const uint32_t mine = first_lane < a.seqs ? pa_seq(a, len).units : 0;
        uint32_t pre = wave_scan(mine);
        const uint32_t all = lane_u32(pre, kWave - 1);
        const FastDiv share = share_of(all);
        setup = all * rows > share.d;
        total = (all + setup * a.seqs) * rows;
        pre += setup * (first_lane + 1);
        run = share.div(PACKED ? total : total + share.d - 1);
        cur = block * run;
        if constexpr (PACKED) {
            more = total - run * share.d;
            cur += block < more ? block : more;
        }
        if (cur >= total) return;
        s = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(__popcll(__ballot(first_lane < a.seqs && pre * rows <= cur))));
        base = lane_u32(pre - mine - setup, s) * rows;
        s_len = static_cast<int32_t>(lane_u32(static_cast<uint32_t>(len), s));
    } else {
        const uint32_t per = (a.seqs + kBlock - 1) / kBlock;
        const uint32_t s0 = thread * per < a.seqs ? thread * per : a.seqs, s1 = s0 + per < a.seqs ? s0 + per : a.seqs;
        uint32_t mine = 0;
#pragma unroll 1
        for (uint32_t i = s0; i < s1; ++i) mine += pa_seq(a, pa_len(a, i)).units;
        uint32_t pre = wave_scan(mine);
        if (first_lane == kWave - 1) scan[wave] = pre;
        __syncthreads();
        uint32_t all = 0;
        for (int w = 0; w < kWaves; ++w) {
            if (static_cast<uint32_t>(w) < wave) pre += scan[w];
            all += scan[w];
        }
        const FastDiv share = share_of(all);
        setup = all * rows > share.d;
        pre += setup * s0 - mine;
        mine += setup * (s1 - s0);
        total = (all + setup * a.seqs) * rows;
        run = share.div(PACKED ? total : total + share.d - 1);
        cur = block * run;
        if constexpr (PACKED) {
            more = total - run * share.d;
            cur += block < more ? block : more;
        }
        if (cur >= total) return;
        if (mine && pre * rows <= cur && cur < (pre + mine) * rows) {
            uint32_t i = s0;
#pragma unroll 1
            for (uint32_t u = pa_seq(a, pa_len(a, i)).units + setup; (pre + u) * rows <= cur; u = pa_seq(a, pa_len(a, i)).units + setup) {
                pre += u;
                ++i;
            }
            found[0] = i;
            found[1] = pre;
        }
        __syncthreads();
        s = found[0];
        base = found[1] * rows;
        s_len = pa_len(a, s);
    }
    const uint32_t end = PACKED ? cur + run + (block < more) : cur + run < total ? cur + run : total;
    // the block that has a unit
    auto block_of = [&](uint32_t u) {
        if (!PACKED) return u / run;
        const uint32_t longer = more * (run + 1);
        return u < longer ? u / (run + 1) : more + (u - longer) / run;
    };

    PaSeq sq = pa_seq(a, s_len);
    uint32_t units = sq.units + setup;
    uint32_t row = (cur - base) / units;
    uint32_t row_at = base + row * units;

    while (cur < end) {
        // What follows from the thread's number is worked out where it is used:
        // the compiler would gather all of it ahead of this loop, some 470
        // instructions that a workgroup of one short segment waits for.
        uint32_t tid = thread;
        asm volatile("" : "+v"(tid));
        const uint32_t lane = tid % kWave, col = lane % 16, g = lane / 16;
        // the head of a column, and which of each set's blocks it stands for
        const uint32_t head = col / F, part = col % F, quarter = col % 4;
        const uint32_t n0 = cur - row_at, n1 = end - row_at < units ? end - row_at : units;
        const uint32_t u0 = n0 > setup ? n0 - setup : 0, u1 = n1 - setup;
        if (PACKED && n1 <= setup) break; // a row's start, whose units are all another's
        const uint32_t mine = PACKED ? row * pl.side + lane_row : row;
        const uint32_t kh = pl.hgroups.div(mine), h0 = kh * pl.group + (mine - kh * pl.hgroups.d) * 16;
        const uint32_t heads = (kh + 1) * pl.group - h0 < 16 ? (kh + 1) * pl.group - h0 : 16;

        const uint16_t *kbase = a.k_pool.data + static_cast<int64_t>(kh) * a.k_pool.st_head;
        const uint16_t *vbase = a.v_pool.data + static_cast<int64_t>(kh) * a.v_pool.st_head;
        const int32_t *table = a.table + static_cast<int64_t>(s) * a.table_st[1];
        float m = -__builtin_inff(), l = 0.0f;
        v4f acc[kAcc];
        for (int j = 0; j < kAcc; ++j) acc[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        int raised[kSets]; // packed: acc of a set is taken by 2^raised
        for (int &r : raised) r = kRaise;
        bool bad = sq.bad;

        const uint32_t t_end = sq.tokens < u1 * kPaUnit ? sq.tokens : u1 * kPaUnit;
        uint32_t t0 = u0 * kPaUnit + wave * 32;
        // the page of lane % 32's token, a step ahead of its use
        auto page_of = [&](uint32_t t) {
            return t < t_end ? table[static_cast<int64_t>(pl.page.div(sq.first + t)) * a.table_st[0]] : 0;
        };
        int32_t next = PACKED ? 0 : page_of(t0 + lane % 32);

        // score operands, lane (col, g): dims 32 e + 8 g .. + 7 of head col;
        // each wave lays out every fourth e
        float inv = 1.0f;
        u4 *planes = reinterpret_cast<u4 *>(joined);
        {
            const float *q = a.q + static_cast<int64_t>(h0 + head) * a.q_st[1] + static_cast<int64_t>(s) * a.q_st[2];
            const float c = a.soft_cap > 0.0f ? a.scale / a.soft_cap : a.scale * 1.44269504088896340736f;
            auto eight = [&](uint32_t e, float x[8]) {
                const uint32_t d = 32 * e + 8 * g;
                if (head < heads && d < dim) {
                    if (__builtin_expect(a.q_st[0] == 1, 1)) {
                        const v4f lo = *reinterpret_cast<const v4f_any *>(q + d), hi = *reinterpret_cast<const v4f_any *>(q + d + 4);
                        for (int i = 0; i < 4; ++i) {
                            x[i] = lo[i] * c;
                            x[4 + i] = hi[i] * c;
                        }
                    } else {
                        if constexpr (PACKED) {
                            const float *from = q + static_cast<int64_t>(d) * a.q_st[0];
#pragma unroll 1
                            for (int i = 0; i < 8; ++i, from += a.q_st[0])
                                for (int j = 0; j < 8; ++j) x[j] = i == j ? *from * c : x[j];
                        } else {
                            for (int i = 0; i < 8; ++i) x[i] = q[static_cast<int64_t>(d + i) * a.q_st[0]] * c;
                        }
                    }
                } else {
                    for (int i = 0; i < 8; ++i) x[i] = 0.0f;
                }
            };
            float up = 1.0f;
            constexpr int kKept = kSets <= 4 ? kSets : 1;
            float own_q[kKept][8]; // packed: of the column's blocks, where they are few
            if constexpr (!BF16) { // the head's largest value to [2^14, 2^15)
                float top = 0.0f;
                auto fold = [&](const float x[8]) {
                    for (int i = 0; i < 8; ++i) top = __builtin_fmaxf(top, __builtin_fabsf(x[i]));
                };
                if constexpr (PACKED) {
                    if constexpr (kKept == kSets) {
                        for (int e = 0; e < kSets; ++e) eight(e * F + part, own_q[e]);
                        for (int e = 0; e < kSets; ++e) fold(own_q[e]);
                    } else {
#pragma unroll 1
                        for (int e = 0; e < kSets; ++e) {
                            eight(e * F + part, own_q[0]);
                            fold(own_q[0]);
                        }
                    }
                } else if constexpr (KS <= 4) { // all loads at once
                    float x[KS][8];
                    for (int e = 0; e < KS; ++e) eight(e, x[e]);
                    for (int e = 0; e < KS; ++e) fold(x[e]);
                } else {
#pragma unroll 2
                    for (int e = 0; e < KS; ++e) {
                        float x[8];
                        eight(e, x);
                        fold(x);
                    }
                }
                top = rows16(top, [](float u, float v) { return __builtin_fmaxf(u, v); });
                if constexpr (F > 1)
                    for (int x = 1; x < F; x *= 2) top = __builtin_fmaxf(top, __shfl_xor(top, x, kWave));
                int e = static_cast<int>((__builtin_bit_cast(uint32_t, top) >> 23) & 255u) - 127;
                e = top == 0.0f || e == 128 ? 0 : e < -110 ? -110 : e; // infinite: the wave walks below
                up = __builtin_bit_cast(float, static_cast<uint32_t>(127 + 14 - e) << 23);
                inv = __builtin_bit_cast(float, static_cast<uint32_t>(127 - 14 + e) << 23);
            }
            if constexpr (PACKED) {
                auto lay = [&](uint32_t e, const float x[8]) {
                    u4 w[P];
                    for (int i = 0; i < 4; ++i) {
                        uint32_t even[3], odd[3];
                        split<false>(x[2 * i] * up, even);
                        split<false>(x[2 * i + 1] * up, odd);
                        for (int p = 0; p < P; ++p) w[p][i] = even[p] | (odd[p] << 16);
                    }
                    for (int p = 0; p < P; ++p) {
                        planes[(e * P + p) * kPlane + lane] = w[p];
                        if (lane == 0) planes[(e * P + p) * kPlane + kWave] = u4{0, 0, 0, 0};
                    }
                };
                if constexpr (kKept == kSets) {
                    for (int e = 0; e < kSets; ++e)
                        if (static_cast<uint32_t>(e) == wave) lay(e, own_q[e]);
                } else {
#pragma unroll 1
                    for (uint32_t e = wave; e < kSets; e += kWaves) {
                        eight(e * F + part, own_q[0]);
                        lay(e, own_q[0]);
                    }
                }
            }
#pragma unroll 1
            for (uint32_t e = wave; e < (PACKED ? 0 : KS); e += kWaves) {
                float x[8];
                eight(e, x);
                u4 w[P];
                for (int i = 0; i < 4; ++i) {
                    uint32_t even[3], odd[3];
                    split<BF16>(x[2 * i] * up, even);
                    split<BF16>(x[2 * i + 1] * up, odd);
                    for (int p = 0; p < P; ++p) w[p][i] = even[p] | (odd[p] << 16);
                }
                for (int p = 0; p < P; ++p) qop[(e * P + p) * kWave + lane] = w[p];
            }
        }
        __syncthreads();
        // The packed loop runs ahead of itself: a step's keys are asked for when
        // the last one's scores are done with theirs, its values behind the last
        // one's sums, so each load has half a step of instructions to come in (the
        // last step asks for its own last token once more).
        uint32_t kw[2][PACKED ? (K4 ? 1 : 2) * KS : 1];
        uint32_t vw[8][kWords];              // the words of each token that hold the lane's values
        uint16_t bits[PACKED ? KS : 1];      // the scales of lane % 32's token, of keys or values
        uint32_t inside = 0; // the place of its token in the page `next`
        // Behind the end the last token stands for what is missing, so that
        // these loads need no branch, which would have to wait for them.
        auto ask_page = [&](uint32_t t) {
            t = sq.first + (t < t_end ? t : t_end - 1);
            const uint32_t page = pl.page.div(t);
            inside = t - page * pl.page.d;
            next = table[static_cast<int64_t>(page) * a.table_st[0]];
        };
        auto ask_keys = [&](uint32_t t1) {
            const bool ok = static_cast<uint32_t>(next) < a.pages;
            bad |= !ok;
            const int64_t p = ok ? next : 0, i = inside;
            const PagePool &pool = lane < 32 ? a.k_pool : a.v_pool;
            const int64_t o = p * pool.st_page + i * pool.st_tok;
            __builtin_amdgcn_wave_barrier();
            off[wave][lane / 32][lane % 32] = o;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            ask_page(t1 + lane % 32 + kPaUnit);
            const uint16_t *row = (lane < 32 ? kbase + KI * KS : vbase + VI * KS) + o; // a row's last KS halves
            __builtin_memcpy(bits, row, sizeof bits);
            for (int b = 0; b < 2; ++b) __builtin_memcpy(kw[b], kbase + off[wave][0][16 * b + col] + g * (KI * KS / 4), sizeof kw[b]);
        };
        // Of a quarter of a set's numbers, which lie side by side, four lanes take
        // a quarter each: bytes from `skip` on, of a word that two or all of them load where it is less.
        constexpr int kByte = V4 ? 1 : 2; // bytes of a lane and block
        auto skip = [&](int n) { return n * kByte == 1 ? 0u : n * kByte == 2 ? quarter / 2 * 4 : quarter * n * kByte; };
        auto first = [&](int n) { return n * kByte == 1 ? quarter : n * kByte == 2 ? quarter % 2 * 2 : 0u; };
        auto ask_values = [&] {
            for (int b = 0; b < 8; ++b) {
                const uint8_t *p = reinterpret_cast<const uint8_t *>(vbase + off[wave][1][16 * (b / 4) + 4 * g + b % 4] + col / 4 * (VI * KS / 4));
                for (int e = 0; e < kSets; ++e) {
                    const int n = blocks_of(e);
                    __builtin_memcpy(&vw[b][e * words_of(F)], p + 4 * kByte * F * e + skip(n), 4 * words_of(n));
                }
            }
        };
        // the scales of this step into LDS; what is not a token counts for nothing
        auto place_scales = [&] {
            __builtin_amdgcn_wave_barrier();
            for (int e = 0; e < KS; ++e) scales[wave][lane / 32][e][lane % 32] = t0 + lane % 32 < t_end || lane < 32 ? pk_scale(bits[e]) : 0.0f;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        };
        // the scales of the column's block of set e, of the lane's four tokens of tile b
        auto four = [&](int of, int e, int b) {
            const uint32_t at = e * F + part;
            return *reinterpret_cast<const v4f *>(&scales[wave][of][KS % F == 0 || at < KS ? at : 0][16 * b + 4 * g]);
        };
        uint32_t magic = 0x64006400u; // in a register: an instruction holds one constant
        asm volatile("" : "+v"(magic));
        float one = 1.0f; // one that the compiler does not know: x * one - h takes a half as it is, x - h a conversion first
        asm volatile("" : "+s"(one));
        if constexpr (PACKED) {
            if (t0 < t_end) {
                ask_page(t0 + lane % 32);
                ask_keys(t0);
                ask_values();
            }
        }
        for (; PACKED && t0 < t_end; t0 += kPaUnit) {
            float z[8];
            u4 early[kEarly ? KS * P : 1]; // the operands, asked for ahead of the scales where registers hold them
            if constexpr (kEarly) {
                for (int i = 0; i < KS * P; ++i) early[i] = planes[(i / P / F * P + i % P) * kPlane + (part == static_cast<uint32_t>(i / P % F) ? lane : kWave)];
                __builtin_amdgcn_sched_barrier(0);
            }
            place_scales();
            v4f sum[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
            for (int e = 0; e < kSets; ++e) {
                v4f c[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
                for (int i = e * F; i < e * F + blocks_of(e); ++i) {
                    const uint32_t at = part == static_cast<uint32_t>(i % F) ? lane : kWave; // no other block's
                    u4 x[2];
                    for (int b = 0; b < 2; ++b) {
                        if constexpr (K4) x[b] = pk_halves4(kw[b][i], magic);
                        else x[b] = pk_halves8(kw[b][2 * i], kw[b][2 * i + 1], magic);
                    }
                    for (int p = P - 1; p >= 0; --p)
                        for (int b = 0; b < 2; ++b) c[b] = mfma32<false>(x[b], kEarly ? early[kEarly ? i * P + p : 0] : planes[(e * P + p) * kPlane + at], c[b]);
                }
                if (e == kSets - 1) ask_keys(t0 + kPaUnit);
                for (int b = 0; b < 2; ++b) {
                    const v4f d = four(0, e, b);
                    for (int i = 0; i < 4; ++i)
                        sum[b][i] = blocks_of(e) == F || part < static_cast<uint32_t>(blocks_of(e)) ? __builtin_fmaf(c[b][i], d[i], sum[b][i]) : sum[b][i];
                }
            }
            for (int i = 0; i < 8; ++i) {
                float x = sum[i / 4][i % 4];
                if constexpr (F > 1) x += dpp_f32<kDppXor1>(x);
                if constexpr (F > 2) x += dpp_f32<kDppXor2>(x);
                if constexpr (F > 4) x += dpp_f32<kDppHalfMirror>(x);
                z[i] = x;
            }
            float by = inv; // what scores are to be multiplied by
            if (__builtin_expect(a.soft_cap > 0.0f, 0)) {
                for (int i = 0; i < 8; ++i) z[i] = pa_tanh(z[i] * inv) * (a.soft_cap * 1.44269504088896340736f);
                by = 1.0f;
            }
            if (t0 + 32 > t_end)
                for (int b = 0; b < 8; ++b)
                    if (t0 + 16 * (b / 4) + 4 * g + b % 4 >= t_end) z[b] = -__builtin_inff();
            float top = z[0];
            for (int i = 1; i < 8; ++i) top = __builtin_fmaxf(top, z[i]);
            top = rows16(top, [](float x, float y) { return __builtin_fmaxf(x, y); }) * by;
            int due[kSets] = {}; // what a set's power would be past its most: its sums are taken down by it
            if (__any(top > m)) {
                // whole numbers, so that it moves by powers of two, which the sets' powers take up
                const float m1 = __builtin_ceilf(__builtin_fmaxf(m, top));
                const int down = static_cast<int>(__builtin_fmaxf(m - m1, -1000.0f)); // m = -inf: all of it
                for (int e = 0; e < kSets; ++e) {
                    const int to = raised[e] - down;
                    raised[e] = to < kRaise ? to : kRaise;
                    due[e] = raised[e] - to;
                }
                l *= __builtin_ldexpf(1.0f, down);
                m = m1;
            }
            // 1 for the largest weight: a power of two within the exponent would cost it bits
            const float ref = m == -__builtin_inff() ? 0.0f : m;
            float w[8];
            for (int i = 0; i < 8; ++i) {
                w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[i], by, -ref));
                l += w[i];
            }
            for (int e = 0; e < kSets; ++e) {
                u4 hi, lo; // the weights by a block's scales, as halves that add up to 22 bits
                float x[8], most = 0.0f;
                const float up = __builtin_ldexpf(1.0f, raised[e]);
                for (int b = 0; b < 2; ++b) {
                    const v4f d = four(1, e, b);
                    for (int i = 0; i < 4; ++i) x[4 * b + i] = w[4 * b + i] * up * d[i];
                }
                for (int i = 0; i < 8; ++i) most = __builtin_fmaxf(most, __builtin_fabsf(x[i]));
                // A factor past what halves hold: eight times as large ones fit from
                // here on, so that few steps come by.
                if (__any(most >= 0x1p15f || due[e] < 0)) {
                    most = rows16(most, [](float u, float v) { return __builtin_fmaxf(u, v); });
                    const int down = most >= 0x1p15f ? static_cast<int>((__builtin_bit_cast(uint32_t, most) >> 23) & 255u) - 127 - 11 : 0;
                    const float f = __builtin_ldexpf(1.0f, due[e] - down), fx = __builtin_ldexpf(1.0f, -down);
                    raised[e] -= down;
                    for (int j = 2 * F * e; j < 2 * F * e + 2 * blocks_of(e); ++j) acc[j] *= f;
                    for (float &v : x) v *= fx;
                }
                for (int i = 0; i < 4; ++i) {
                    const v2h h = __builtin_convertvector((v2f{x[2 * i], x[2 * i + 1]}), v2h);
                    const v2f r = {__builtin_fmaf(x[2 * i], one, -static_cast<float>(h[0])), __builtin_fmaf(x[2 * i + 1], one, -static_cast<float>(h[1]))};
                    hi[i] = __builtin_bit_cast(uint32_t, h);
                    lo[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, v2h));
                }
                const int n = blocks_of(e);
                for (int j = 0; j < 2 * n; ++j) {
                    // the lane's j-th number of the set, of tokens 2i and 2i + 1
                    const int byte = V4 ? j / 2 : j, word = e * words_of(F) + byte / 4;
                    const uint32_t pick = 0x0c040c00u + (first(n) + byte % 4) * 0x10001u;
                    u4 x;
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (V4) x[i] = pk_pair4(vw[2 * i][word], vw[2 * i + 1][word], pick, j % 2, magic);
                        else x[i] = pk_pair8(vw[2 * i][word], vw[2 * i + 1][word], pick, magic);
                    }
                    v4f &sum = acc[2 * F * e + j];
                    sum = mfma32<false>(x, lo, sum);
                    sum = mfma32<false>(x, hi, sum);
                }
            }
            ask_values();
        }
        for (; !PACKED && t0 < t_end; t0 += kPaUnit) {
            {
                const uint32_t t = t0 + lane % 32;
                const bool ok = t < t_end && static_cast<uint32_t>(next) < a.pages;
                bad |= t < t_end && !ok;
                const int64_t p = ok ? next : 0, i = ok ? pl.page.mod(sq.first + t) : 0;
                const PagePool &pool = lane < 32 ? a.k_pool : a.v_pool;
                __builtin_amdgcn_wave_barrier();
                off[wave][lane / 32][lane % 32] = p * pool.st_page + i * pool.st_tok;
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                next = page_of(t + kPaUnit);
            }
            u4 k[2][KS];
            for (int b = 0; b < 2; ++b) {
                const uint16_t *p = kbase + off[wave][0][16 * b + col];
                for (int e = 0; e < KS; ++e) {
                    const uint32_t d = 32 * e + 8 * g;
                    k[b][e] = *reinterpret_cast<const u4_any *>(p + (d < dim ? d : 0)); // q is 0 past dim
                }
            }
            uint32_t v[8][VW / 2];
            for (int b = 0; b < 8; ++b) {
                const uint16_t *p = vbase + off[wave][1][16 * (b / 4) + 4 * g + b % 4];
                // eights first, then fours behind the eights of all 16 lanes
                for (int e = 0; e < VW / 8; ++e) {
                    const uint32_t d = 128 * e + 8 * col;
                    const u4 x = *reinterpret_cast<const u4_any *>(p + (d < dim ? d : 0));
                    for (int i = 0; i < 4; ++i) v[b][4 * e + i] = x[i];
                }
                if constexpr (VW % 8) {
                    const uint32_t d = VW / 8 * 128 + 4 * col;
                    const u2 x = *reinterpret_cast<const u2_any *>(p + (d < dim ? d : 0));
                    v[b][VW / 2 - 2] = x[0];
                    v[b][VW / 2 - 1] = x[1];
                }
            }
            float z[8];
            for (int b = 0; b < 2; ++b) {
                v4f c = {0.0f, 0.0f, 0.0f, 0.0f};
                for (int e = 0; e < KS; ++e)
                    for (int p = P - 1; p >= 0; --p) c = mfma32<BF16>(k[b][e], qop[(e * P + p) * kWave + lane], c);
                for (int i = 0; i < 4; ++i) z[4 * b + i] = BF16 ? c[i] : c[i] * inv;
            }
            if (__builtin_expect(a.soft_cap > 0.0f, 0))
                for (int i = 0; i < 8; ++i) z[i] = pa_tanh(z[i]) * (a.soft_cap * 1.44269504088896340736f);
            if (t0 + 32 > t_end) { // the sequence ends in this step: nothing of what lies behind it counts
                for (int b = 0; b < 8; ++b) {
                    if (t0 + 16 * (b / 4) + 4 * g + b % 4 < t_end) continue;
                    z[b] = -__builtin_inff();
                    for (int i = 0; i < VW / 2; ++i) v[b][i] = 0;
                }
            }
            float top = z[0];
            for (int i = 1; i < 8; ++i) top = __builtin_fmaxf(top, z[i]);
            top = rows16(top, [](float x, float y) { return __builtin_fmaxf(x, y); });
            if (__any(top > m)) {
                const float m1 = __builtin_fmaxf(m, top);
                const float f = m1 > m ? __builtin_amdgcn_exp2f(m - m1) : 1.0f; // m = -inf: 0
                l *= f;
                for (int j = 0; j < VW; ++j) acc[j] *= f;
                m = m1;
            }
            const float ref = (m == -__builtin_inff() ? 0.0f : m) - kLift;
            uint32_t part[8][3];
            for (int i = 0; i < 8; ++i) {
                const float w = __builtin_amdgcn_exp2f(z[i] - ref);
                l += w;
                split<BF16>(w, part[i]);
            }
            u4 w[P];
            for (int p = 0; p < P; ++p)
                for (int i = 0; i < 4; ++i) w[p][i] = part[2 * i][p] | (part[2 * i + 1][p] << 16);
            for (int j = 0; j < VW; ++j) {
                u4 x;
                for (int i = 0; i < 4; ++i) // halves j of tokens 2i and 2i + 1
                    x[i] = __builtin_amdgcn_perm(v[2 * i + 1][j / 2], v[2 * i][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
                for (int p = P - 1; p >= 0; --p) acc[j] = mfma32<BF16>(x, w[p], acc[j]);
            }
        }

        // packed: of each set the eight g of the column's block, from the rows 4 g
        // + i that hold its numbers
        float eight[kSets][8];
        for (int e = 0; PACKED && e < kSets; ++e) {
            const int n = blocks_of(e);
            for (int i = 0; i < 8; ++i) {
                constexpr int order[8] = {0, 4, 1, 5, 2, 6, 3, 7}; // Q4_0: the nibble of each value
                const int at = V4 ? order[i] : i;
                auto of = [&](int b) { // number `at` of the set's block b: row by row, 2 n of them
                    const int q = 8 * b + at;
                    return acc[2 * F * e + q % (2 * n)][q / (2 * n)];
                };
                eight[e][i] = of(0);
                for (int b = 1; b < n; ++b) eight[e][i] = part == static_cast<uint32_t>(b) ? of(b) : eight[e][i];
            }
            const float down = __builtin_ldexpf(1.0f, -raised[e]);
            for (float &x : eight[e]) x *= down;
        }
        // the wave's part: [head][dim], dims of lane row c = 4 g + i
        float *own = joined + wave * heads * pitch;
        l = rows16(l, [](float x, float y) { return x + y; });
        v4f size = {l, 0.0f, 0.0f, 0.0f};
        for (int e = 0; PACKED && e < kSets; ++e)
            for (int i = 0; i < 8; ++i) size[i % 4] += part < static_cast<uint32_t>(blocks_of(e)) ? __builtin_fabsf(eight[e][i]) : 0.0f;
        for (int j = 0; j < (PACKED ? 0 : kAcc); ++j)
            for (int i = 0; i < 4; ++i) size[i] += __builtin_fabsf(acc[j][i]);
        const bool odd = !((size[0] + size[1]) + (size[2] + size[3]) < (BF16 ? 0x1p97f : __builtin_inff()));
        bad = __any(bad);
        if constexpr (PACKED) __syncthreads(); // the operands' place is the joins' from here on
        if (__builtin_expect(__any(odd && head < heads) && !bad, 0)) {
            // as the formula stands: a head and a token at a time, a lane four dims
            constexpr float down = BF16 ? 0x1p-34f : 1.0f, above = BF16 ? 34.0f : 0.0f;
            for (uint32_t h = 0; h < heads; ++h) {
                const float *q = a.q + static_cast<int64_t>(h0 + h) * a.q_st[1] + static_cast<int64_t>(s) * a.q_st[2];
                float qv[4], av[4] = {}, mm = -__builtin_inff(), ll = 0.0f;
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t d = 4 * lane + i;
                    qv[i] = d < dim ? q[static_cast<int64_t>(d) * a.q_st[0]] : 0.0f;
                }
                // a NaN in q is in every score; the sum that it leaves makes the head NaN
                const bool nan = __any(__builtin_isnan(qv[0]) || __builtin_isnan(qv[1]) || __builtin_isnan(qv[2]) || __builtin_isnan(qv[3]));
                if (nan) ll = __builtin_nanf("");
                for (uint32_t t1 = u0 * kPaUnit + wave * 32; t1 < (nan ? 0 : t_end); t1 += kPaUnit) {
                    for (uint32_t t = t1; t < t1 + 32 && t < t_end; ++t) {
                        const int64_t p = table[static_cast<int64_t>(pl.page.div(sq.first + t)) * a.table_st[0]];
                        const int64_t i0 = pl.page.mod(sq.first + t);
                        const uint16_t *kp = kbase + p * a.k_pool.st_page + i0 * a.k_pool.st_tok;
                        const uint16_t *vp = vbase + p * a.v_pool.st_page + i0 * a.v_pool.st_tok;
                        float zz = 0.0f;
                        auto value = [&](const uint16_t *row, bool key, uint32_t d) {
                            if constexpr (PACKED) return key ? pk_value<K4>(row, KS, d) : pk_value<V4>(row, KS, d);
                            else return from_half<BF16>(row[d]);
                        };
                        for (uint32_t i = 0; i < 4; ++i)
                            if (4 * lane + i < dim) zz += qv[i] * value(kp, true, 4 * lane + i);
                        zz = wave_sum(zz) * a.scale;
                        if (a.soft_cap > 0.0f) zz = a.soft_cap * pa_tanh(zz / a.soft_cap);
                        zz *= 1.44269504088896340736f;
                        const float m1 = __builtin_fmaxf(mm, zz);
                        const float ref = m1 == -__builtin_inff() ? 0.0f : m1;
                        const float f = m1 > mm ? __builtin_amdgcn_exp2f(mm - m1) : 1.0f;
                        const float e = __builtin_amdgcn_exp2f(zz - ref);
                        ll = ll * f + e;
                        for (uint32_t i = 0; i < 4; ++i)
                            if (4 * lane + i < dim) av[i] = av[i] * f + e * (value(vp, false, 4 * lane + i) * down);
                        mm = m1;
                    }
                }
                const float lift = BF16 || PACKED ? 1.0f : 16384.0f; // as the parts of waves that do not walk
                for (uint32_t i = 0; i < 4; ++i)
                    if (4 * lane + i < dim) own[h * pitch + 4 * lane + i] = av[i] * lift;
                if (lane == 0) {
                    wm[wave][h] = mm + above;
                    wl[wave][h] = ll * (lift * down);
                }
            }
        } else if (head < heads) {
            if (g == 0 && part == 0) {
                wm[wave][head] = m;
                wl[wave][head] = bad ? __builtin_nanf("") : l;
            }
            for (int e = 0; PACKED && e < kSets; ++e) {
                const float *x = eight[e];
                float *o = own + head * pitch + 32 * (e * F + part) + 8 * g;
                if (part >= static_cast<uint32_t>(blocks_of(e))) continue;
                *reinterpret_cast<v4f *>(o) = v4f{x[0], x[1], x[2], x[3]};
                *reinterpret_cast<v4f *>(o + 4) = v4f{x[4], x[5], x[6], x[7]};
            }
            for (int i = 0; i < (PACKED ? 0 : 4); ++i) {
                const uint32_t c = 4 * g + i;
                for (int e = 0; e < VW / 8; ++e)
                    if (128 * e + 8 * c < dim)
                        for (int j = 0; j < 8; j += 4)
                            *reinterpret_cast<v4f *>(own + col * pitch + 128 * e + 8 * c + j) =
                                v4f{acc[8 * e + j][i], acc[8 * e + j + 1][i], acc[8 * e + j + 2][i], acc[8 * e + j + 3][i]};
                if constexpr (!PACKED && VW % 8) {
                    const uint32_t d = VW / 8 * 128 + 4 * c;
                    if (d < dim)
                        *reinterpret_cast<v4f *>(own + col * pitch + d) = v4f{acc[VW - 4][i], acc[VW - 3][i], acc[VW - 2][i], acc[VW - 1][i]};
                }
            }
        }
        __syncthreads();
        const bool begins = PACKED ? u0 == 0 : n0 == 0;
        const bool whole = begins && n1 == units;
        const uint32_t w0 = begins ? block : block_of(row_at + (PACKED ? setup : 0)); // the row's first workgroup
        const uint32_t own_block = PACKED ? block * pl.side + lane_row : block;
        float *slot = pl.parts + static_cast<size_t>(2 * own_block + (begins ? 1 : 0)) * pl.slot;
        // the waves' maximum and sum of a head, and each wave's weight
        auto join = [&](uint32_t h, float f[kWaves], float &sum) {
            float top = wm[0][h];
            for (int w = 1; w < kWaves; ++w) top = __builtin_fmaxf(top, wm[w][h]);
            sum = 0.0f;
            for (int w = 0; w < kWaves; ++w) {
                f[w] = pa_weight(wm[w][h], top);
                sum += wl[w][h] * f[w];
            }
            return top;
        };
        asm volatile("" : "+v"(tid));
        if constexpr (PACKED) {
            pa_ends(a, pl, PaEnd{sq.tokens == 0 && !sq.bad, whole, heads, h0, s, w0, lane_row, whole ? 1 : block_of(row_at + units - 1) - w0 + 1}, slot, joined,
                    &wm[0][0], &wl[0][0], &last, tid);
            __syncthreads(); // the next segment reuses the shared arrays
            cur = row_at + n1;
            row_at += units;
            if (++row == rows && cur < end) {
                row = 0;
                sq = pa_seq(a, pa_len(a, ++s));
                units = sq.units + setup;
            }
            continue;
        }
        const uint32_t cells = heads * dim; // dim is even: pairs do not cross heads
        float *out = a.y + static_cast<int64_t>(h0) * a.y_st[1] + static_cast<int64_t>(s) * a.y_st[2];
        auto put = [&](uint32_t h, uint32_t d, float x, float y) {
            float *o = out + static_cast<int64_t>(d) * a.y_st[0] + static_cast<int64_t>(h) * a.y_st[1];
            o[0] = x;
            o[a.y_st[0]] = y;
        };
        for (uint32_t e = 2 * tid; e < cells; e += 2 * kBlock) {
            const uint32_t h = pl.dim.div(e), d = e - h * dim;
            float f[kWaves], sum, x = 0.0f, y = 0.0f;
            join(h, f, sum);
            for (int w = 0; w < kWaves; ++w) {
                x += joined[(w * heads + h) * pitch + d] * f[w];
                y += joined[(w * heads + h) * pitch + d + 1] * f[w];
            }
            if (!whole) pa_store2(slot + 32 + e, x, y);
            else if (sq.tokens == 0 && !sq.bad) put(h, d, 0.0f, 0.0f);
            else put(h, d, x * (1.0f / sum), y * (1.0f / sum));
        }
        if (__builtin_expect(!whole, 0)) {
            if (tid < heads) {
                float f[kWaves], sum;
                pa_store(slot + tid, join(tid, f, sum));
                pa_store(slot + 16 + tid, sum);
            }
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            const uint32_t pieces = (row_at + units - 1) / run - w0 + 1;
            if (tid == 0) {
                uint32_t *arrived = pl.arrived + static_cast<size_t>(w0) * kPaLine;
                last = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == pieces - 1;
                if (last) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (last) {
                asm volatile("" : "+v"(tid));
                auto piece = [&](uint32_t p) { return pl.parts + static_cast<size_t>(2 * (w0 + p) + (p == 0 ? 1 : 0)) * pl.slot; };
                float *weight = joined; // [piece][head]
                // The first loads of everything go out together: maxima and
                // sums (16 threads a head), then the thread's first pair.
                const uint32_t hh = tid / 16 < heads ? tid / 16 : 0, i0 = tid % 16;
                float pm[4], ps[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t p = i0 + 16 * i;
                    const float *from = piece(p < pieces ? p : pieces - 1) + hh;
                    pm[i] = pa_load(from);
                    ps[i] = pa_load(from + 16);
                }
                float2 v[16];
                auto sixteen = [&](uint32_t p0, uint32_t e) {
#pragma unroll
                    for (uint32_t i = 0; i < 16; ++i) v[i] = pa_load2(piece(p0 + i < pieces ? p0 + i : pieces - 1) + 32 + e);
                };
                sixteen(0, 2 * tid < cells ? 2 * tid : 0);
                float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) top = __builtin_fmaxf(top, pm[i]); // a repeated last piece changes nothing
                const uint32_t more = tid / 16 < heads ? pieces : 0; // past 64, of the threads with a head
                for (uint32_t p = i0 + 64; p < more; p += 16) {
                    const float m1 = pa_load(piece(p) + hh);
                    weight[p * heads + hh] = m1;
                    top = __builtin_fmaxf(top, m1);
                }
                for (int d = 8; d > 0; d >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, d, 16));
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t p = i0 + 16 * i;
                    const float f = pa_weight(pm[i], top);
                    if (p < pieces) {
                        sum += ps[i] * f;
                        if (tid / 16 < heads) weight[p * heads + hh] = f;
                    }
                }
                for (uint32_t p = i0 + 64; p < more; p += 16) {
                    const float f = pa_weight(weight[p * heads + hh], top);
                    sum += pa_load(piece(p) + 16 + hh) * f;
                    weight[p * heads + hh] = f;
                }
                for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 16);
                if (i0 == 0 && tid / 16 < heads) jl[hh] = sum;
                __syncthreads();
                for (uint32_t e = 2 * tid; e < cells; e += 2 * kBlock) {
                    const uint32_t h = pl.dim.div(e), d = e - h * dim;
                    float x = 0.0f, y = 0.0f;
                    for (uint32_t p0 = 0; p0 < pieces; p0 += 16) {
                        if (p0 > 0 || e != 2 * tid) sixteen(p0, e);
#pragma unroll
                        for (uint32_t i = 0; i < 16; ++i)
                            if (p0 + i < pieces) {
                                const float f = weight[(p0 + i) * heads + h];
                                x += v[i].x * f;
                                y += v[i].y * f;
                            }
                    }
                    if (sq.tokens == 0 && !sq.bad) put(h, d, 0.0f, 0.0f);
                    else put(h, d, x * (1.0f / jl[h]), y * (1.0f / jl[h]));
                }
            }
        }
        __syncthreads(); // the next segment reuses the shared arrays
        cur = row_at + n1;
        row_at += units;
        if (++row == rows && cur < end) {
            row = 0;
            sq = pa_seq(a, pa_len(a, ++s));
            units = sq.units + setup;
        }
    }
}

} // namespace
} // namespace emel
