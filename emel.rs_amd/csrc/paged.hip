// paged.hip -- the paged key-value cache: new tokens' keys and values rounded or
// packed into their slots and read back, and the attention of one new token per
// sequence over pages of halves.
#include "common.hpp"
#include "launch.hpp"
#include "paged_attn.hpp"

namespace emel {
namespace {

// ---- new tokens into their slots ---------------------------------------------------------
//
// Bound by the tokens' bytes: 4 read and 2 written a value.  A workgroup takes
// T consecutive tokens, eight values a lane and step.  Of tokens with one slot
// the last is stored: each workgroup looks through the slots behind its own and leaves a
// token whose slot a later one names to that one.  Eight tokens a workgroup
// share that look (it reads 4 bytes of each later token, and 8001 tokens of 1024 values took
// 37 us with one token a workgroup, bound by it, and 23.9 with eight: 4.1 TB/s);
// few tokens take one each, for more workgroups.  A launch takes 2^17 tokens
// at most, so that the looks grow with the tokens and not with their square: of
// tokens in different launches the later launch's is stored, being later.
// (2^17 tokens of 1024 values 1000 us, 2^18 2000 against 4000 in one launch;
// 2^20 of 64 values 7.2 ms against 60.  Up to 2^15 tokens the looks are
// a small part: 2^15 of 1024 values 106 us.)

// dim: values of a head, in eights where VEC.
template <bool BF16, uint32_t T, bool VEC>
__global__ __launch_bounds__(kBlock) void k_pa_append(PagedAppendArgs a, FastDiv page, FastDiv head, FastDiv token)
{
    __shared__ uint32_t gone;
    const uint32_t t0 = blockIdx.x * T;
    int32_t mine[T];
    const uint32_t drop = pa_dropped<T>(a, t0, mine, &gone);
    // an item: eight values (or one) of a head, of a token, of keys or values
    for (uint32_t e = threadIdx.x; e < 2 * T * token.d; e += kBlock) {
        const uint32_t i = token.div(e), r = e - i * token.d, k = i % T;
        if ((drop >> k) & 1u) continue;
        const uint32_t h = head.div(r), d = (r - h * head.d) * (VEC ? 8 : 1);
        int32_t slot = mine[0]; // no index at run time: the slots stay in registers
        for (uint32_t q = 1; q < T; ++q) slot = k == q ? mine[q] : slot;
        const uint32_t p = page.div(static_cast<uint32_t>(slot)), at = static_cast<uint32_t>(slot) - p * page.d;
        const bool val = i >= T;
        const float *src = val ? a.v : a.k;
        const int64_t *st = val ? a.v_st : a.k_st;
        const PagePool &pool = val ? a.v_pool : a.k_pool;
        src += d * st[0] + h * st[1] + static_cast<int64_t>(t0 + k) * st[2];
        uint16_t *dst = pool.data + p * pool.st_page + h * pool.st_head + at * pool.st_tok + d;
        if constexpr (VEC) {
            const v4f lo = *reinterpret_cast<const v4f_any *>(src), hi = *reinterpret_cast<const v4f_any *>(src + 4);
            u4 w;
            for (int q = 0; q < 4; ++q) {
                const float x = q < 2 ? lo[2 * q] : hi[2 * q - 4], y = q < 2 ? lo[2 * q + 1] : hi[2 * q - 3];
                w[q] = to_half<BF16>(x) | static_cast<uint32_t>(to_half<BF16>(y)) << 16;
            }
            *reinterpret_cast<u4_any *>(dst) = w;
        } else {
            *dst = to_half<BF16>(*src);
        }
    }
}

// ---- new tokens into packed pages ----------------------------------------------------------
//
// A row is one token's head: dim / 32 blocks of 32 values.  Its whole numbers
// come first, by eights (the first eight of every block, then the second, third
// and fourth: what a lane of the attention reads of a row lies side by side),
// the blocks' f16 scales behind them.  Eight Q4_0 numbers are one word: values 0,
// 2, 4 and 6 in its low half and 1, 3, 5 and 7 in the high one, so that a shift
// and a mask give two neighbours as halves.
//
// A lane packs one eight, four lanes a block: its largest magnitude and, for Q4_0,
// that value's sign go over a quad by DPP.  The numbers are nearest to x / d for
// the scale as it is stored: the quotient by 1/d is off by one at most, and
// x - n d, which is exact in f32 (x is a multiple of 2^-25 d or below d / 2), says so.
//
// Bound by the bytes, 4 read a value and 1.0625 or 0.5625 written: 8001 tokens of 1024
// keys in Q8_0 and values in Q4_0 25.5 us (79 MB, 3.1 TB/s), of which the look through
// the later slots, as for halves, is 4.4; a few tokens by the launch.

// What is to be added to n so that it is the nearest whole number of scales in
// x, ties to even, for an n that is off by one at most.
__device__ __forceinline__ float off_by(float x, float n, float d)
{
    const float over = __builtin_fmaf(-n, d, x) * (d < 0.0f ? -1.0f : 1.0f), half = 0.5f * __builtin_fabsf(d);
    const bool odd = static_cast<int>(n) & 1;
    return over > half || (over == half && odd) ? 1.0f : over < -half || (over == -half && odd) ? -1.0f : 0.0f;
}

// Packs a lane's eight values of a block; every lane of a quad is active.
__device__ __forceinline__ void pack_eight(bool q4, const float x[8], uint8_t *row, uint32_t blocks, uint32_t eight)
{
    const uint32_t block = eight / 4, part = eight % 4, unit = part * blocks + block;
    float high = -__builtin_inff(), low = high, zero = 0.0f; // the largest value, the largest opposite one, 0 or NaN
    for (int i = 0; i < 8; ++i) {
        high = __builtin_fmaxf(high, x[i]);
        low = __builtin_fmaxf(low, -x[i]);
        zero = __builtin_fmaf(x[i], 0.0f, zero);
    }
    high = __builtin_fmaxf(high, dpp_f32<kDppXor1>(high));
    low = __builtin_fmaxf(low, dpp_f32<kDppXor1>(low));
    zero += dpp_f32<kDppXor1>(zero);
    high = __builtin_fmaxf(high, dpp_f32<kDppXor2>(high));
    low = __builtin_fmaxf(low, dpp_f32<kDppXor2>(low));
    zero += dpp_f32<kDppXor2>(zero);
    const float top = __builtin_fmaxf(high, low);
    const bool fine = zero == 0.0f;
    float d = top * (high > low ? -0.125f : 0.125f);
    if (!q4) {
        d = top / 127.0f;
    } else if (__any(high == low)) { // both signs: the first value of that magnitude, by its number and sign
        uint32_t first = ~0u;
        for (int i = 7; i >= 0; --i)
            if (__builtin_fabsf(x[i]) == top) first = (8 * part + i) << 1 | (__builtin_bit_cast(uint32_t, x[i]) >> 31);
        first = min(first, dpp32<kDppXor1>(first));
        first = min(first, dpp32<kDppXor2>(first));
        d = high == low ? top * (first & 1 ? 0.125f : -0.125f) : d;
    }
    const _Float16 scale = static_cast<_Float16>(__builtin_fminf(__builtin_fmaxf(d, -65504.0f), 65504.0f));
    d = static_cast<float>(scale);
    const float inv = d == 0.0f || !fine ? 0.0f : __builtin_amdgcn_rcpf(d);
    float n[8], most = 0.0f;
    for (int i = 0; i < 8; ++i) {
        n[i] = fine ? __builtin_rintf(x[i] * inv) : 0.0f;
        most = __builtin_fmaxf(most, __builtin_fabsf(__builtin_fmaf(-n[i], d, x[i])));
    }
    if (__any(most >= 0.5f * __builtin_fabsf(d))) // seldom: a tie, or 1 / d rounded to the wrong side of one
        for (int i = 0; i < 8; ++i) n[i] += inv == 0.0f ? 0.0f : off_by(x[i], n[i], d);
    uint16_t *scales = reinterpret_cast<uint16_t *>(row + (q4 ? 16 : 32) * blocks);
    if (part == 0) scales[block] = fine ? __builtin_bit_cast(uint16_t, scale) : uint16_t{0x7e00};
    if (q4) {
        uint32_t w = 0;
        for (int i = 0; i < 8; ++i)
            w |= static_cast<uint32_t>(static_cast<int>(__builtin_fminf(__builtin_fmaxf(n[i], -8.0f), 7.0f)) + 8) << (4 * (i / 2 + i % 2 * 4));
        *reinterpret_cast<u1_any *>(row + 4 * unit) = w;
    } else {
        u2 w = {0, 0};
        for (int i = 0; i < 8; ++i)
            w[i / 4] |= (static_cast<uint32_t>(static_cast<int>(__builtin_fminf(__builtin_fmaxf(n[i], -127.0f), 127.0f))) & 255u) << (8 * (i % 4));
        *reinterpret_cast<u2_any *>(row + 8 * unit) = w;
    }
}

// How a workgroup's waves share `jobs` tokens, keys and values apart, of
// `items` lanes' work each: a wave takes the items of one run of 64 for every
// wpc-th job, so that a token's place is the same for its lanes and worked out once.
struct WaveShare {
    uint32_t chunk, chunks, step, job, wpc;
};
__device__ __forceinline__ WaveShare wave_share(uint32_t items)
{
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), chunks = (items + kWave - 1) / kWave;
    const uint32_t wpc = chunks == 1 ? 4 : chunks == 2 ? 2 : 1;
    return {wave / wpc, chunks, 4 / wpc, wave % wpc, wpc};
}

// As k_pk_append for tokens of 64 items or more; UNIT: keys and values are read
// with unit stride.
template <uint32_t T, bool UNIT>
__global__ __launch_bounds__(kBlock) void k_pk_append_wide(PagedAppendArgs a, FastDiv page, FastDiv head, uint32_t items)
{
    __shared__ uint32_t gone;
    const uint32_t t0 = blockIdx.x * T;
    int32_t mine[T];
    const uint32_t drop = pa_dropped<T>(a, t0, mine, &gone);
    constexpr uint32_t kBatch = T == 1 ? 1 : 4;
    const WaveShare w = wave_share(items);
    for (uint32_t c = w.chunk; c < w.chunks; c += w.step) {
        const uint32_t r = c * kWave + threadIdx.x % kWave;
        if (r >= items) continue;
        const uint32_t h = head.div(r), eight = r - h * head.d;
        for (uint32_t j0 = w.job; j0 < 2 * T; j0 += kBatch * w.wpc) {
            float x[kBatch][8];
            uint8_t *row[kBatch];
#pragma unroll
            for (uint32_t n = 0; n < kBatch; ++n) {
                const uint32_t j = j0 + n * w.wpc, k = j % T;
                row[n] = nullptr;
                if (j >= 2 * T || ((drop >> k) & 1u)) continue;
                const bool val = j >= T;
                const int64_t *st = val ? a.v_st : a.k_st;
                const PagePool &pool = val ? a.v_pool : a.k_pool;
                const uint32_t slot = static_cast<uint32_t>(a.slots[static_cast<int64_t>(t0 + k) * a.slots_st]);
                const uint32_t p = page.div(slot), at = slot - p * page.d;
                row[n] = reinterpret_cast<uint8_t *>(pool.data + p * pool.st_page + at * pool.st_tok + h * pool.st_head);
                const float *src = (val ? a.v : a.k) + static_cast<int64_t>(t0 + k) * st[2] + h * st[1] + static_cast<int64_t>(8 * eight) * st[0];
                if constexpr (UNIT) {
                    const v4f lo = *reinterpret_cast<const v4f_any *>(src), hi = *reinterpret_cast<const v4f_any *>(src + 4);
                    for (int q = 0; q < 4; ++q) {
                        x[n][q] = lo[q];
                        x[n][4 + q] = hi[q];
                    }
                } else {
                    for (int q = 0; q < 8; ++q) x[n][q] = src[q * st[0]];
                }
            }
#pragma unroll
            for (uint32_t n = 0; n < kBatch; ++n)
                if (row[n]) pack_eight((j0 + n * w.wpc >= T ? a.v_pool : a.k_pool).kind == PoolKind::Q4_0, x[n], row[n], head.d / 4, eight);
        }
    }
}

template <uint32_t T>
__global__ __launch_bounds__(kBlock) void k_pk_append(PagedAppendArgs a, FastDiv page, FastDiv head, FastDiv token)
{
    __shared__ uint32_t gone;
    const uint32_t t0 = blockIdx.x * T;
    int32_t mine[T];
    const uint32_t drop = pa_dropped<T>(a, t0, mine, &gone);
    // an item: eight values of a head, of a token, of keys or values; a quad of lanes has a block's four
    for (uint32_t e = threadIdx.x; e < 2 * T * token.d; e += kBlock) {
        const uint32_t i = token.div(e), r = e - i * token.d, k = i % T;
        if ((drop >> k) & 1u) continue;
        const uint32_t h = head.div(r), eight = r - h * head.d;
        int32_t slot = mine[0];
        for (uint32_t q = 1; q < T; ++q) slot = k == q ? mine[q] : slot;
        const uint32_t p = page.div(static_cast<uint32_t>(slot)), at = static_cast<uint32_t>(slot) - p * page.d;
        const bool val = i >= T;
        const int64_t *st = val ? a.v_st : a.k_st;
        const PagePool &pool = val ? a.v_pool : a.k_pool;
        const float *src = (val ? a.v : a.k) + static_cast<int64_t>(8 * eight) * st[0] + h * st[1] + static_cast<int64_t>(t0 + k) * st[2];
        float x[8];
        for (int q = 0; q < 8; ++q) x[q] = src[q * st[0]];
        uint16_t *row = pool.data + p * pool.st_page + h * pool.st_head + at * pool.st_tok;
        pack_eight(pool.kind == PoolKind::Q4_0, x, reinterpret_cast<uint8_t *>(row), head.d / 4, eight);
    }
}

// ---- tokens read back ------------------------------------------------------------------------
//
// Bound by the tokens' bytes, 4 written a value: 40001 tokens of 1024 keys and values in
// Q8_0 100 us (415 MB, 4.2 TB/s).  An item is eight values, or one
// of halves whose dim is no multiple of 8.

constexpr uint32_t kPaRead = 8;              // tokens of a workgroup
constexpr uint32_t kPaReadTokens = 1u << 25; // tokens of a launch: its threads are counted in 32 bits

struct ReadItem {
    u4 word;
    uint16_t scale;
};

template <bool EIGHT>
__device__ __forceinline__ ReadItem read_item(const PagePool &pool, const uint16_t *row, uint32_t blocks, uint32_t at)
{
    ReadItem x = {};
    if constexpr (!EIGHT) {
        x.word[0] = row[at];
    } else if (!pool.packed()) {
        x.word = *reinterpret_cast<const u4_any *>(row + 8 * at);
    } else { // part at % 4 of block at / 4
        const uint32_t unit = at % 4 * blocks + at / 4;
        if (pool.kind == PoolKind::Q4_0) {
            x.word[0] = *reinterpret_cast<const u1_any *>(row + 2 * unit);
            x.scale = row[8 * blocks + at / 4];
        } else {
            const u2 w = *reinterpret_cast<const u2_any *>(row + 4 * unit);
            x.word[0] = w[0];
            x.word[1] = w[1];
            x.scale = row[16 * blocks + at / 4];
        }
    }
    return x;
}

template <bool EIGHT>
__device__ __forceinline__ void write_item(PoolKind kind, const ReadItem &it, float *dst, int64_t st)
{
    constexpr int N = EIGHT ? 8 : 1;
    float x[N];
    if (EIGHT && kind == PoolKind::Q8_0) {
        const float d = pk_scale(it.scale);
        for (int q = 0; q < N; ++q) x[q] = static_cast<float>(static_cast<int8_t>(it.word[q / 4] >> (8 * (q % 4)))) * d;
    } else if (EIGHT && kind == PoolKind::Q4_0) {
        const float d = pk_scale(it.scale);
        for (int q = 0; q < N; ++q) x[q] = static_cast<float>(static_cast<int>((it.word[0] >> (q % 2 * 16 + q / 2 * 4)) & 15u) - 8) * d;
    } else {
        for (int q = 0; q < N; ++q) {
            const uint16_t b = static_cast<uint16_t>(it.word[q / 2] >> (16 * (q % 2)));
            x[q] = kind == PoolKind::Bf16 ? from_half<true>(b) : from_half<false>(b);
        }
    }
    if (EIGHT && st == 1) { // nothing here reads them again
        for (int q = 0; q < N; q += 4)
            __builtin_nontemporal_store((v4f{x[q], x[(q + 1) % N], x[(q + 2) % N], x[(q + 3) % N]}), reinterpret_cast<v4f_any *>(dst + q));
        return;
    }
    for (int q = 0; q < N; ++q) dst[q * st] = x[q];
}

template <bool EIGHT>
__global__ __launch_bounds__(kBlock) void k_pa_read(PagedReadArgs a, uint32_t per, FastDiv page, FastDiv head, FastDiv token)
{
    const uint64_t slots = static_cast<uint64_t>(a.page) * a.pages;
    const uint32_t t0 = blockIdx.x * per, blocks = head.d / 4; // of a packed row
    for (uint32_t e = threadIdx.x; e < 2 * per * token.d; e += kBlock) {
        const uint32_t i = token.div(e), r = e - i * token.d;
        const bool val = i >= per;
        const uint32_t t = t0 + (val ? i - per : i);
        const int32_t slot = t < a.tokens ? a.slots[static_cast<int64_t>(t) * a.slots_st] : -1;
        if (slot < 0 || static_cast<uint64_t>(slot) >= slots) continue;
        const uint32_t h = head.div(r), at = r - h * head.d;
        const uint32_t p = page.div(static_cast<uint32_t>(slot)), in = static_cast<uint32_t>(slot) - p * page.d;
        const PagePool &pool = val ? a.v_pool : a.k_pool;
        const int64_t *st = val ? a.v_st : a.k_st;
        const ReadItem it = read_item<EIGHT>(pool, pool.data + p * pool.st_page + h * pool.st_head + in * pool.st_tok, blocks, at);
        write_item<EIGHT>(pool.kind, it, (val ? a.v : a.k) + static_cast<int64_t>(EIGHT ? 8 * at : at) * st[0] + h * st[1] + static_cast<int64_t>(t) * st[2], st[0]);
    }
}

// As k_pa_read by eights, for tokens of 64 items or more, whose waves are whole
// (8000 tokens of 64 items in Q4_0 10.1 us, 10.5 there; of 32 8.3 and 7.1).
__global__ __launch_bounds__(kBlock) void k_pa_read_wide(PagedReadArgs a, uint32_t per, FastDiv page, FastDiv head, uint32_t items)
{
    constexpr uint32_t kBatch = 2;
    const uint64_t slots = static_cast<uint64_t>(a.page) * a.pages;
    const uint32_t t0 = blockIdx.x * per, blocks = head.d / 4;
    const WaveShare w = wave_share(items);
    for (uint32_t c = w.chunk; c < w.chunks; c += w.step) {
        const uint32_t r = c * kWave + threadIdx.x % kWave;
        if (r >= items) continue;
        const uint32_t h = head.div(r), at = r - h * head.d;
        for (uint32_t j0 = w.job; j0 < 2 * per; j0 += kBatch * w.wpc) {
            ReadItem it[kBatch];
            int32_t slot[kBatch];
#pragma unroll
            for (uint32_t n = 0; n < kBatch; ++n) {
                const uint32_t j = j0 + n * w.wpc, t = t0 + (j >= per ? j - per : j);
                slot[n] = j < 2 * per && t < a.tokens ? a.slots[static_cast<int64_t>(t) * a.slots_st] : -1;
                if (slot[n] >= 0 && static_cast<uint64_t>(slot[n]) >= slots) slot[n] = -1;
            }
#pragma unroll
            for (uint32_t n = 0; n < kBatch; ++n) {
                if (slot[n] < 0) continue;
                const PagePool &pool = j0 + n * w.wpc >= per ? a.v_pool : a.k_pool;
                const uint32_t p = page.div(static_cast<uint32_t>(slot[n])), in = static_cast<uint32_t>(slot[n]) - p * page.d;
                it[n] = read_item<true>(pool, pool.data + p * pool.st_page + in * pool.st_tok + h * pool.st_head, blocks, at);
            }
#pragma unroll
            for (uint32_t n = 0; n < kBatch; ++n) {
                if (slot[n] < 0) continue;
                const uint32_t j = j0 + n * w.wpc, t = t0 + (j >= per ? j - per : j);
                const bool val = j >= per;
                const int64_t *st = val ? a.v_st : a.k_st;
                write_item<true>((val ? a.v_pool : a.k_pool).kind, it[n], (val ? a.v : a.k) + static_cast<int64_t>(t) * st[2] + h * st[1] + static_cast<int64_t>(8 * at) * st[0], st[0]);
            }
        }
    }
}

} // namespace

template <bool BF16, uint32_t T>
static void pa_append(const PagedAppendArgs &a, hipStream_t stream)
{
    const bool vec = a.dim % 8 == 0 && a.k_st[0] == 1 && a.v_st[0] == 1;
    const uint32_t head = vec ? a.dim / 8 : a.dim;
    const uint32_t grid = (a.tokens + T - 1) / T;
    const FastDiv page(a.page), per_head(head), per_token(head * a.kv_heads);
    if (vec) k_pa_append<BF16, T, true><<<grid, kBlock, 0, stream>>>(a, page, per_head, per_token);
    else k_pa_append<BF16, T, false><<<grid, kBlock, 0, stream>>>(a, page, per_head, per_token);
}

template <uint32_t T>
static void pk_append(const PagedAppendArgs &a, hipStream_t stream)
{
    const uint32_t head = a.dim / 8, grid = (a.tokens + T - 1) / T, items = head * a.kv_heads;
    const FastDiv page(a.page), per_head(head), per_token(items);
    // 8000 tokens in Q4_0: of 128 items 39.4 us for a write and a read of all with whole
    // waves, 53.6 without; of 64 25.2 and 32.1; of 32 the same, of 16 21.9 and 16.9
    if (items < kWave) k_pk_append<T><<<grid, kBlock, 0, stream>>>(a, page, per_head, per_token);
    else if (a.k_st[0] == 1 && a.v_st[0] == 1) k_pk_append_wide<T, true><<<grid, kBlock, 0, stream>>>(a, page, per_head, items);
    else k_pk_append_wide<T, false><<<grid, kBlock, 0, stream>>>(a, page, per_head, items);
}

hipError_t launch_paged_append(const PagedAppendArgs &a, hipStream_t stream)
{
    PagedAppendArgs b = a;
    for (uint64_t t = 0; t < a.tokens; t += kPaAppend) {
        b.tokens = static_cast<uint32_t>(a.tokens - t < kPaAppend ? a.tokens - t : kPaAppend);
        b.k = a.k + static_cast<int64_t>(t) * a.k_st[2];
        b.v = a.v + static_cast<int64_t>(t) * a.v_st[2];
        b.slots = a.slots + static_cast<int64_t>(t) * a.slots_st;
        const bool many = b.tokens >= 2048; // a workgroup per compute unit, of eight tokens
        if (b.k_pool.packed()) many ? pk_append<8>(b, stream) : pk_append<1>(b, stream);
        else if (b.k_pool.kind == PoolKind::Bf16) many ? pa_append<true, 8>(b, stream) : pa_append<true, 1>(b, stream);
        else many ? pa_append<false, 8>(b, stream) : pa_append<false, 1>(b, stream);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_paged_read(const PagedReadArgs &a, hipStream_t stream)
{
    const bool eight = a.dim % 8 == 0;
    const uint32_t head = eight ? a.dim / 8 : a.dim, items = head * a.kv_heads;
    const FastDiv page(a.page), per_head(head), per_token(items);
    PagedReadArgs b = a;
    for (uint64_t t = 0; t < a.tokens; t += kPaReadTokens) {
        b.tokens = static_cast<uint32_t>(a.tokens - t < kPaReadTokens ? a.tokens - t : kPaReadTokens);
        b.slots = a.slots + static_cast<int64_t>(t) * a.slots_st;
        b.k = a.k + static_cast<int64_t>(t) * a.k_st[2];
        b.v = a.v + static_cast<int64_t>(t) * a.v_st[2];
        const uint32_t per = a.tokens >= 2048 ? kPaRead : 1, grid = (b.tokens + per - 1) / per;
        if (eight && items >= kWave) k_pa_read_wide<<<grid, kBlock, 0, stream>>>(b, per, page, per_head, items);
        else if (eight) k_pa_read<true><<<grid, kBlock, 0, stream>>>(b, per, page, per_head, per_token);
        else k_pa_read<false><<<grid, kBlock, 0, stream>>>(b, per, page, per_head, per_token);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

namespace {

uint32_t pa_heads(const PagedAttnArgs &a) // of a row
{
    const uint32_t group = a.heads / a.kv_heads;
    return group < 16 ? group : 16;
}

PaPages pa_pages(const PagedAttnArgs &a)
{
    const PoolKind k = a.k_pool.kind, v = a.v_pool.kind;
    if (!a.k_pool.packed()) return k == PoolKind::Bf16 ? PaPages::Bf16 : PaPages::F16;
    if (k == PoolKind::Q8_0) return v == PoolKind::Q8_0 ? PaPages::Q8Q8 : PaPages::Q8Q4;
    return v == PoolKind::Q8_0 ? PaPages::Q4Q8 : PaPages::Q4Q4;
}

// Workgroups that run at once, by registers and LDS, and their LDS: more would
// wait for a second round with as large a run each.
struct PaGrid {
    uint32_t workgroups, few, side, lds;
};

// Packed rows side by side: as many as the rows and a die's workgroups divide by
// (64 sequences of 90 to 9000 tokens, a token's 8 heads in a row, 54.8 us, 72.9 with each
// row by itself; two of 40001 to 60001 tokens with 32 heads in Q8_0 212 us, 218 with
// 8 side by side, 269 with each by itself, in Q4_0 143, 156 and 211; pages of a head's
// tokens in a row the same within 3%).
uint32_t pa_side(const PagedAttnArgs &a, uint32_t workgroups)
{
    if (!a.k_pool.packed()) return 1;
    const uint64_t group = a.heads / a.kv_heads, rows = a.kv_heads * ((group + 15) / 16);
    uint32_t side = 1;
    while (side < 32 && rows % (2 * side) == 0 && workgroups % (2 * side * kDies) == 0) side *= 2;
    return side;
}

// Floats of a workspace slot.
uint32_t pa_slot(const PagedAttnArgs &a)
{
    return 2 * kPaLead + pa_heads(a) * a.dim;
}

PaGrid pa_grid(const PagedAttnArgs &a)
{
    static const uint32_t cus = [] {
        int dev = 0, n = 0;
        if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
            n = 256;
        return static_cast<uint32_t>(n);
    }();
    const uint32_t ks = (a.dim + 31) / 32, fixed = a.k_pool.packed() ? 4096 + ks * 1024 : 4096 + ks * 3 * 1024;
    const int fold = a.k_pool.packed() ? pa_fold(static_cast<int>(ks), a.heads / a.kv_heads) : 0;
    const uint32_t planes = fold ? (ks + fold - 1) / fold * 2 * (kWave + 1) * 4 : 0; // of score operands
    uint32_t per = pa_per_cu(static_cast<int>(ks), fold);
    for (;; --per) {
        const uint32_t side = pa_side(a, cus * per);
        const uint32_t joined = 4 * pa_heads(a) * (a.dim + 4), weights = (a.k_pool.packed() ? kPaLead : 0) + pa_heads(a) * (cus * per / side);
        uint32_t lds = 4 * (joined > weights ? joined : weights);
        if (lds < 4 * planes) lds = 4 * planes;
        if (per == 1 || per * (fixed + lds) <= 160 * 1024) return {cus * per, cus * (per < 2 ? per : 2), side, lds};
    }
}

template <PaPages PAGES>
hipError_t pa_launch(const PagedAttnArgs &a, const PaPlan &pl, uint32_t grid, uint32_t lds, hipStream_t stream)
{
    switch ((a.dim + 31) / 32) {
    case 1: k_pa_attn<PAGES, 1, 4><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 2: k_pa_attn<PAGES, 2, 4><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 3: k_pa_attn<PAGES, 3, 8><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 4: k_pa_attn<PAGES, 4, 8><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 5: k_pa_attn<PAGES, 5, 12><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 6: k_pa_attn<PAGES, 6, 12><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 7: k_pa_attn<PAGES, 7, 16><<<grid, kBlock, lds, stream>>>(a, pl); break;
    default: k_pa_attn<PAGES, 8, 16><<<grid, kBlock, lds, stream>>>(a, pl); break;
    }
    return hipGetLastError();
}

} // namespace

PagedScratch paged_attn_scratch(const PagedAttnArgs &a)
{
    const uint64_t n = pa_grid(a).workgroups;
    return {n * 2 * pa_slot(a) * sizeof(float), n * kPaLine * sizeof(uint32_t)};
}

uint32_t paged_attn_seqs(const PagedAttnArgs &a)
{
    const uint64_t group = a.heads / a.kv_heads, rows = a.kv_heads * ((group + 15) / 16);
    const uint64_t units = (static_cast<uint64_t>(a.max_pages) * a.page + kPaUnit - 1) / kPaUnit + 1;
    const uint64_t n = 0x7fff0000ull / rows / units; // both factors are below 2^32
    return static_cast<uint32_t>(n < a.seqs ? n : a.seqs);
}

hipError_t launch_paged_attn(const PagedAttnArgs &a, hipStream_t stream)
{
    PaPlan pl;
    pl.page = FastDiv(a.page);
    pl.dim = FastDiv(a.dim);
    pl.group = a.heads / a.kv_heads;
    pl.hgroups = FastDiv((pl.group + 15) / 16);
    pl.rows = a.kv_heads * pl.hgroups.d;
    const PaGrid grid = pa_grid(a);
    pl.side = grid.side;
    pl.grid = FastDiv(grid.workgroups / pl.side);
    pl.few = FastDiv(grid.few);
    pl.slot = pa_slot(a);
    pl.parts = static_cast<float *>(a.workspace);
    pl.arrived = static_cast<uint32_t *>(a.counters);
    // units are counted in 32 bits: a batch with more of them runs in parts
    PagedAttnArgs b = a;
    const uint32_t step = paged_attn_seqs(a);
    for (uint64_t s = 0; s < a.seqs; s += step) {
        b.seqs = static_cast<uint32_t>(a.seqs - s < step ? a.seqs - s : step);
        b.q = a.q + static_cast<int64_t>(s) * a.q_st[2];
        b.y = a.y + static_cast<int64_t>(s) * a.y_st[2];
        b.table = a.table + static_cast<int64_t>(s) * a.table_st[1];
        b.lengths = a.lengths + static_cast<int64_t>(s) * a.lengths_st;
        hipError_t e = hipSuccess;
        const uint32_t n = grid.workgroups, lds = grid.lds;
        switch (pa_pages(a)) {
        case PaPages::F16: e = pa_launch<PaPages::F16>(b, pl, n, lds, stream); break;
        case PaPages::Bf16: e = pa_launch<PaPages::Bf16>(b, pl, n, lds, stream); break;
        case PaPages::Q8Q8: e = packed_attn<PaPages::Q8Q8>(b, pl, n, lds, stream); break;
        case PaPages::Q8Q4: e = packed_attn<PaPages::Q8Q4>(b, pl, n, lds, stream); break;
        case PaPages::Q4Q8: e = packed_attn<PaPages::Q4Q8>(b, pl, n, lds, stream); break;
        case PaPages::Q4Q4: e = packed_attn<PaPages::Q4Q4>(b, pl, n, lds, stream); break;
        }
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

} // namespace emel
