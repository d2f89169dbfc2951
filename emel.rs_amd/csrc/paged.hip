// paged.hip -- the paged key-value cache: new tokens' keys and values rounded
// into their slots, and the attention of one new token per sequence over it.
#include "common.hpp"
#include "launch.hpp"

namespace emel {
namespace {

template <bool BF16>
__device__ __forceinline__ uint16_t to_half(float v)
{
    if constexpr (BF16) return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
    else return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}

template <bool BF16>
__device__ __forceinline__ float from_half(uint16_t h)
{
    if constexpr (BF16) return __builtin_bit_cast(float, static_cast<uint32_t>(h) << 16);
    else return static_cast<float>(__builtin_bit_cast(_Float16, h));
}

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

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef u4 u4_any __attribute__((aligned(2))); // pools may start at any half
typedef v4f v4f_any __attribute__((aligned(4)));

constexpr uint32_t kPaAppend = 1u << 17; // tokens of a launch

// dim: values of a head, in eights where VEC.
template <bool BF16, uint32_t T, bool VEC>
__global__ __launch_bounds__(kBlock) void k_pa_append(PagedAppendArgs a, FastDiv page, FastDiv head, FastDiv token)
{
    __shared__ uint32_t gone;
    const uint64_t slots = static_cast<uint64_t>(a.page) * a.pages;
    const uint32_t t0 = blockIdx.x * T;
    int32_t mine[T];
    uint32_t skip = 0;
    for (uint32_t i = 0; i < T; ++i) {
        mine[i] = t0 + i < a.tokens ? a.slots[static_cast<int64_t>(t0 + i) * a.slots_st] : -1;
        if (mine[i] < 0 || static_cast<uint64_t>(mine[i]) >= slots) skip |= 1u << i;
    }
    if (threadIdx.x == 0) gone = skip;
    __syncthreads();
    uint32_t later = 0;
#pragma unroll 4
    for (uint32_t u = t0 + 1 + threadIdx.x; u < a.tokens; u += kBlock) {
        const int32_t s = a.slots[static_cast<int64_t>(u) * a.slots_st];
        for (uint32_t i = 0; i < T; ++i) later |= s == mine[i] && u > t0 + i ? 1u << i : 0u;
    }
    if (later & ~skip) atomicOr(&gone, later);
    __syncthreads();
    const uint32_t drop = gone;
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

constexpr uint32_t kPaUnit = 128;  // tokens of a unit, 32 a wave
constexpr uint32_t kPaLine = 64;   // words between arrival counters (a cache line each)

// Workgroups that a compute unit holds at once: the registers that their
// launch bounds leave them.
constexpr uint32_t pa_per_cu(int ks) { return ks <= 2 ? 4 : ks <= 4 ? 3 : 2; }

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef u2 u2_any __attribute__((aligned(2)));

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

// What a launch derives on the host.
struct PaPlan {
    FastDiv page;       // tokens per page
    FastDiv dim, hgroups;
    FastDiv grid, few;  // workgroups: all, and two a compute unit
    uint32_t group;     // query heads of a cache head
    uint32_t rows;      // rows of a sequence: kv_heads * hgroups
    uint32_t slot;      // floats of a workspace slot
    float *parts;       // 2 slots a workgroup
    uint32_t *arrived;  // a counter per workgroup, zero between launches
};

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

// KS: 32-dim steps of a score; VW: dims of a lane's values (4, 8, 12 or 16).
template <bool BF16, int KS, int VW>
__global__ __launch_bounds__(kBlock, pa_per_cu(KS)) void k_pa_attn(PagedAttnArgs a, PaPlan pl)
{
    constexpr int P = kParts<BF16>;
    constexpr int kWaves = kBlock / kWave;
    constexpr float kLift = BF16 ? 0.0f : 14.0f;
    extern __shared__ __attribute__((aligned(16))) float joined[];            // [wave][head of the group][dim]
    __shared__ u4 qop[KS * P * kWave];           // score operands, lane after lane
    __shared__ int64_t off[kWaves][2][32];       // a step's tokens in the key and value pools
    __shared__ float wm[kWaves][16], wl[kWaves][16], jl[16];
    __shared__ uint32_t scan[kWaves], found[2];
    __shared__ uint32_t last;
    const uint32_t thread = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(thread / kWave);
    const uint32_t dim = a.dim, pitch = dim + 4; // of a head in joined

    // Rows of a few units are mostly set-up, which more workgroups hide; long
    // ones stream best with two a compute unit (64 sequences of 90 to 9000
    // tokens 106 us, 113 with three; 640 of 100 tokens 90 us, 77 with three).
    auto share_of = [&](uint32_t units) { return units > 4 * a.seqs ? pl.few : pl.grid; };
    // This workgroup's run of units, and the sequence it starts in.  A row's
    // set-up and end cost about a unit: it counts as one more, but where there
    // is no more than a unit to a workgroup (that would only part the rows).
    const uint32_t first_lane = thread % kWave;
    uint32_t total, run, cur, base; // base: the sequence's first unit
    uint32_t s, setup;
    int32_t s_len;
    if (__builtin_expect(a.seqs <= kWave, 1)) { // every wave for itself: a sequence per first_lane
        const int32_t len = first_lane < a.seqs ? pa_len(a, first_lane) : 0;
        const uint32_t mine = first_lane < a.seqs ? pa_seq(a, len).units : 0;
        uint32_t pre = wave_scan(mine);
        const uint32_t all = lane_u32(pre, kWave - 1);
        const FastDiv share = share_of(all);
        setup = all * pl.rows > share.d;
        total = (all + setup * a.seqs) * pl.rows;
        pre += setup * (first_lane + 1);
        run = share.div(total + share.d - 1);
        cur = blockIdx.x * run;
        if (cur >= total) return;
        s = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(__popcll(__ballot(first_lane < a.seqs && pre * pl.rows <= cur))));
        base = lane_u32(pre - mine - setup, s) * pl.rows;
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
        setup = all * pl.rows > share.d;
        pre += setup * s0 - mine;
        mine += setup * (s1 - s0);
        total = (all + setup * a.seqs) * pl.rows;
        run = share.div(total + share.d - 1);
        cur = blockIdx.x * run;
        if (cur >= total) return;
        if (mine && pre * pl.rows <= cur && cur < (pre + mine) * pl.rows) {
            uint32_t i = s0;
#pragma unroll 1
            for (uint32_t u = pa_seq(a, pa_len(a, i)).units + setup; (pre + u) * pl.rows <= cur; u = pa_seq(a, pa_len(a, i)).units + setup) {
                pre += u;
                ++i;
            }
            found[0] = i;
            found[1] = pre;
        }
        __syncthreads();
        s = found[0];
        base = found[1] * pl.rows;
        s_len = pa_len(a, s);
    }
    const uint32_t end = cur + run < total ? cur + run : total;

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
        const uint32_t n0 = cur - row_at, n1 = end - row_at < units ? end - row_at : units;
        const uint32_t u0 = n0 > setup ? n0 - setup : 0, u1 = n1 - setup;
        const uint32_t kh = pl.hgroups.div(row), h0 = kh * pl.group + (row - kh * pl.hgroups.d) * 16;
        const uint32_t heads = (kh + 1) * pl.group - h0 < 16 ? (kh + 1) * pl.group - h0 : 16;

        const uint16_t *kbase = a.k_pool.data + static_cast<int64_t>(kh) * a.k_pool.st_head;
        const uint16_t *vbase = a.v_pool.data + static_cast<int64_t>(kh) * a.v_pool.st_head;
        const int32_t *table = a.table + static_cast<int64_t>(s) * a.table_st[1];
        float m = -__builtin_inff(), l = 0.0f;
        v4f acc[VW];
        for (int j = 0; j < VW; ++j) acc[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        bool bad = sq.bad;

        const uint32_t t_end = sq.tokens < u1 * kPaUnit ? sq.tokens : u1 * kPaUnit;
        uint32_t t0 = u0 * kPaUnit + wave * 32;
        // the page of lane % 32's token, a step ahead of its use
        auto page_of = [&](uint32_t t) {
            return t < t_end ? table[static_cast<int64_t>(pl.page.div(sq.first + t)) * a.table_st[0]] : 0;
        };
        int32_t next = page_of(t0 + lane % 32);

        // score operands, lane (col, g): dims 32 e + 8 g .. + 7 of head col;
        // each wave lays out every fourth e
        float inv = 1.0f;
        {
            const float *q = a.q + static_cast<int64_t>(h0 + col) * a.q_st[1] + static_cast<int64_t>(s) * a.q_st[2];
            const float c = a.soft_cap > 0.0f ? a.scale / a.soft_cap : a.scale * 1.44269504088896340736f;
            auto eight = [&](uint32_t e, float x[8]) {
                const uint32_t d = 32 * e + 8 * g;
                if (col < heads && d < dim) {
                    if (__builtin_expect(a.q_st[0] == 1, 1)) {
                        const v4f lo = *reinterpret_cast<const v4f_any *>(q + d), hi = *reinterpret_cast<const v4f_any *>(q + d + 4);
                        for (int i = 0; i < 4; ++i) {
                            x[i] = lo[i] * c;
                            x[4 + i] = hi[i] * c;
                        }
                    } else {
                        for (int i = 0; i < 8; ++i) x[i] = q[static_cast<int64_t>(d + i) * a.q_st[0]] * c;
                    }
                } else {
                    for (int i = 0; i < 8; ++i) x[i] = 0.0f;
                }
            };
            float up = 1.0f;
            if constexpr (!BF16) { // the head's largest value to [2^14, 2^15)
                float top = 0.0f;
                auto fold = [&](const float x[8]) {
                    for (int i = 0; i < 8; ++i) top = __builtin_fmaxf(top, __builtin_fabsf(x[i]));
                };
                if constexpr (KS <= 4) { // all loads at once
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
                int e = static_cast<int>((__builtin_bit_cast(uint32_t, top) >> 23) & 255u) - 127;
                e = top == 0.0f || e == 128 ? 0 : e < -110 ? -110 : e; // infinite: the wave walks below
                up = __builtin_bit_cast(float, static_cast<uint32_t>(127 + 14 - e) << 23);
                inv = __builtin_bit_cast(float, static_cast<uint32_t>(127 - 14 + e) << 23);
            }
#pragma unroll 1
            for (uint32_t e = wave; e < KS; e += kWaves) {
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
        for (; t0 < t_end; t0 += kPaUnit) {
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

        // the wave's part: [head][dim], dims of lane row c = 4 g + i
        float *own = joined + wave * heads * pitch;
        l = rows16(l, [](float x, float y) { return x + y; });
        v4f size = {l, 0.0f, 0.0f, 0.0f};
        for (int j = 0; j < VW; ++j)
            for (int i = 0; i < 4; ++i) size[i] += __builtin_fabsf(acc[j][i]);
        const bool odd = !((size[0] + size[1]) + (size[2] + size[3]) < (BF16 ? 0x1p97f : __builtin_inff()));
        bad = __any(bad);
        if (__builtin_expect(__any(odd && col < heads) && !bad, 0)) {
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
                        for (uint32_t i = 0; i < 4; ++i)
                            if (4 * lane + i < dim) zz += qv[i] * from_half<BF16>(kp[4 * lane + i]);
                        zz = wave_sum(zz) * a.scale;
                        if (a.soft_cap > 0.0f) zz = a.soft_cap * pa_tanh(zz / a.soft_cap);
                        zz *= 1.44269504088896340736f;
                        const float m1 = __builtin_fmaxf(mm, zz);
                        const float ref = m1 == -__builtin_inff() ? 0.0f : m1;
                        const float f = m1 > mm ? __builtin_amdgcn_exp2f(mm - m1) : 1.0f;
                        const float e = __builtin_amdgcn_exp2f(zz - ref);
                        ll = ll * f + e;
                        for (uint32_t i = 0; i < 4; ++i)
                            if (4 * lane + i < dim) av[i] = av[i] * f + e * (from_half<BF16>(vp[4 * lane + i]) * down);
                        mm = m1;
                    }
                }
                const float lift = BF16 ? 1.0f : 16384.0f; // as the parts of waves that do not walk
                for (uint32_t i = 0; i < 4; ++i)
                    if (4 * lane + i < dim) own[h * pitch + 4 * lane + i] = av[i] * lift;
                if (lane == 0) {
                    wm[wave][h] = mm + above;
                    wl[wave][h] = ll * (lift * down);
                }
            }
        } else if (col < heads) {
            if (g == 0) {
                wm[wave][col] = m;
                wl[wave][col] = bad ? __builtin_nanf("") : l;
            }
            for (int i = 0; i < 4; ++i) {
                const uint32_t c = 4 * g + i;
                for (int e = 0; e < VW / 8; ++e)
                    if (128 * e + 8 * c < dim)
                        for (int j = 0; j < 8; j += 4)
                            *reinterpret_cast<v4f *>(own + col * pitch + 128 * e + 8 * c + j) =
                                v4f{acc[8 * e + j][i], acc[8 * e + j + 1][i], acc[8 * e + j + 2][i], acc[8 * e + j + 3][i]};
                if constexpr (VW % 8) {
                    const uint32_t d = VW / 8 * 128 + 4 * c;
                    if (d < dim)
                        *reinterpret_cast<v4f *>(own + col * pitch + d) = v4f{acc[VW - 4][i], acc[VW - 3][i], acc[VW - 2][i], acc[VW - 1][i]};
                }
            }
        }
        __syncthreads();
        const bool whole = n0 == 0 && n1 == units;
        const uint32_t w0 = n0 == 0 ? blockIdx.x : row_at / run; // the row's first workgroup
        float *slot = pl.parts + static_cast<size_t>(2 * blockIdx.x + (n0 == 0 ? 1 : 0)) * pl.slot;
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
        if (++row == pl.rows && cur < end) {
            row = 0;
            sq = pa_seq(a, pa_len(a, ++s));
            units = sq.units + setup;
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

hipError_t launch_paged_append(const PagedAppendArgs &a, hipStream_t stream)
{
    PagedAppendArgs b = a;
    for (uint64_t t = 0; t < a.tokens; t += kPaAppend) {
        b.tokens = static_cast<uint32_t>(a.tokens - t < kPaAppend ? a.tokens - t : kPaAppend);
        b.k = a.k + static_cast<int64_t>(t) * a.k_st[2];
        b.v = a.v + static_cast<int64_t>(t) * a.v_st[2];
        b.slots = a.slots + static_cast<int64_t>(t) * a.slots_st;
        const bool many = b.tokens >= 2048; // a workgroup per compute unit, of eight tokens
        if (b.bf16) many ? pa_append<true, 8>(b, stream) : pa_append<true, 1>(b, stream);
        else many ? pa_append<false, 8>(b, stream) : pa_append<false, 1>(b, stream);
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

// Workgroups that run at once, by registers and LDS, and their LDS: more would
// wait for a second round with as large a run each.
struct PaGrid {
    uint32_t workgroups, few, lds;
};
PaGrid pa_grid(const PagedAttnArgs &a)
{
    static const uint32_t cus = [] {
        int dev = 0, n = 0;
        if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
            n = 256;
        return static_cast<uint32_t>(n);
    }();
    const uint32_t ks = (a.dim + 31) / 32, fixed = 4096 + ks * 3 * 1024;
    uint32_t per = pa_per_cu(static_cast<int>(ks));
    for (;; --per) {
        const uint32_t joined = 4 * pa_heads(a) * (a.dim + 4), weights = pa_heads(a) * cus * per;
        const uint32_t lds = 4 * (joined > weights ? joined : weights);
        if (per == 1 || per * (fixed + lds) <= 160 * 1024) return {cus * per, cus * (per < 2 ? per : 2), lds};
    }
}

template <bool BF16>
hipError_t pa_launch(const PagedAttnArgs &a, const PaPlan &pl, hipStream_t stream)
{
    const PaGrid g = pa_grid(a);
    const uint32_t grid = g.workgroups, lds = g.lds;
    switch ((a.dim + 31) / 32) {
    case 1: k_pa_attn<BF16, 1, 4><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 2: k_pa_attn<BF16, 2, 4><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 3: k_pa_attn<BF16, 3, 8><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 4: k_pa_attn<BF16, 4, 8><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 5: k_pa_attn<BF16, 5, 12><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 6: k_pa_attn<BF16, 6, 12><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 7: k_pa_attn<BF16, 7, 16><<<grid, kBlock, lds, stream>>>(a, pl); break;
    default: k_pa_attn<BF16, 8, 16><<<grid, kBlock, lds, stream>>>(a, pl); break;
    }
    return hipGetLastError();
}

} // namespace

PagedScratch paged_attn_scratch(const PagedAttnArgs &a)
{
    const uint64_t n = pa_grid(a).workgroups;
    return {n * 2 * (32 + static_cast<uint64_t>(pa_heads(a)) * a.dim) * sizeof(float), n * kPaLine * sizeof(uint32_t)};
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
    pl.grid = FastDiv(grid.workgroups);
    pl.few = FastDiv(grid.few);
    pl.slot = 32 + pa_heads(a) * a.dim;
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
        const hipError_t e = b.bf16 ? pa_launch<true>(b, pl, stream) : pa_launch<false>(b, pl, stream);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

} // namespace emel
