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

// A workgroup per token.  Of tokens with one slot the last is stored: a
// workgroup whose slot a later token names leaves it to that one.
template <bool BF16>
__global__ __launch_bounds__(kBlock) void k_pa_append(PagedAppendArgs a)
{
    const uint64_t slots = static_cast<uint64_t>(a.page) * a.pages;
    const uint32_t per = a.dim * a.kv_heads;
    for (uint32_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
        const int32_t slot = a.slots[static_cast<int64_t>(t) * a.slots_st];
        if (slot < 0 || static_cast<uint64_t>(slot) >= slots) continue;
        bool later = false;
        for (uint32_t u = t + 1 + threadIdx.x; u < a.tokens; u += kBlock)
            later |= a.slots[static_cast<int64_t>(u) * a.slots_st] == slot;
        if (__syncthreads_or(later)) continue;
        const uint32_t p = static_cast<uint32_t>(slot) / a.page, i = static_cast<uint32_t>(slot) % a.page;
        for (uint32_t e = threadIdx.x; e < per; e += kBlock) {
            const int64_t h = e / a.dim, d = e % a.dim;
            a.k_pool.data[p * a.k_pool.st_page + h * a.k_pool.st_head + i * a.k_pool.st_tok + d] =
                to_half<BF16>(a.k[d * a.k_st[0] + h * a.k_st[1] + t * a.k_st[2]]);
            a.v_pool.data[p * a.v_pool.st_page + h * a.v_pool.st_head + i * a.v_pool.st_tok + d] =
                to_half<BF16>(a.v[d * a.v_st[0] + h * a.v_st[1] + t * a.v_st[2]]);
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
// The weights P go in as halves that add up to f32's 24 bits for bf16, 22 for
// f16 (hi + lo, scaled by 2^14 so that lo stays normal down to 2^-28 of the largest).
// A wave's (m, l, out) are joined through LDS, a row's segments of several
// workgroups through the workspace by the last of them to finish: stores and
// loads at agent scope and an arrival counter, as in reduce.hip.  The order
// of every sum depends on the lengths alone.
//
// Splitting a factor into parts breaks 0 * inf and inf - inf.  A wave whose
// results are not all finite walks its tokens again one by one in f32, as the
// formula stands, and takes those.

constexpr uint32_t kPaUnit = 128;  // tokens of a unit, 32 a wave
constexpr uint32_t kPaLine = 64;   // words between arrival counters (a cache line each)
constexpr uint32_t kPaPerCu = 3;   // workgroups per compute unit

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
// pools may start at any half
typedef u4 u4_any __attribute__((aligned(2)));
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

// What a launch derives on the host.
struct PaPlan {
    FastDiv page;       // tokens per page
    uint32_t group;     // query heads of a cache head
    uint32_t hgroups;   // 16s of them
    uint32_t rows;      // rows of a sequence: kv_heads * hgroups
    uint32_t slot;      // floats of a workspace slot
    float *parts;       // 2 slots a workgroup
    uint32_t *arrived;  // a counter per workgroup, zero between launches
};

struct PaSeq {
    uint32_t first, tokens, units;
    bool bad;
};

__device__ __forceinline__ PaSeq pa_seq(const PagedAttnArgs &a, uint32_t s)
{
    const int32_t len = a.lengths[static_cast<int64_t>(s) * a.lengths_st];
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

// 2^(m - ref) of a part whose maximum is m, in a whole whose maximum is ref.
__device__ __forceinline__ float pa_weight(float m, float ref)
{
    return __builtin_amdgcn_exp2f(m - (ref == -__builtin_inff() ? 0.0f : ref));
}

// KS: 32-dim steps of a score; VW: dims of a lane's values (4, 8, 12 or 16).
template <bool BF16, int KS, int VW>
__global__ __launch_bounds__(kBlock) void k_pa_attn(PagedAttnArgs a, PaPlan pl)
{
    constexpr int P = kParts<BF16>;
    constexpr int kWaves = kBlock / kWave;
    constexpr float kLift = BF16 ? 0.0f : 14.0f;
    extern __shared__ float joined[];            // [wave][head of the group][dim]
    __shared__ u4 qop[KS * P * kWave];           // score operands, lane after lane
    __shared__ float qinv[16];
    __shared__ int64_t off[kWaves][2][32];       // a step's tokens in the key and value pools
    __shared__ float wm[kWaves][16], wl[kWaves][16], jm[16], jl[16];
    __shared__ uint64_t scan[kWaves], found[2];
    __shared__ uint32_t last;
    const uint32_t tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const uint32_t col = lane % 16, g = lane / 16;
    const uint32_t dim = a.dim;

    // this workgroup's run of units, and the sequence it starts in
    const uint32_t per = (a.seqs + kBlock - 1) / kBlock;
    const uint32_t s0 = tid * per < a.seqs ? tid * per : a.seqs, s1 = s0 + per < a.seqs ? s0 + per : a.seqs;
    uint64_t mine = 0;
    for (uint32_t s = s0; s < s1; ++s) mine += pa_seq(a, s).units;
    uint64_t pre = mine;
    for (int d = 1; d < kWave; d <<= 1) {
        const uint64_t up = __shfl_up(pre, d, kWave);
        if (lane >= static_cast<uint32_t>(d)) pre += up;
    }
    if (lane == kWave - 1) scan[wave] = pre;
    __syncthreads();
    uint64_t all = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (static_cast<uint32_t>(w) < wave) pre += scan[w];
        all += scan[w];
    }
    pre -= mine;
    const uint64_t total = all * pl.rows;
    const uint64_t run = (total + gridDim.x - 1) / gridDim.x;
    uint64_t cur = blockIdx.x * run;
    if (cur >= total) return;
    const uint64_t end = cur + run < total ? cur + run : total;
    if (mine && pre * pl.rows <= cur && cur < (pre + mine) * pl.rows) {
        uint32_t s = s0;
        uint64_t at = pre;
        for (uint32_t u = pa_seq(a, s).units; (at + u) * pl.rows <= cur; u = pa_seq(a, s).units) {
            at += u;
            ++s;
        }
        found[0] = s;
        found[1] = at;
    }
    __syncthreads();
    uint32_t s = static_cast<uint32_t>(found[0]);
    uint64_t base = found[1] * pl.rows; // the sequence's first unit

    while (cur < end) {
        const PaSeq sq = pa_seq(a, s);
        const uint32_t row = static_cast<uint32_t>((cur - base) / sq.units);
        const uint64_t row_at = base + static_cast<uint64_t>(row) * sq.units;
        const uint32_t u0 = static_cast<uint32_t>(cur - row_at);
        const uint32_t u1 = end - row_at < sq.units ? static_cast<uint32_t>(end - row_at) : sq.units;
        const uint32_t kh = row / pl.hgroups, h0 = kh * pl.group + (row % pl.hgroups) * 16;
        const uint32_t heads = (kh + 1) * pl.group - h0 < 16 ? (kh + 1) * pl.group - h0 : 16;

        // score operands: thread (head, i) takes dims i, i + 16, ... of its head
        {
            const uint32_t h = tid / 16, i = tid % 16;
            const float *q = a.q + static_cast<int64_t>(h0 + h) * a.q_st[1] + static_cast<int64_t>(s) * a.q_st[2];
            const float c = a.soft_cap > 0.0f ? a.scale / a.soft_cap : a.scale * 1.44269504088896340736f;
            float v[2 * KS], top = 0.0f;
            for (int e = 0; e < 2 * KS; ++e) {
                const uint32_t d = 16 * e + i;
                v[e] = h < heads && d < dim ? q[static_cast<int64_t>(d) * a.q_st[0]] * c : 0.0f;
                const float m = __builtin_fabsf(v[e]);
                top = m > top && m < __builtin_inff() ? m : top;
            }
            float up = 1.0f;
            if constexpr (!BF16) {
                for (int d = 8; d > 0; d >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, d, 16));
                int e = static_cast<int>((__builtin_bit_cast(uint32_t, top) >> 23) & 255u) - 127;
                e = top == 0.0f ? 0 : e < -110 ? -110 : e;
                up = __builtin_bit_cast(float, static_cast<uint32_t>(127 + 14 - e) << 23);
                if (i == 0) qinv[h] = __builtin_bit_cast(float, static_cast<uint32_t>(127 - 14 + e) << 23);
            }
            uint16_t *halves = reinterpret_cast<uint16_t *>(qop);
            for (int e = 0; e < 2 * KS; ++e) {
                const uint32_t d = 16 * e + i;
                uint32_t part[3];
                split<BF16>(v[e] * up, part);
                for (int p = 0; p < P; ++p)
                    halves[(((d / 32) * P + p) * kWave + (d % 32) / 8 * 16 + h) * 8 + d % 8] = static_cast<uint16_t>(part[p]);
            }
        }
        __syncthreads();

        const uint16_t *kbase = a.k_pool.data + static_cast<int64_t>(kh) * a.k_pool.st_head;
        const uint16_t *vbase = a.v_pool.data + static_cast<int64_t>(kh) * a.v_pool.st_head;
        const int32_t *table = a.table + static_cast<int64_t>(s) * a.table_st[1];
        const float inv = BF16 ? 1.0f : qinv[col];
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
            if (a.soft_cap > 0.0f)
                for (int i = 0; i < 8; ++i) z[i] = tanhf(z[i]) * (a.soft_cap * 1.44269504088896340736f);
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
        float *own = joined + static_cast<size_t>(wave) * heads * dim;
        l = rows16(l, [](float x, float y) { return x + y; });
        bool odd = !(__builtin_fabsf(l) < __builtin_inff());
        for (int j = 0; j < VW; ++j)
            for (int i = 0; i < 4; ++i) odd |= !(__builtin_fabsf(acc[j][i]) < __builtin_inff());
        bad = __any(bad);
        if (__any(odd && col < heads) && !bad) {
            // as the formula stands: a head and a token at a time, a lane four dims
            for (uint32_t h = 0; h < heads; ++h) {
                const float *q = a.q + static_cast<int64_t>(h0 + h) * a.q_st[1] + static_cast<int64_t>(s) * a.q_st[2];
                float qv[4], av[4] = {}, mm = -__builtin_inff(), ll = 0.0f;
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t d = 4 * lane + i;
                    qv[i] = d < dim ? q[static_cast<int64_t>(d) * a.q_st[0]] : 0.0f;
                }
                for (uint32_t t1 = u0 * kPaUnit + wave * 32; t1 < t_end; t1 += kPaUnit) {
                    for (uint32_t t = t1; t < t1 + 32 && t < t_end; ++t) {
                        const int64_t p = table[static_cast<int64_t>(pl.page.div(sq.first + t)) * a.table_st[0]];
                        const int64_t i0 = pl.page.mod(sq.first + t);
                        const uint16_t *kp = kbase + p * a.k_pool.st_page + i0 * a.k_pool.st_tok;
                        const uint16_t *vp = vbase + p * a.v_pool.st_page + i0 * a.v_pool.st_tok;
                        float zz = 0.0f;
                        for (uint32_t i = 0; i < 4; ++i)
                            if (4 * lane + i < dim) zz += qv[i] * from_half<BF16>(kp[4 * lane + i]);
                        zz = wave_sum(zz) * a.scale;
                        if (a.soft_cap > 0.0f) zz = a.soft_cap * tanhf(zz / a.soft_cap);
                        zz *= 1.44269504088896340736f;
                        const float m1 = __builtin_fmaxf(mm, zz);
                        const float ref = m1 == -__builtin_inff() ? 0.0f : m1;
                        const float f = m1 > mm ? __builtin_amdgcn_exp2f(mm - m1) : 1.0f;
                        const float e = __builtin_amdgcn_exp2f(zz - ref);
                        ll = ll * f + e;
                        for (uint32_t i = 0; i < 4; ++i)
                            if (4 * lane + i < dim) av[i] = av[i] * f + e * from_half<BF16>(vp[4 * lane + i]);
                        mm = m1;
                    }
                }
                const float lift = BF16 ? 1.0f : 16384.0f;
                for (uint32_t i = 0; i < 4; ++i)
                    if (4 * lane + i < dim) own[h * dim + 4 * lane + i] = av[i] * lift;
                if (lane == 0) {
                    wm[wave][h] = mm;
                    wl[wave][h] = ll * lift;
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
                        for (int j = 0; j < 8; ++j) own[col * dim + 128 * e + 8 * c + j] = acc[8 * e + j][i];
                if constexpr (VW % 8) {
                    const uint32_t d = VW / 8 * 128 + 4 * c;
                    if (d < dim)
                        for (int j = 0; j < 4; ++j) own[col * dim + d + j] = acc[VW - 4 + j][i];
                }
            }
        }
        __syncthreads();
        if (tid < heads) {
            float top = wm[0][tid], sum = 0.0f;
            for (int w = 1; w < kWaves; ++w) top = __builtin_fmaxf(top, wm[w][tid]);
            for (int w = 0; w < kWaves; ++w) sum += wl[w][tid] * pa_weight(wm[w][tid], top);
            jm[tid] = top;
            jl[tid] = sum;
        }
        __syncthreads();
        const bool whole = u0 == 0 && u1 == sq.units;
        const uint32_t w0 = static_cast<uint32_t>(row_at / run); // the row's first workgroup
        float *slot = pl.parts + static_cast<size_t>(2 * blockIdx.x + (blockIdx.x == w0 ? 1 : 0)) * pl.slot;
        const uint32_t cells = heads * dim;
        for (uint32_t e = tid; e < cells; e += kBlock) {
            const uint32_t h = e / dim, d = e % dim;
            float v = 0.0f;
            for (int w = 0; w < kWaves; ++w)
                v += joined[static_cast<size_t>(w) * cells + e] * pa_weight(wm[w][h], jm[h]);
            if (whole)
                a.y[static_cast<int64_t>(d) * a.y_st[0] + static_cast<int64_t>(h0 + h) * a.y_st[1] + static_cast<int64_t>(s) * a.y_st[2]] =
                    sq.tokens == 0 && !sq.bad ? 0.0f : v / jl[h];
            else
                pa_store(slot + 32 + e, v);
        }
        if (!whole) {
            if (tid < heads) {
                pa_store(slot + tid, jm[tid]);
                pa_store(slot + 16 + tid, jl[tid]);
            }
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            const uint32_t w1 = static_cast<uint32_t>((row_at + sq.units - 1) / run), pieces = w1 - w0 + 1;
            if (tid == 0) {
                uint32_t *arrived = pl.arrived + static_cast<size_t>(w0) * kPaLine;
                last = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == pieces - 1;
                if (last) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (last) {
                auto piece = [&](uint32_t p) { return pl.parts + static_cast<size_t>(2 * (w0 + p) + (p == 0 ? 1 : 0)) * pl.slot; };
                if (tid / 16 < heads) { // 16 threads a head
                    const uint32_t h = tid / 16;
                    float top = -__builtin_inff(), sum = 0.0f;
                    for (uint32_t p = tid % 16; p < pieces; p += 16) top = __builtin_fmaxf(top, pa_load(piece(p) + h));
                    for (int d = 8; d > 0; d >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, d, 16));
                    for (uint32_t p = tid % 16; p < pieces; p += 16) sum += pa_load(piece(p) + 16 + h) * pa_weight(pa_load(piece(p) + h), top);
                    for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 16);
                    if (tid % 16 == 0) {
                        jm[h] = top;
                        jl[h] = sum;
                    }
                }
                __syncthreads();
                for (uint32_t e = tid; e < cells; e += kBlock) {
                    const uint32_t h = e / dim, d = e % dim;
                    float v = 0.0f;
#pragma unroll 4
                    for (uint32_t p = 0; p < pieces; ++p) v += pa_load(piece(p) + 32 + e) * pa_weight(pa_load(piece(p) + h), jm[h]);
                    a.y[static_cast<int64_t>(d) * a.y_st[0] + static_cast<int64_t>(h0 + h) * a.y_st[1] + static_cast<int64_t>(s) * a.y_st[2]] = v / jl[h];
                }
            }
        }
        __syncthreads(); // the next segment reuses the shared arrays
        cur = row_at + u1;
        if (u1 == sq.units && row + 1 == pl.rows) {
            ++s;
            base += static_cast<uint64_t>(sq.units) * pl.rows;
        }
    }
}

} // namespace

hipError_t launch_paged_append(const PagedAppendArgs &a, hipStream_t stream)
{
    const uint32_t grid = a.tokens < (1u << 20) ? a.tokens : 1u << 20;
    if (a.bf16) k_pa_append<true><<<grid, kBlock, 0, stream>>>(a);
    else k_pa_append<false><<<grid, kBlock, 0, stream>>>(a);
    return hipGetLastError();
}

namespace {

uint32_t pa_workgroups()
{
    static const uint32_t n = [] {
        int dev = 0, cus = 0;
        if (hipGetDevice(&dev) != hipSuccess ||
            hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
            cus = 256;
        return static_cast<uint32_t>(cus) * kPaPerCu;
    }();
    return n;
}

uint32_t pa_heads(const PagedAttnArgs &a) // of a row
{
    const uint32_t group = a.heads / a.kv_heads;
    return group < 16 ? group : 16;
}

template <bool BF16>
hipError_t pa_launch(const PagedAttnArgs &a, const PaPlan &pl, hipStream_t stream)
{
    const uint32_t lds = 4 * pa_heads(a) * a.dim * sizeof(float);
    const dim3 grid(pa_workgroups());
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
    const uint64_t n = pa_workgroups();
    return {n * 2 * (32 + static_cast<uint64_t>(pa_heads(a)) * a.dim) * sizeof(float), n * kPaLine * sizeof(uint32_t)};
}

hipError_t launch_paged_attn(const PagedAttnArgs &a, hipStream_t stream)
{
    PaPlan pl;
    pl.page = FastDiv(a.page);
    pl.group = a.heads / a.kv_heads;
    pl.hgroups = (pl.group + 15) / 16;
    pl.rows = a.kv_heads * pl.hgroups;
    pl.slot = 32 + pa_heads(a) * a.dim;
    pl.parts = static_cast<float *>(a.workspace);
    pl.arrived = static_cast<uint32_t *>(a.counters);
    return a.bf16 ? pa_launch<true>(a, pl, stream) : pa_launch<false>(a, pl, stream);
}

} // namespace emel
