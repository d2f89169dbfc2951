// logits.hip -- penalties for repeated tokens, biases and a token mask on
// rows of logits, ahead of the sampler.
//
// Bound by one read and one write of the logits; what goes with them is
// sparse.  A workgroup takes a run of 4096 tokens of one row, 16 a
// thread, whose logits it loads first, or of 1024, 4 a thread, where all
// of those run at once: up to kLaFew logits, what counts is the chain of a run's
// loads, and shorter runs clear and walk fewer cells (one row of 151936 4.1 us
// against 5.8, eight 7.2 against 9.3, sixteen 10.9 against 10.1).  While they are on their way it counts
// the row's history ids that fall in its run, and the last bias entry of each
// token there, in LDS (integer atomics: the result does not depend on their
// order), then passes over the run once.  Both fit one word a token where there
// are fewer than 2^16 of either, which leaves a compute unit eight workgroups
// instead of four (64 rows of 151936 with a history of 2048 and a mask: 21.0 us, 3.8 TB/s, against 27.2).  Each of a row's runs reads the whole
// history and all its biases: a few KB from the L2 for 4 or 16 KB of logits.  That
// is made for the histories of a penalty's window; the walk sets the time of
// longer ones: one row of 151936 4.4 us with 2048 ids, 12 with 16384, 40 with
// 65535, 73 with 131072; 64 rows 19, 56 and 182 with the first three.  Runs
// start at 16-byte boundaries of the output, wherever its rows start.
#include "common.hpp"
#include "launch.hpp"

namespace emel {
namespace {

constexpr uint64_t kLaFew = 1u << 21; // 1024 tokens for each of eight workgroups on 256 compute units
constexpr uint32_t la_tokens(uint32_t quads) { return quads * 4 * kBlock; }

__device__ __forceinline__ float row_value(const RowTable &t, uint32_t row, float none)
{
    return t.data ? static_cast<const float *>(t.data)[row * t.row_st] : none;
}

// PACKED: count in the low half of a word, entry in the high half.
// VEC: both rows have unit stride and the same place in a 16-byte line.
// INPLACE: only tokens that change are read and written.
// Q: float4 a thread.
template <uint32_t Q, bool PACKED, bool VEC, bool INPLACE>
__global__ __launch_bounds__(kBlock) void k_la_adjust(LogitsAdjustArgs a, uint32_t runs, uint64_t items)
{
    constexpr uint32_t kLaTokens = la_tokens(Q);
    __shared__ __attribute__((aligned(16))) uint32_t count[kLaTokens];
    __shared__ __attribute__((aligned(16))) uint32_t entry[PACKED ? 4 : kLaTokens]; // 1 + the last bias entry
    __shared__ uint32_t words[kLaTokens / 32 + 2];
    const uint32_t tid = threadIdx.x;
    for (uint64_t it = blockIdx.x; it < items; it += gridDim.x) {
        const uint32_t row = static_cast<uint32_t>(it / runs);
        const float *x = a.x + row * a.x_row;
        float *y = a.y + row * a.y_row;
        const int64_t shift = VEC ? (reinterpret_cast<uintptr_t>(y) / 4) % 4 : 0;
        const int64_t t0 = static_cast<int64_t>(it % runs) * kLaTokens - shift, card = a.card; // t0 + i is token of cell i
        if (t0 >= card) continue; // a run that only other rows have
        float4 v[Q];
        auto cell = [&](uint32_t q) { return 4 * (tid + q * kBlock); };
        auto whole = [&](uint32_t q) { return t0 + cell(q) >= 0 && t0 + cell(q) + 3 < card; };
        if constexpr (VEC && !INPLACE) {
#pragma unroll
            for (uint32_t q = 0; q < Q; ++q)
                if (whole(q)) v[q] = ld_nt(reinterpret_cast<const float4 *>(x + t0 + cell(q)));
        }
        __syncthreads(); // the cells of the run before
        const uint4 none = make_uint4(0, 0, 0, 0);
        for (uint32_t q = 0; q < Q; ++q) {
            *reinterpret_cast<uint4 *>(count + cell(q)) = none;
            if constexpr (!PACKED) *reinterpret_cast<uint4 *>(entry + cell(q)) = none;
        }
        const int64_t w0 = t0 < 0 ? 0 : t0 / 32; // the mask's first word of the run
        if (a.allowed.data && tid < kLaTokens / 32 + 2 && w0 + tid < a.allowed.entries)
            words[tid] = static_cast<const uint32_t *>(a.allowed.data)[row * a.allowed.row_st + (w0 + tid) * a.allowed.st];
        __syncthreads();
        // ids of other runs, of no token and below zero are all outside [t0, t0 + kLaTokens) or past its live cells
        auto place = [&](int32_t id) {
            const int64_t i = static_cast<int64_t>(id) - t0;
            return id >= 0 && id < card && i >= 0 && i < static_cast<int64_t>(kLaTokens) ? static_cast<uint32_t>(i) : ~0u;
        };
        if (a.bias.data) {
            const int32_t *ids = static_cast<const int32_t *>(a.bias_ids.data) + row * a.bias_ids.row_st;
            for (uint32_t i = tid; i < a.bias.entries; i += kBlock) {
                const uint32_t p = place(ids[i * a.bias_ids.st]);
                if (p != ~0u) atomicMax(PACKED ? &count[p] : &entry[p], (i + 1) << (PACKED ? 16 : 0));
            }
            if constexpr (PACKED) __syncthreads(); // entries are in before counts are added to their words
        }
        if (a.history.data) {
            int64_t len = a.history.entries;
            if (a.history_len.data) {
                const int64_t n = static_cast<const int32_t *>(a.history_len.data)[row * a.history_len.row_st];
                len = n < 0 ? 0 : n < len ? n : len;
            }
            const int32_t *ids = static_cast<const int32_t *>(a.history.data) + row * a.history.row_st;
#pragma unroll 4
            for (int64_t i = tid; i < len; i += kBlock) {
                const uint32_t p = place(ids[i * a.history.st]);
                if (p != ~0u) atomicAdd(&count[p], 1u);
            }
        }
        __syncthreads();
        const float repeat = row_value(a.repeat, row, 1.0f);
        const float frequency = row_value(a.frequency, row, 0.0f);
        const float presence = row_value(a.presence, row, 0.0f);
        auto adjust = [&](float l, uint32_t c, uint32_t e, bool masked) {
            if (c) {
                l = l > 0.0f ? l / repeat : l * repeat;
                l = (l - static_cast<float>(c) * frequency) - presence;
            }
            if (e) l += static_cast<const float *>(a.bias.data)[(e - 1) * a.bias.st + row * a.bias.row_st];
            return masked ? -__builtin_inff() : l;
        };
        auto masked_at = [&](int64_t t) { return a.allowed.data && !((words[t / 32 - w0] >> (t % 32)) & 1u); };
#pragma unroll
        for (uint32_t q = 0; q < Q; ++q) {
            const uint32_t i = cell(q);
            const int64_t t = t0 + i;
            uint4 c = *reinterpret_cast<const uint4 *>(count + i), e;
            if constexpr (PACKED) {
                e = make_uint4(c.x >> 16, c.y >> 16, c.z >> 16, c.w >> 16);
                c = make_uint4(c.x & 0xffffu, c.y & 0xffffu, c.z & 0xffffu, c.w & 0xffffu);
            } else {
                e = *reinterpret_cast<const uint4 *>(entry + i);
            }
            if (VEC && whole(q)) {
                const bool m0 = masked_at(t), m1 = masked_at(t + 1), m2 = masked_at(t + 2), m3 = masked_at(t + 3);
                if constexpr (INPLACE) {
                    const bool touched = (c.x | c.y | c.z | c.w | e.x | e.y | e.z | e.w) || m0 || m1 || m2 || m3;
                    if (!touched) continue;
                    if (!(m0 && m1 && m2 && m3)) v[q] = *reinterpret_cast<const float4 *>(x + t);
                }
                if (c.x | c.y | c.z | c.w | e.x | e.y | e.z | e.w) {
                    v[q].x = adjust(v[q].x, c.x, e.x, false);
                    v[q].y = adjust(v[q].y, c.y, e.y, false);
                    v[q].z = adjust(v[q].z, c.z, e.z, false);
                    v[q].w = adjust(v[q].w, c.w, e.w, false);
                }
                const float low = -__builtin_inff();
                v[q].x = m0 ? low : v[q].x;
                v[q].y = m1 ? low : v[q].y;
                v[q].z = m2 ? low : v[q].z;
                v[q].w = m3 ? low : v[q].w;
                if constexpr (INPLACE) *reinterpret_cast<float4 *>(y + t) = v[q];
                else st_nt(reinterpret_cast<float4 *>(y + t), v[q]);
            } else {
                const uint32_t cs[4] = {c.x, c.y, c.z, c.w}, es[4] = {e.x, e.y, e.z, e.w};
                for (int k = 0; k < 4; ++k) {
                    if (t + k < 0 || t + k >= card) continue;
                    const bool m = masked_at(t + k);
                    if (INPLACE && !cs[k] && !es[k] && !m) continue;
                    y[(t + k) * a.y_st] = adjust(x[(t + k) * a.x_st], cs[k], es[k], m);
                }
            }
        }
    }
}

template <uint32_t Q, bool PACKED>
void la_launch(const LogitsAdjustArgs &a, bool vec, bool inplace, hipStream_t stream)
{
    const uint64_t runs = (static_cast<uint64_t>(a.card) + (vec ? 3 : 0) + la_tokens(Q) - 1) / la_tokens(Q);
    const uint64_t items = runs * a.rows;
    const uint32_t grid = static_cast<uint32_t>(items < (1u << 20) ? items : 1u << 20), n = static_cast<uint32_t>(runs);
    if (vec && inplace) k_la_adjust<Q, PACKED, true, true><<<grid, kBlock, 0, stream>>>(a, n, items);
    else if (vec) k_la_adjust<Q, PACKED, true, false><<<grid, kBlock, 0, stream>>>(a, n, items);
    else if (inplace) k_la_adjust<Q, PACKED, false, true><<<grid, kBlock, 0, stream>>>(a, n, items);
    else k_la_adjust<Q, PACKED, false, false><<<grid, kBlock, 0, stream>>>(a, n, items);
}

} // namespace

hipError_t launch_logits_adjust(const LogitsAdjustArgs &a, hipStream_t stream)
{
    const bool inplace = a.x == a.y; // and then of one layout
    const uint64_t apart = (reinterpret_cast<uintptr_t>(a.x) ^ reinterpret_cast<uintptr_t>(a.y)) % 16;
    const bool vec = a.x_st == 1 && a.y_st == 1 && apart == 0 && (a.rows == 1 || (a.x_row - a.y_row) % 4 == 0);
    const bool packed = a.history.entries < 65536 && a.bias.entries < 65535;
    const bool few = static_cast<uint64_t>(a.card) * a.rows <= kLaFew;
    if (few) packed ? la_launch<1, true>(a, vec, inplace, stream) : la_launch<1, false>(a, vec, inplace, stream);
    else packed ? la_launch<4, true>(a, vec, inplace, stream) : la_launch<4, false>(a, vec, inplace, stream);
    return hipGetLastError();
}

} // namespace emel
