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

// A wave per (head, sequence), one position at a time, each lane four dims:
// running maximum m, sum l and weighted values.
template <bool BF16>
__global__ __launch_bounds__(kWave) void k_pa_attn(PagedAttnArgs a)
{
    const unsigned lane = threadIdx.x;
    const uint64_t rows = static_cast<uint64_t>(a.heads) * a.seqs;
    const float nan = __builtin_nanf("");
    for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const int64_t h = row % a.heads, s = row / a.heads;
        const int64_t kh = h / (a.heads / a.kv_heads);
        const int64_t len = a.lengths[s * a.lengths_st];
        const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page;
        bool bad = len < 0 || len > cap;
        float q[4], acc[4] = {};
        for (int i = 0; i < 4; ++i) {
            const uint32_t d = lane * 4 + i;
            q[i] = d < a.dim ? a.q[d * a.q_st[0] + h * a.q_st[1] + s * a.q_st[2]] : 0.0f;
        }
        float m = -__builtin_inff(), l = 0.0f;
        const int64_t first = a.window && len > a.window ? len - a.window : 0;
        for (int64_t j = first; j < len && !bad; ++j) {
            const int32_t p = a.table[(j / a.page) * a.table_st[0] + s * a.table_st[1]];
            if (p < 0 || static_cast<uint32_t>(p) >= a.pages) {
                bad = true;
                break;
            }
            const int64_t i0 = j % a.page;
            const uint16_t *k = a.k_pool.data + p * a.k_pool.st_page + kh * a.k_pool.st_head + i0 * a.k_pool.st_tok;
            const uint16_t *v = a.v_pool.data + p * a.v_pool.st_page + kh * a.v_pool.st_head + i0 * a.v_pool.st_tok;
            float z = 0.0f;
            for (uint32_t i = 0; i < 4; ++i)
                if (lane * 4 + i < a.dim) z += q[i] * from_half<BF16>(k[lane * 4 + i]);
            z = wave_sum(z) * a.scale;
            if (a.soft_cap > 0.0f) z = a.soft_cap * tanhf(z / a.soft_cap);
            const float mn = z > m || z != z ? z : m;
            const float ref = mn == -__builtin_inff() ? 0.0f : mn;
            const float f = expf(m - ref), e = expf(z - ref);
            l = l * f + e;
            for (uint32_t i = 0; i < 4; ++i)
                if (lane * 4 + i < a.dim) acc[i] = acc[i] * f + e * from_half<BF16>(v[lane * 4 + i]);
            m = mn;
        }
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t d = lane * 4 + i;
            if (d < a.dim)
                a.y[d * a.y_st[0] + h * a.y_st[1] + s * a.y_st[2]] = bad ? nan : len == 0 ? 0.0f : acc[i] / l;
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

uint64_t paged_attn_workspace_bytes(const PagedAttnArgs &) { return 0; }

hipError_t launch_paged_attn(const PagedAttnArgs &a, hipStream_t stream)
{
    const uint64_t rows = static_cast<uint64_t>(a.heads) * a.seqs;
    const uint32_t grid = static_cast<uint32_t>(rows < (1u << 20) ? rows : 1u << 20);
    if (a.bf16) k_pa_attn<true><<<grid, kWave, 0, stream>>>(a);
    else k_pa_attn<false><<<grid, kWave, 0, stream>>>(a);
    return hipGetLastError();
}

} // namespace emel
