// quantmat.hip -- products of packed 4-bit weights with f32 columns:
//   y[r, c] = sum over k of W[r, k] x[k, c],
// W[r, k] = (q - 8) d for Q4_0 (blocks of 32 values: an f16 d, 16 bytes of
// nibbles, the low ones first) and d sc q - dmin m for Q4_K (blocks of 256: f16 d and
// dmin, eight 6-bit sc and m, 128 bytes of nibbles).
#include "common.hpp"
#include "launch.hpp"
#include "libm_replica.hpp"

namespace emel {
namespace {

__device__ __forceinline__ float ld_half(const unsigned char *p)
{
    return hw_fp16_to_f32(static_cast<uint16_t>(p[0] | (p[1] << 8)));
}

// A wave per output, a block of 32 values per lane and step.
template <bool Q4K>
__global__ __launch_bounds__(kBlock) void k_qm_wave(QMatArgs a, uint64_t outputs)
{
    const unsigned lane = threadIdx.x % kWave;
    const uint64_t waves = static_cast<uint64_t>(gridDim.x) * (kBlock / kWave);
    const uint32_t groups = a.k / 32;
    const uint64_t row_bytes = Q4K ? static_cast<uint64_t>(a.k / 256) * 144 : static_cast<uint64_t>(groups) * 18;
    for (uint64_t o = static_cast<uint64_t>(blockIdx.x) * (kBlock / kWave) + threadIdx.x / kWave; o < outputs; o += waves) {
        const uint64_t r = o % a.m, c = o / a.m;
        const unsigned char *row = static_cast<const unsigned char *>(a.w) + r * row_bytes;
        const float *x = a.x + static_cast<int64_t>(c) * a.x_st[1];
        float sum = 0.0f;
        for (uint32_t g = lane; g < groups; g += kWave) {
            float d, off;
            const unsigned char *q;
            unsigned shift;
            if constexpr (Q4K) {
                const unsigned char *b = row + static_cast<uint64_t>(g / 8) * 144;
                const unsigned j = g % 8;
                const unsigned char *s = b + 4;
                const unsigned sc = j < 4 ? s[j] & 63u : (s[j + 4] & 15u) | ((s[j - 4] >> 6) << 4);
                const unsigned mn = j < 4 ? s[j + 4] & 63u : (s[j + 4] >> 4) | ((s[j] >> 6) << 4);
                d = ld_half(b) * static_cast<float>(sc);
                off = ld_half(b + 2) * static_cast<float>(mn);
                q = b + 16 + 32 * (j / 2);
                shift = 4 * (j % 2);
            } else {
                const unsigned char *b = row + static_cast<uint64_t>(g) * 18;
                d = ld_half(b);
                off = 8.0f * d;
                q = b + 2;
                shift = 0;
            }
            for (unsigned i = 0; i < 32; ++i) {
                const unsigned v = Q4K ? (q[i] >> shift) & 15u : (i < 16 ? q[i] & 15u : q[i - 16] >> 4);
                const float w = d * static_cast<float>(v) - off;
                sum += w * x[static_cast<int64_t>(g * 32ull + i) * a.x_st[0]];
            }
        }
        sum = wave_sum_dpp(sum);
        if (lane == 0) a.y[static_cast<int64_t>(r) * a.y_st[0] + static_cast<int64_t>(c) * a.y_st[1]] = sum;
    }
}

} // namespace

uint64_t quant_mat_workspace_bytes(const QMatArgs &) { return 0; }

hipError_t launch_quant_mat(const QMatArgs &a, hipStream_t stream)
{
    const uint64_t outputs = static_cast<uint64_t>(a.m) * a.n;
    const uint64_t wgs = (outputs + 3) / 4;
    const uint32_t grid = static_cast<uint32_t>(wgs < 16384 ? wgs : 16384);
    if (a.q4k) k_qm_wave<true><<<grid, kBlock, 0, stream>>>(a, outputs);
    else k_qm_wave<false><<<grid, kBlock, 0, stream>>>(a, outputs);
    return hipGetLastError();
}

} // namespace emel
