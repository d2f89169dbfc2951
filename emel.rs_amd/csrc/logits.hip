// logits.hip -- penalties for repeated tokens, biases and a token mask on
// rows of logits, ahead of the sampler.
//
// A workgroup takes a run of kLaTokens tokens of one row.  It counts the
// row's history ids that fall in its run, and the last bias entry of each
// token there, in LDS (integer atomics: the result does not depend on their
// order), then passes over the run once.
#include "common.hpp"
#include "launch.hpp"

namespace emel {
namespace {

constexpr uint32_t kLaTokens = 4096;

__device__ __forceinline__ float row_value(const RowTable &t, uint32_t row, float none)
{
    return t.data ? static_cast<const float *>(t.data)[row * t.row_st] : none;
}

__global__ __launch_bounds__(kBlock) void k_la_adjust(LogitsAdjustArgs a, uint32_t runs, uint64_t items)
{
    __shared__ uint32_t count[kLaTokens];
    __shared__ uint32_t entry[kLaTokens]; // 1 + the last bias entry
    for (uint64_t it = blockIdx.x; it < items; it += gridDim.x) {
        const uint32_t row = static_cast<uint32_t>(it / runs);
        const uint32_t t0 = static_cast<uint32_t>(it % runs) * kLaTokens;
        const uint32_t n = a.card - t0 < kLaTokens ? a.card - t0 : kLaTokens;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < kLaTokens; i += kBlock) count[i] = entry[i] = 0;
        __syncthreads();
        if (a.history.data) {
            int64_t len = a.history.entries;
            if (a.history_len.data) {
                const int64_t v = static_cast<const int32_t *>(a.history_len.data)[row * a.history_len.row_st];
                len = v < 0 ? 0 : v < len ? v : len;
            }
            const int32_t *ids = static_cast<const int32_t *>(a.history.data) + row * a.history.row_st;
            for (int64_t i = threadIdx.x; i < len; i += kBlock) {
                const uint32_t t = static_cast<uint32_t>(ids[i * a.history.st]) - t0;
                if (t < n) atomicAdd(&count[t], 1u);
            }
        }
        if (a.bias.data) {
            const int32_t *ids = static_cast<const int32_t *>(a.bias_ids.data) + row * a.bias_ids.row_st;
            for (uint32_t i = threadIdx.x; i < a.bias.entries; i += kBlock) {
                const uint32_t t = static_cast<uint32_t>(ids[i * a.bias_ids.st]) - t0;
                if (t < n) atomicMax(&entry[t], i + 1);
            }
        }
        __syncthreads();
        const float repeat = row_value(a.repeat, row, 1.0f);
        const float frequency = row_value(a.frequency, row, 0.0f);
        const float presence = row_value(a.presence, row, 0.0f);
        for (uint32_t i = threadIdx.x; i < n; i += kBlock) {
            const uint32_t t = t0 + i;
            float l = a.x[t * a.x_st + row * a.x_row];
            if (const uint32_t c = count[i]) {
                l = l > 0.0f ? l / repeat : l * repeat;
                l = (l - static_cast<float>(c) * frequency) - presence;
            }
            if (const uint32_t e = entry[i])
                l += static_cast<const float *>(a.bias.data)[(e - 1) * a.bias.st + row * a.bias.row_st];
            if (a.allowed.data) {
                const int32_t *bits = static_cast<const int32_t *>(a.allowed.data) + row * a.allowed.row_st;
                if (!((static_cast<uint32_t>(bits[(t / 32) * a.allowed.st]) >> (t % 32)) & 1u)) l = -__builtin_inff();
            }
            a.y[t * a.y_st + row * a.y_row] = l;
        }
    }
}

} // namespace

hipError_t launch_logits_adjust(const LogitsAdjustArgs &a, hipStream_t stream)
{
    const uint32_t runs = (a.card + kLaTokens - 1) / kLaTokens;
    const uint64_t items = static_cast<uint64_t>(runs) * a.rows;
    const uint32_t grid = static_cast<uint32_t>(items < (1u << 20) ? items : 1u << 20);
    k_la_adjust<<<grid, kBlock, 0, stream>>>(a, runs, items);
    return hipGetLastError();
}

} // namespace emel
