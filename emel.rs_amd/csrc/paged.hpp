// paged.hpp -- what the kernels of the paged key-value cache share.
#pragma once

#include "common.hpp"
#include "launch.hpp"

namespace emel {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef u4 u4_any __attribute__((aligned(2))); // pools may start at any half
typedef u2 u2_any __attribute__((aligned(2)));
typedef uint32_t u1_any __attribute__((aligned(2)));
typedef v4f v4f_any __attribute__((aligned(4)));

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

template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}

// A block's scale: what is not finite stands for NaN.
__device__ __forceinline__ float pk_scale(uint16_t bits)
{
    const float d = from_half<false>(bits);
    return __builtin_fmaf(d, 0.0f, d);
}

// ---- attention -----------------------------------------------------------------------------

constexpr uint32_t kPaUnit = 128;  // tokens of a unit, 32 a wave
constexpr uint32_t kPaLead = 16;   // packed: heads of a row
constexpr uint32_t kDies = 8;      // that blocks are dealt to in turn
constexpr uint32_t kPaLine = 64;   // words between arrival counters (a cache line each)

// What the pages of keys and of values hold.
enum class PaPages : int { F16 = 0, Bf16, Q8Q8, Q8Q4, Q4Q8, Q4Q4 };

// Columns of a packed row's head of ks blocks, whose keys `group` heads share: as
// many as 16 columns and its blocks allow (64 sequences of 90 to 9000 tokens with
// 32/8 heads of 128 in Q4_0 54.8 us with four, 68.8 with one; one of 4001 12.4 and 14.8).
constexpr int pa_fold(int ks, uint32_t group)
{
    int f = 8;
    while (f > 1 && (f / 2 >= ks || group > 16u / f)) f /= 2; // group * f may pass 32 bits
    return f;
}

// Workgroups that a compute unit holds at once: the registers that their
// launch bounds leave them.  `fold` is 0 for halves.  Packed heads of 96 and 128 with a
// column each (more than 8 heads share their keys) scale and split a block's
// weights at a time, which 168 registers do not hold: 64 sequences of 90 to 9000
// tokens with 32/2 heads of 128 in Q4_0 35.0 us, 44.9 with three, in Q8_0 38.9 and 60.3.
// Heads of 64 with a column each do not fit 128 registers: 24/2 heads in Q4_0 23.2 us, 24.7
// with four, in Q8_0 25.2 and 40.1.  Three kernels (Q8_0 with 4 blocks and 4 columns, Q8_0 keys
// with 8 blocks and one) keep two to four registers of a segment in scratch, none of a step.
constexpr uint32_t pa_per_cu(int ks, int fold)
{
    if (fold == 1 && ks > 1) return ks == 2 ? 3 : 2;
    return ks <= 2 ? 4 : ks <= 4 ? 3 : 2;
}

// What a launch derives on the host.
struct PaPlan {
    FastDiv page;       // tokens per page
    FastDiv dim, hgroups;
    FastDiv grid, few;  // workgroups: all, and two a compute unit
    uint32_t group;     // query heads of a cache head
    uint32_t rows;      // rows of a sequence: kv_heads * hgroups
    uint32_t slot;      // floats of a workspace slot
    uint32_t side;      // packed: rows side by side
    float *parts;       // 2 slots a workgroup
    uint32_t *arrived;  // a counter per workgroup, zero between launches
};

// The launch over packed pages, a source for each pair of types.
template <PaPages PAGES>
hipError_t packed_attn(const PagedAttnArgs &args, const PaPlan &plan, uint32_t grid, uint32_t lds, hipStream_t stream);

// ---- new tokens ------------------------------------------------------------------------------

constexpr uint32_t kPaAppend = 1u << 17; // tokens of a launch

// The slots of T tokens from t0 on, and (as bits) which of them are not
// stored: without a slot of the pool, or with one that a later token names.
template <uint32_t T>
__device__ __forceinline__ uint32_t pa_dropped(const PagedAppendArgs &a, uint32_t t0, int32_t mine[T], uint32_t *gone)
{
    const uint64_t slots = static_cast<uint64_t>(a.page) * a.pages;
    uint32_t skip = 0;
    for (uint32_t i = 0; i < T; ++i) {
        mine[i] = t0 + i < a.tokens ? a.slots[static_cast<int64_t>(t0 + i) * a.slots_st] : -1;
        if (mine[i] < 0 || static_cast<uint64_t>(mine[i]) >= slots) skip |= 1u << i;
    }
    if (threadIdx.x == 0) *gone = skip;
    __syncthreads();
    uint32_t later = 0;
#pragma unroll 4
    for (uint32_t u = t0 + 1 + threadIdx.x; u < a.tokens; u += kBlock) {
        const int32_t s = a.slots[static_cast<int64_t>(u) * a.slots_st];
        for (uint32_t i = 0; i < T; ++i) later |= s == mine[i] && u > t0 + i ? 1u << i : 0u;
    }
    if (later & ~skip) atomicOr(gone, later);
    __syncthreads();
    return *gone;
}

} // namespace emel
