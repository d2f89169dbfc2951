// packed_attn.hpp -- the attention over packed pages of one pair of types; a source
// each builds its kernels, so that they build side by side.
#pragma once

#include "paged_attn.hpp"

namespace emel {
namespace {

// With pa_fold's columns a head, which the launch's LDS is for.
template <PaPages PAGES, int KS, int F = pa_fold(KS, 1)>
void attend(const PagedAttnArgs &a, const PaPlan &pl, uint32_t grid, uint32_t lds, hipStream_t stream)
{
    if constexpr (F > 1)
        if (pa_fold(KS, pl.group) < F) return attend<PAGES, KS, F / 2>(a, pl, grid, lds, stream);
    k_pa_attn<PAGES, KS, 2 * KS, F><<<grid, kBlock, lds, stream>>>(a, pl);
}

} // namespace

template <PaPages PAGES>
hipError_t packed_attn(const PagedAttnArgs &a, const PaPlan &pl, uint32_t grid, uint32_t lds, hipStream_t stream)
{
    switch (a.dim / 32) {
    case 1: attend<PAGES, 1>(a, pl, grid, lds, stream); break;
    case 2: attend<PAGES, 2>(a, pl, grid, lds, stream); break;
    case 3: attend<PAGES, 3>(a, pl, grid, lds, stream); break;
    case 4: attend<PAGES, 4>(a, pl, grid, lds, stream); break;
    case 5: attend<PAGES, 5>(a, pl, grid, lds, stream); break;
    case 6: attend<PAGES, 6>(a, pl, grid, lds, stream); break;
    case 7: attend<PAGES, 7>(a, pl, grid, lds, stream); break;
    default: attend<PAGES, 8>(a, pl, grid, lds, stream); break;
    }
    return hipGetLastError();
}

} // namespace emel
