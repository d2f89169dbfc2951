// packed.hip -- the attention of one new token per sequence over pages of packed
// rows (Q8_0, Q4_0): the kernels, of which paged.hip plans the launches.
#include "paged_attn.hpp"

namespace emel {
namespace {

template <PaPages PAGES>
hipError_t launch(const PagedAttnArgs &a, const PaPlan &pl, uint32_t grid, uint32_t lds, hipStream_t stream)
{
    switch (a.dim / 32) {
    case 1: k_pa_attn<PAGES, 1, 2><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 2: k_pa_attn<PAGES, 2, 4><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 3: k_pa_attn<PAGES, 3, 6><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 4: k_pa_attn<PAGES, 4, 8><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 5: k_pa_attn<PAGES, 5, 10><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 6: k_pa_attn<PAGES, 6, 12><<<grid, kBlock, lds, stream>>>(a, pl); break;
    case 7: k_pa_attn<PAGES, 7, 14><<<grid, kBlock, lds, stream>>>(a, pl); break;
    default: k_pa_attn<PAGES, 8, 16><<<grid, kBlock, lds, stream>>>(a, pl); break;
    }
    return hipGetLastError();
}

} // namespace

hipError_t launch_packed_attn(PaPages pages, const PagedAttnArgs &a, const PaPlan &pl, uint32_t grid, uint32_t lds, hipStream_t stream)
{
    switch (pages) {
    case PaPages::Q8Q8: return launch<PaPages::Q8Q8>(a, pl, grid, lds, stream);
    case PaPages::Q8Q4: return launch<PaPages::Q8Q4>(a, pl, grid, lds, stream);
    case PaPages::Q4Q8: return launch<PaPages::Q4Q8>(a, pl, grid, lds, stream);
    default: return launch<PaPages::Q4Q4>(a, pl, grid, lds, stream);
    }
}

} // namespace emel
