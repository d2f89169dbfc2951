// packed_q4q4.hip -- the attention over pages of Q4_0 keys and Q4_0 values.
#include "packed_attn.hpp"

namespace emel {

template hipError_t packed_attn<PaPages::Q4Q4>(const PagedAttnArgs &, const PaPlan &, uint32_t, uint32_t, hipStream_t);

} // namespace emel
