// packed_q8q4.hip -- the attention over pages of Q8_0 keys and Q4_0 values.
#include "packed_attn.hpp"

namespace emel {

template hipError_t packed_attn<PaPages::Q8Q4>(const PagedAttnArgs &, const PaPlan &, uint32_t, uint32_t, hipStream_t);

} // namespace emel
