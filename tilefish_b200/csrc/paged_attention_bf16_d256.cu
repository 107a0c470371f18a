// Attention over a paged bf16 cache, heads of 129 to 256 elements.
#include "paged_attention.cuh"

namespace tf {

template struct AttendCall<256, false, 8>;
template struct AttendCall<256, false, 16>;
template struct AttendCall<256, false, 32>;
template struct AttendCall<256, false, 64>;

}  // namespace tf
