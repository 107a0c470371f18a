// Attention over a paged bf16 cache, heads of 65 to 96 elements.
#include "paged_attention.cuh"

namespace tf {

template struct AttendCall<96, false, 8>;
template struct AttendCall<96, false, 16>;
template struct AttendCall<96, false, 24>;
template struct AttendCall<96, false, 32>;
template struct AttendCall<96, false, 48>;
template struct AttendCall<96, false, 64>;

}  // namespace tf
