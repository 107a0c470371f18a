// Attention over a paged e4m3 cache, heads of 65 to 96 elements.
#include "paged_attention.cuh"

namespace tf {

template struct AttendCall<96, true, 8>;
template struct AttendCall<96, true, 16>;
template struct AttendCall<96, true, 24>;
template struct AttendCall<96, true, 32>;
template struct AttendCall<96, true, 48>;
template struct AttendCall<96, true, 64>;

}  // namespace tf
