// Attention over a paged e4m3 cache, heads of up to 64 elements.
#include "paged_attention.cuh"

namespace tf {

template struct AttendCall<64, true, 8>;
template struct AttendCall<64, true, 16>;
template struct AttendCall<64, true, 24>;
template struct AttendCall<64, true, 32>;
template struct AttendCall<64, true, 48>;
template struct AttendCall<64, true, 64>;

}  // namespace tf
