// Attention over a paged e4m3 cache, heads of 129 to 256 elements.
#include "paged_attention.cuh"

namespace tf {

template struct AttendCall<256, true, 8>;
template struct AttendCall<256, true, 16>;
template struct AttendCall<256, true, 32>;
template struct AttendCall<256, true, 64>;

}  // namespace tf
