// Attention over a paged e4m3 cache, heads of 97 to 128 elements.
#include "paged_attention.cuh"

namespace tf {

template struct AttendCall<128, true, 8>;
template struct AttendCall<128, true, 16>;
template struct AttendCall<128, true, 24>;
template struct AttendCall<128, true, 32>;
template struct AttendCall<128, true, 48>;
template struct AttendCall<128, true, 64>;

}  // namespace tf
