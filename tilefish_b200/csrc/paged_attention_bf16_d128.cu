// Attention over a paged bf16 cache, heads of 97 to 128 elements.
#include "paged_attention.cuh"

namespace tf {

template struct AttendCall<128, false, 8>;
template struct AttendCall<128, false, 16>;
template struct AttendCall<128, false, 24>;
template struct AttendCall<128, false, 32>;
template struct AttendCall<128, false, 48>;
template struct AttendCall<128, false, 64>;

}  // namespace tf
