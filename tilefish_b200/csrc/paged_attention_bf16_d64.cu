// Attention over a paged bf16 cache, heads of up to 64 elements.
#include "paged_attention.cuh"

namespace tf {

template struct AttendCall<64, false, 8>;
template struct AttendCall<64, false, 16>;
template struct AttendCall<64, false, 24>;
template struct AttendCall<64, false, 32>;
template struct AttendCall<64, false, 48>;
template struct AttendCall<64, false, 64>;

}  // namespace tf
