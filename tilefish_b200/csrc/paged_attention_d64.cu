// Attention over a paged cache for heads of up to 64 elements.
#include "paged_attention.cuh"

namespace tf {

template struct AttendCall<64, false, 1>;
template struct AttendCall<64, false, 2>;
template struct AttendCall<64, false, 4>;
template struct AttendCall<64, true, 1>;
template struct AttendCall<64, true, 2>;
template struct AttendCall<64, true, 4>;

}  // namespace tf
