// Attention over a paged cache for heads of 65 to 128 elements.
#include "paged_attention.cuh"

namespace tf {

template struct AttendCall<128, false, 1>;
template struct AttendCall<128, false, 2>;
template struct AttendCall<128, false, 4>;
template struct AttendCall<128, true, 1>;
template struct AttendCall<128, true, 2>;
template struct AttendCall<128, true, 4>;

}  // namespace tf
