// Attention over a paged cache for heads of 129 to 256 elements.
#include "paged_attention.cuh"

namespace tf {

template struct AttendCall<256, false, 1>;
template struct AttendCall<256, false, 2>;
template struct AttendCall<256, false, 4>;
template struct AttendCall<256, true, 1>;
template struct AttendCall<256, true, 2>;
template struct AttendCall<256, true, 4>;

}  // namespace tf
