// Few-columns forward kernels for f16 inputs and head sizes up to 96.
#include "attend_few.inl"

namespace vk {
hipError_t attend_few_f16_96(const AttendArgs& a, hipStream_t stream) { return attend::launch_few<attend::F16, 96>(a, stream); }
}  // namespace vk
