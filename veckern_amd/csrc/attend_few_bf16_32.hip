// Few-columns forward kernels for bf16 inputs and head sizes up to 32.
#include "attend_few.inl"

namespace vk {
hipError_t attend_few_bf16_32(const AttendArgs& a, hipStream_t stream) { return attend::launch_few<attend::Bf16, 32>(a, stream); }
}  // namespace vk
