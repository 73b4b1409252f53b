// Forward tile kernels for bf16 inputs and head sizes up to 32.
#include "attend_forward.inl"

namespace vk {
hipError_t attend_forward_bf16_32(const AttendArgs& a, hipStream_t stream) { return attend::launch_forward<attend::Bf16, 32>(a, stream); }
}  // namespace vk
