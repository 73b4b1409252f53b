// Backward tile kernels for f16 inputs and head sizes up to 32.
#include "attend_backward.inl"

namespace vk {
hipError_t attend_grad_q_f16_32(const AttendGradArgs& g, hipStream_t stream) { return attend::launch_grad_q<attend::F16, 32>(g, stream); }
hipError_t attend_grad_kv_f16_32(const AttendGradArgs& g, hipStream_t stream) { return attend::launch_grad_kv<attend::F16, 32>(g, stream); }
}  // namespace vk
