// Backward tile kernels for f16 inputs and head sizes up to 96.
#include "attend_backward.inl"

namespace vk {
hipError_t attend_grad_q_f16_96(const AttendGradArgs& g, hipStream_t stream) { return attend::launch_grad_q<attend::F16, 96>(g, stream); }
hipError_t attend_grad_kv_f16_96(const AttendGradArgs& g, hipStream_t stream) { return attend::launch_grad_kv<attend::F16, 96>(g, stream); }
}  // namespace vk
