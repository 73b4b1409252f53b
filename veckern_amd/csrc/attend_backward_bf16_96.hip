// Backward tile kernels for bf16 inputs and head sizes up to 96.
#include "attend_backward.inl"

namespace vk {
hipError_t attend_grad_q_bf16_96(const AttendGradArgs& g, hipStream_t stream) { return attend::launch_grad_q<attend::Bf16, 96>(g, stream); }
hipError_t attend_grad_kv_bf16_96(const AttendGradArgs& g, hipStream_t stream) { return attend::launch_grad_kv<attend::Bf16, 96>(g, stream); }
}  // namespace vk
