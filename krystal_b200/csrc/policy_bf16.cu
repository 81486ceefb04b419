// policy_bf16.cu — the policy rows of bf16 values.
#include "policy_launch.cuh"

namespace kc {
namespace pol {
cudaError_t draw_bf16(const DrawArg& a, int sms, cudaStream_t s) { return draw_as<__nv_bfloat16>(a, sms, s); }
cudaError_t loss_bf16(const LossArg& a, int sms, cudaStream_t s) { return loss_as<__nv_bfloat16>(a, sms, s); }
cudaError_t prepare_bf16() { return prepare_as<__nv_bfloat16>(); }
}  // namespace pol
}  // namespace kc
