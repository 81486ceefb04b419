// policy_f32.cu — the policy rows of f32 values.
#include "policy_launch.cuh"

namespace kc {
namespace pol {
cudaError_t draw_f32(const DrawArg& a, int sms, cudaStream_t s) { return draw_as<float>(a, sms, s); }
cudaError_t loss_f32(const LossArg& a, int sms, cudaStream_t s) { return loss_as<float>(a, sms, s); }
cudaError_t prepare_f32() { return prepare_as<float>(); }
}  // namespace pol
}  // namespace kc
