// policy_f16.cu — the policy rows of f16 values.
#include "policy_launch.cuh"

namespace kc {
namespace pol {
cudaError_t draw_f16(const DrawArg& a, int sms, cudaStream_t s) { return draw_as<__half>(a, sms, s); }
cudaError_t loss_f16(const LossArg& a, int sms, cudaStream_t s) { return loss_as<__half>(a, sms, s); }
cudaError_t prepare_f16() { return prepare_as<__half>(); }
}  // namespace pol
}  // namespace kc
