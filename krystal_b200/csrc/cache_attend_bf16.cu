// cache_attend_bf16.cu — attention and pointer scores of bf16 questions.
#include "cache_attend.cuh"

namespace kc {
namespace cache {
cudaError_t attend_bf16(const AttendArg& a, int sms, cudaStream_t s, uint64_t* n) { return attend_as<__nv_bfloat16>(a, sms, s, n); }
cudaError_t scores_bf16(const ScoreArg& a, int sms, cudaStream_t s, uint64_t* n) { return scores_as<__nv_bfloat16>(a, sms, s, n); }
cudaError_t prepare_bf16() { return prepare_as<__nv_bfloat16>(); }
}  // namespace cache
}  // namespace kc
