// cache_attend_f32.cu — attention and pointer scores of f32 questions.
#include "cache_attend.cuh"

namespace kc {
namespace cache {
cudaError_t attend_f32(const AttendArg& a, int sms, cudaStream_t s, uint64_t* n) { return attend_as<float>(a, sms, s, n); }
cudaError_t scores_f32(const ScoreArg& a, int sms, cudaStream_t s, uint64_t* n) { return scores_as<float>(a, sms, s, n); }
cudaError_t prepare_f32() { return prepare_as<float>(); }
}  // namespace cache
}  // namespace kc
