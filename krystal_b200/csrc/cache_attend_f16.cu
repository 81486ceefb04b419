// cache_attend_f16.cu — attention and pointer scores of f16 questions.
#include "cache_attend.cuh"

namespace kc {
namespace cache {
cudaError_t attend_f16(const AttendArg& a, int sms, cudaStream_t s, uint64_t* n) { return attend_as<__half>(a, sms, s, n); }
cudaError_t scores_f16(const ScoreArg& a, int sms, cudaStream_t s, uint64_t* n) { return scores_as<__half>(a, sms, s, n); }
cudaError_t prepare_f16() { return prepare_as<__half>(); }
}  // namespace cache
}  // namespace kc
