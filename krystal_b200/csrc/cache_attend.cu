// cache_attend.cu — how attention calls over the bank cache are cut, and their
// launchers by question type.
#include "cache_attend.cuh"

namespace kc {
namespace cache {

// A call whose sequences (or lists) are long beside the number of its units is cut
// along them, so that about kWaves CTAs run on every place for one; a part keeps
// at least four cells a team, below which its start costs more than it brings.
uint64_t plan_attend(AttendArg& a, int sms) {
  constexpr uint64_t kWaves = 4;
  const Shape sh = shape_of(a, sms);
  const uint32_t blocks = std::max(1u, a.block_count ? a.block_count : (a.t.max_len + kPage - 1) / kPage);
  const uint64_t ctas = std::max<uint64_t>(1, (sh.items + sh.hg - 1) / sh.hg), places = uint64_t(sms) * (a.c.dim == 128 ? 1 : 2);
  const uint64_t want = std::max<uint64_t>(1, places * kWaves / ctas);
  a.chunk = uint32_t(std::max<uint64_t>(2 * sh.kg, (blocks + want - 1) / want));
  a.splits = (blocks + a.chunk - 1) / a.chunk;
  return a.splits == 1 ? 0 : uint64_t(a.a.questions) * a.a.heads * a.splits * (a.c.dim + 4);
}

cudaError_t launch_attend(const AttendArg& a, int sms, cudaStream_t s, uint64_t* launches) {
  if (a.a.questions == 0 || a.t.seqs == 0) return cudaSuccess;
  return a.a.dtype == kF32 ? attend_f32(a, sms, s, launches)
       : a.a.dtype == kF16 ? attend_f16(a, sms, s, launches) : attend_bf16(a, sms, s, launches);
}

cudaError_t launch_scores(const ScoreArg& a, int sms, cudaStream_t s, uint64_t* launches) {
  if (a.a.questions == 0 || a.t.seqs == 0) return cudaSuccess;
  return a.a.dtype == kF32 ? scores_f32(a, sms, s, launches)
       : a.a.dtype == kF16 ? scores_f16(a, sms, s, launches) : scores_bf16(a, sms, s, launches);
}

cudaError_t prepare() {
  cudaError_t e;
  if ((e = prepare_store()) || (e = prepare_f32()) || (e = prepare_f16()) || (e = prepare_bf16())) return e;
  return cudaSuccess;
}

}  // namespace cache
}  // namespace kc
