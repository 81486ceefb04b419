// cache_attend.cu — how attention calls over the bank cache are cut, and their
// launchers by question type.
#include "cache_attend.cuh"

namespace kc {
namespace cache {

// A call whose sequences (or lists) are long beside the number of its units is cut
// along them: into as many parts as fill every place for a CTA once, where all are
// of one length (lists, a single sequence: 54 us against 79 for 4 times as many
// parts of 400003 rows), and 4 times where lengths may differ, so that long ones do
// not run on alone (32 sequences of 1 to 16384 rows: 112 against 121 us). A part
// keeps at least four cells a team, below which its start costs more than it brings.
uint64_t plan_attend(AttendArg& a, int sms) {
  const Shape sh = shape_of(a, sms);
  const uint32_t blocks = std::max(1u, a.block_count ? a.block_count : (a.t.max_len + kPage - 1) / kPage);
  const uint64_t waves = a.block_count || a.t.seqs == 1 ? 1 : 4;
  const uint64_t ctas = std::max<uint64_t>(1, (sh.items + sh.hg - 1) / sh.hg);
  const uint64_t places = uint64_t(sms) * (a.c.dim == 128 ? 1 : 2) * (kWarps / sh.warps);
  const uint64_t want = std::max<uint64_t>(1, places * waves / ctas);
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
