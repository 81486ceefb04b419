// policy.cu — the launchers of the policy rows (policy.cuh, by element type) and
// of the gradient clipping (clip.cuh).
#include <algorithm>

#include "clip.cuh"
#include "policy_args.h"

namespace kc {
namespace pol {

cudaError_t prepare() {
  cudaError_t e;
  if ((e = prepare_f32()) || (e = prepare_f16()) || (e = prepare_bf16())) return e;
  return cudaSuccess;
}

cudaError_t launch_draw(const DrawArg& a, int dtype, int sms, cudaStream_t stream, uint64_t* launches) {
  if (a.r.rows == 0) return cudaSuccess;
  ++*launches;
  return dtype == kF32 ? draw_f32(a, sms, stream) : dtype == kF16 ? draw_f16(a, sms, stream) : draw_bf16(a, sms, stream);
}

cudaError_t launch_policy_loss(const LossArg& a, int dtype, int sms, cudaStream_t stream, uint64_t* launches) {
  if (a.r.rows == 0) return cudaSuccess;
  ++*launches;
  return dtype == kF32 ? loss_f32(a, sms, stream) : dtype == kF16 ? loss_f16(a, sms, stream) : loss_bf16(a, sms, stream);
}

}  // namespace pol

namespace clip {
namespace {

template <uint32_t N>
unsigned fill(Table<N>& tb, Tensor* t, uint32_t count, uint32_t ctas) {
  uint64_t bytes = 0, chunk = 0;
  for (uint32_t i = 0; i < count; i++) bytes += t[i].n * dtype_bytes(t[i].dtype);
  tb.chunk_bytes = kMinChunk;
  while (tb.chunk_bytes < kMaxChunk && uint64_t(tb.chunk_bytes) * ctas < bytes) tb.chunk_bytes *= 2;
  for (uint32_t i = 0; i < count; i++) {
    tb.t[i] = t[i];
    tb.t[i].chunk0 = uint32_t(chunk);
    const uint64_t per = tb.chunk_bytes / dtype_bytes(t[i].dtype);
    chunk += (t[i].n + per - 1) / per;
  }
  tb.count = count;
  tb.chunks = uint32_t(chunk);
  return tb.chunks;
}

template <uint32_t N>
cudaError_t run(Tensor* t, uint64_t count, double max_norm, double* workspace, double* result, int sms,
                cudaStream_t stream, uint64_t* launches) {
  const uint32_t most = std::min<uint32_t>(kMaxCtas, uint32_t(sms) * 4);
  static thread_local Table<N> tb;
  const bool one = count <= N;
  uint32_t partials = 0;
  for (int pass = 0; pass < 2; pass++) {
    uint64_t at = 0;
    do {
      const uint32_t chunks = fill(tb, t + at, uint32_t(std::min<uint64_t>(N, count - at)), most);
      const unsigned grid = std::max(1u, std::min(most, chunks));
      if (pass == 0) {
        k_norm<N><<<grid, kThreads, 0, stream>>>(tb, workspace + partials);
        partials += grid;
      } else {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(grid);
        cfg.blockDim = dim3(kThreads);
        cfg.stream = stream;
        cudaLaunchAttribute early[1];
        early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        early[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = early;
        cfg.numAttrs = one ? 1 : 0;  // the launch ahead is k_norm's
        const cudaError_t e = cudaLaunchKernelEx(&cfg, k_scale<N>, tb, static_cast<const double*>(workspace),
                                                 one ? partials : 0u, max_norm, result);
        if (e) return e;
      }
      ++*launches;
      at += N;
    } while (at < count);
    if (pass == 0 && !one) {
      k_join<<<1, kThreads, 0, stream>>>(workspace, partials, max_norm, result);
      ++*launches;
    }
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_clip(Tensor* t, uint64_t count, double max_norm, double* workspace, double* result, int sms,
                        cudaStream_t stream, uint64_t* launches) {
  return count <= kShortTable ? run<kShortTable>(t, count, max_norm, workspace, result, sms, stream, launches)
                              : run<kTable>(t, count, max_norm, workspace, result, sms, stream, launches);
}

}  // namespace clip
}  // namespace kc
