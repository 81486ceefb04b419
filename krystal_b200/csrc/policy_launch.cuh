// policy_launch.cuh — which group of warps a row of the longest length takes,
// for one element type; policy_f32.cu, policy_f16.cu and policy_bf16.cu
// instantiate it, a file a type so that they compile side by side.
#pragma once
#include "policy.cuh"

namespace kc {
namespace pol {

// One launch of kernel K over the rows, CL CTAs a row (W > 1) or four rows a
// CTA (W = 1).
template <typename A>
cudaError_t go(void (*kernel)(A), const A& a, int w, int cl, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(w == 1 ? 128 : unsigned(w) * 32);
  const uint64_t ctas = w == 1 ? (uint64_t(a.r.rows) + 3) / 4 : uint64_t(a.r.rows) * cl;
  if (ctas > 0x7fffffffu) return cudaErrorInvalidConfiguration;
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (cl > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(cl);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

// The group that holds the longest row, a vector's misalignment included.
template <typename T>
inline cudaError_t draw_as(const DrawArg& a, cudaStream_t s) {
  const uint64_t need = a.r.row_len + 16 / sizeof(T) - 1;
  constexpr int kMid = sizeof(T) == 4 ? 20 : 24;  // the largest bank, misaligned, in 8 warps
  if (need <= 256) return go(k_draw<T, 8, 1, 1>, a, 1, 1, s);
  if (need <= 1024) return go(k_draw<T, 32, 1, 1>, a, 1, 1, s);
  if (need <= 8 * 32 * kMid) return go(k_draw<T, kMid, 8, 1>, a, 8, 1, s);
  if (need <= 16384) return go(k_draw<T, 32, 16, 1>, a, 16, 1, s);
  if (need <= 32768) return go(k_draw<T, 64, 16, 1>, a, 16, 1, s);
  return go(k_draw<T, 64, 16, 8>, a, 16, 8, s);
}
template <typename T>
inline cudaError_t whole_as(const LossArg& a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const uint64_t need = a.r.row_len + V - 1;
  if (need <= 256) return go(k_policy_whole<T, 8 / V, 1, 1>, a, 1, 1, s);
  if (need <= 1024) return go(k_policy_whole<T, 32 / V, 1, 1>, a, 1, 1, s);
  if (need <= 6144) return go(k_policy_whole<T, 24 / V, 8, 1>, a, 8, 1, s);
  if (need <= 16384) return go(k_policy_whole<T, 32 / V, 16, 1>, a, 16, 1, s);
  constexpr int W = V == 4 ? 32 : 16;  // 8 vectors a thread
  if (need <= 32768) return go(k_policy_whole<T, 8, W, 1>, a, W, 1, s);
  return go(k_policy_whole<T, 8, W, 8>, a, W, 8, s);
}
template <typename T>
inline cudaError_t loss_as(const LossArg& a, cudaStream_t s) {
  const CutArg& c = a.c;
  if (!c.top_k && !c.row_top_k && !(c.top_p < 1.0f) && !c.row_top_p && !(c.min_p > 0.0f) && !c.row_min_p)
    return whole_as<T>(a, s);
  const uint64_t need = a.r.row_len + 16 / sizeof(T) - 1;
  constexpr int kMid = sizeof(T) == 4 ? 20 : 24;
  if (need <= 256) return go(k_policy_loss<T, 8, 1, 1>, a, 1, 1, s);
  if (need <= 1024) return go(k_policy_loss<T, 32, 1, 1>, a, 1, 1, s);
  if (need <= 8 * 32 * kMid) return go(k_policy_loss<T, kMid, 8, 1>, a, 8, 1, s);
  if (need <= 16384) return go(k_policy_loss<T, 32, 16, 1>, a, 16, 1, s);
  if (need <= 32768) return go(k_policy_loss<T, 64, 16, 1>, a, 16, 1, s);
  return go(k_policy_loss<T, 64, 16, 8>, a, 16, 8, s);
}

}  // namespace pol
}  // namespace kc
