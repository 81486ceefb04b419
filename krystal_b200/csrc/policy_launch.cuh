// policy_launch.cuh — which group of warps a row of the longest length takes,
// for one element type; policy_f32.cu, policy_f16.cu and policy_bf16.cu
// instantiate it, a file a type so that they compile side by side.
#pragma once
#include <algorithm>

#include "policy_cut.cuh"
#include "policy_whole.cuh"

namespace kc {
namespace pol {

// One warp a row, four rows a CTA.
template <typename A>
cudaError_t go_warps(void (*kernel)(A), const A& a, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(128);
  cfg.gridDim = dim3(unsigned((uint64_t(a.r.rows) + 3) / 4));
  cfg.stream = stream;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

// A launch of k_policy_rows: `need` entries a row at most, misaligned as they
// may be. The batch is the one whose waves of CTAs take least: a batch costs
// its rows up to their lists, and about one and a half more rows for finishing
// them side by side (any price from 3/4 to 6 rows is within 5 %; without one,
// 4096 rows of 4096 take 168 us and not 122).
constexpr uint32_t kRowEntries = 32768;  // a CTA holds: 4 bytes of key and 2 of place an entry
constexpr size_t kRowSmem = size_t(kRowEntries) * 6;
template <typename T, int W, int CL, typename A>
cudaError_t go_rows(const A& a, uint64_t need, int sms, cudaStream_t stream) {
  constexpr uint64_t per = uint64_t(32) * (16 / sizeof(T)) * W * CL;
  const uint32_t chunks = uint32_t((need + per - 1) / per);
  const size_t smem = size_t(chunks) * per / CL * 6;
  const uint32_t most = CL > 1 ? 1u : uint32_t(std::min(W, kBatch));
  // CTAs that share an SM: by their threads, and by their shared memory (a list is 2.5 KB)
  const uint64_t fit = uint64_t(sms) * std::max<uint64_t>(1, std::min<uint64_t>(32 / W, 230000 / (smem + most * 2700 + 2048)));
  uint32_t batch = 1;
  double least = 1e300;
  for (uint32_t b = 1; b <= most; b++) {
    const double waves = double(((uint64_t(a.r.rows) + b - 1) / b + fit - 1) / fit);
    if (waves * (b + 1.5) < least) {
      least = waves * (b + 1.5);
      batch = b;
    }
  }
  const uint64_t ctas = (uint64_t(a.r.rows) + batch - 1) / batch * CL;
  if (ctas > 0x7fffffffu || smem > kRowSmem) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(W * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CL;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CL > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, k_policy_rows<T, W, CL, A>, a, batch, chunks);
}
template <typename T, typename A>
cudaError_t prepare_rows() {
  const auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
  cudaError_t e;
  if ((e = cudaFuncSetAttribute(k_policy_rows<T, 4, 1, A>, attr, int(kRowSmem))) ||
      (e = cudaFuncSetAttribute(k_policy_rows<T, 8, 1, A>, attr, int(kRowSmem))) ||
      (e = cudaFuncSetAttribute(k_policy_rows<T, 16, 1, A>, attr, int(kRowSmem))) ||
      (e = cudaFuncSetAttribute(k_policy_rows<T, 16, 2, A>, attr, int(kRowSmem))) ||
      (e = cudaFuncSetAttribute(k_policy_rows<T, 16, 4, A>, attr, int(kRowSmem))) ||
      (e = cudaFuncSetAttribute(k_policy_rows<T, 16, 8, A>, attr, int(kRowSmem))))
    return e;
  return cudaSuccess;
}

// The group that holds the longest row, a vector's misalignment included.
template <typename T, typename A>
cudaError_t cut_as(const A& a, int sms, cudaStream_t s) {
  constexpr uint64_t V = 16 / sizeof(T);
  const bool aligned = a.r.frames == 0 && a.r.pitch % V == 0 && (reinterpret_cast<uintptr_t>(a.r.values) & 15) == 0;
  const uint64_t need = a.r.row_len + (aligned ? 0 : V - 1);
  if (a.r.row_len + V - 1 <= kList) {
    // a row a warp, or runs of rows once there are eight for every warp that
    // fits, on twice the CTAs that fit: 34818 rows take 99 us on as many as fit,
    // 94 on twice and 95 on three times that, 97 with a row a warp
    const uint64_t ctas = (uint64_t(a.r.rows) + 3) / 4, fit = uint64_t(sms) * kSmallCtas;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(ctas > 8 * fit ? 2 * fit : ctas));
    cfg.blockDim = dim3(128);
    cfg.stream = s;
    return cudaLaunchKernelEx(&cfg, k_policy_small<T, A>, a);
  }
  // 4, 8 or 16 warps a row, f32 rows under top-k 50 and top-p: 4000 rows of 1900
  // take 55 us on 4 and 74 on 8, of 4000 90 and 94 (of 2500, 63 and 81); 2000
  // rows of 5000 64 on 8 and 77 on 16, 1000 rows of 16000 115 and 88
  if (need <= 2048) return go_rows<T, 4, 1>(a, need, sms, s);
  if (need <= 8192) return go_rows<T, 8, 1>(a, need, sms, s);
  if (need <= kRowEntries) return go_rows<T, 16, 1>(a, need, sms, s);
  // the fewest CTAs that hold the row: 600 rows of 32000 take 103 us in one and
  // 125 in two; 32 rows of 131071 37 us in clusters of 4 and of 8
  if (need <= 2 * kRowEntries) return go_rows<T, 16, 2>(a, need, sms, s);
  if (need <= 4 * kRowEntries) return go_rows<T, 16, 4>(a, need, sms, s);
  return go_rows<T, 16, 8>(a, need, sms, s);
}

// Rows that k_policy_long keeps in shared memory: CL CTAs of NT threads a row,
// up to kSmall bytes a row 64 threads, up to kShort 128, up to kLong 256 (three
// CTAs an SM), beyond that a cluster of 8 x 512. Few threads a row, and so many
// rows an SM, hide one row's reductions behind another's loads: 16384 bf16 rows
// of 8000 take 109 us on 64 threads and 121 on 128; 8192 of 13000 104 on 64 and
// 88 on 128; 4096 of 17000 66 on 128 and 68 on 256; 4096 of 25001 100 on 128, 88
// on 256 and 98 on 384. Up to 1024 entries a warp keeps the row in registers:
// 65536 bf16 rows of 1000 take 98 us, and 197 in shared memory; of 1100 to 2000
// a row in registers is the slower one (102 and 78 us).
constexpr uint64_t kSmall = 16384, kShort = 32768, kLong = 73728;
template <typename T>
constexpr size_t long_smem(uint64_t row_len, int cl) {
  constexpr uint64_t V = 16 / sizeof(T);
  return (((row_len + 2 * V - 2) / V + cl - 1) / cl + 4) * 16;
}
template <typename T>
cudaError_t prepare_as() {
  const auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
  cudaError_t e;
  if ((e = cudaFuncSetAttribute(k_policy_long<T, 64, 1>, attr, int(long_smem<T>(kSmall / sizeof(T), 1)))) ||
      (e = cudaFuncSetAttribute(k_policy_long<T, 128, 1>, attr, int(long_smem<T>(kShort / sizeof(T), 1)))) ||
      (e = cudaFuncSetAttribute(k_policy_long<T, 256, 1>, attr, int(long_smem<T>(kLong / sizeof(T), 1)))) ||
      (e = cudaFuncSetAttribute(k_policy_long<T, 512, 8>, attr, int(long_smem<T>(kMaxRow, 8)))))
    return e;
  if ((e = prepare_rows<T, DrawArg>()) || (e = prepare_rows<T, LossArg>())) return e;
  return cudaSuccess;
}
template <typename T, int NT, int CL>
cudaError_t go_long(const LossArg& a, cudaStream_t stream) {
  const size_t smem = long_smem<T>(a.r.row_len, CL);
  const uint32_t seg = uint32_t(smem / 16 - 4);
  cudaLaunchConfig_t cfg{};
  const uint64_t ctas = uint64_t(a.r.rows) * CL;
  if (ctas > 0x7fffffffu) return cudaErrorInvalidConfiguration;
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CL;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CL > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, k_policy_long<T, NT, CL>, a, seg);
}
template <typename T>
inline cudaError_t whole_as(const LossArg& a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const uint64_t need = a.r.row_len + V - 1;
  if (need <= 256) return go_warps(k_policy_whole<T, 8 / V>, a, s);
  if (need <= 512) return go_warps(k_policy_whole<T, 16 / V>, a, s);
  if (need <= 1024) return go_warps(k_policy_whole<T, 32 / V>, a, s);
  if (need * sizeof(T) <= kSmall) return go_long<T, 64, 1>(a, s);
  if (need * sizeof(T) <= kShort) return go_long<T, 128, 1>(a, s);
  if (need * sizeof(T) <= kLong) return go_long<T, 256, 1>(a, s);
  return go_long<T, 512, 8>(a, s);
}
template <typename T>
inline cudaError_t draw_as(const DrawArg& a, int sms, cudaStream_t s) {
  return cut_as<T>(a, sms, s);
}
template <typename T>
inline cudaError_t loss_as(const LossArg& a, int sms, cudaStream_t s) {
  const CutArg& c = a.c;
  if (!c.top_k && !c.row_top_k && !(c.top_p < 1.0f) && !c.row_top_p && !(c.min_p > 0.0f) && !c.row_min_p)
    return whole_as<T>(a, s);
  return cut_as<T>(a, sms, s);
}

}  // namespace pol
}  // namespace kc
