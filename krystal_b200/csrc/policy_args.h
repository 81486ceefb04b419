// policy_args.h — the arguments of the policy and gradient-clipping kernels and
// their launchers (policy.cu), which krystal_cuda.cu calls for the C ABI.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace kc {

// The element types of the rows and gradients (KC_DTYPE_* of the C ABI).
constexpr int kF32 = 0, kF16 = 1, kBF16 = 2, kF64 = 3;

namespace pol {

constexpr int kKindScores = 0, kKindP = 1;
constexpr uint32_t kNone = 0xffffffffu;
constexpr uint32_t kMaxRow = 262128;  // 8 CTAs of 32768 entries, less a row's two misaligned vectors

struct RowsArg {
  const void* values;
  const uint64_t *q_off, *p_off;  // ragged frames; q_off null: one row a frame
  uint32_t rows, frames;          // frames 0: dense
  uint64_t row_len, pitch;        // dense row length (ragged: longest row allowed), dense pitch
  int kind;
};

struct CutArg {
  double inv_temperature;  // 1 / temperature, 0 at 0
  float temperature;
  uint32_t top_k;
  float top_p, min_p;
  const float* row_temperature;
  const uint32_t* row_top_k;
  const float *row_top_p, *row_min_p;
};

struct DrawArg {
  RowsArg r;
  CutArg c;
  const double* uniforms;
  uint32_t *index, *kept;
  float *logp, *p;
  uint64_t out_pitch;
};

struct LossArg {
  RowsArg r;
  CutArg c;
  const uint32_t* actions;
  const float *advantage, *row_weight;
  float beta;
  float *loss, *logp, *entropy;
  void* grad;
  uint64_t out_pitch;
};

// By element type (policy_f32.cu, policy_f16.cu, policy_bf16.cu).
cudaError_t draw_f32(const DrawArg& a, int sms, cudaStream_t s);
cudaError_t draw_f16(const DrawArg& a, int sms, cudaStream_t s);
cudaError_t draw_bf16(const DrawArg& a, int sms, cudaStream_t s);
cudaError_t loss_f32(const LossArg& a, int sms, cudaStream_t s);
cudaError_t loss_f16(const LossArg& a, int sms, cudaStream_t s);
cudaError_t loss_bf16(const LossArg& a, int sms, cudaStream_t s);

cudaError_t prepare_f32();
cudaError_t prepare_f16();
cudaError_t prepare_bf16();

// What the kernels need once on each device (the current one).
cudaError_t prepare();

// One launch each on `stream`; *launches counts it.
cudaError_t launch_draw(const DrawArg& a, int dtype, int sms, cudaStream_t stream, uint64_t* launches);
cudaError_t launch_policy_loss(const LossArg& a, int dtype, int sms, cudaStream_t stream, uint64_t* launches);

}  // namespace pol

namespace clip {

struct Tensor {
  const void* in;
  void* out;        // null: counted in the norm alone
  uint64_t n;
  double weight;    // the tensor's factor in the norm
  int32_t dtype;
  uint32_t chunk0;  // its first chunk of the launch
};

// Tensors a launch: its table travels in the kernel's parameters, a short one
// for few tensors (30 KB of parameters cost a launch about 2 us more).
constexpr uint32_t kTable = 768, kShortTable = 48;
constexpr uint32_t kMaxCtas = 1184;   // partial sums a norm launch writes (148 SMs x 8 CTAs)

// Doubles of workspace that `count` tensors need.
inline uint64_t workspace_doubles(uint64_t count) { return (count + kTable - 1) / kTable * kMaxCtas; }

// The norm of every tensor's weighted elements and, where out is set, the
// scaled copy; result [2]: norm, scale. t[].chunk0 is filled in here.
cudaError_t launch_clip(Tensor* t, uint64_t count, double max_norm, double* workspace, double* result, int sms,
                        cudaStream_t stream, uint64_t* launches);

}  // namespace clip
}  // namespace kc
