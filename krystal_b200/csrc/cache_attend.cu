// cache_attend.cu — attention and pointer scores of questions over the bank cache.
#include <algorithm>

#include "cache.cuh"

namespace kc {
namespace cache {
namespace {

constexpr int kWarps = 8;

// The sequence of question `row`, and the question's number there and their
// number; false where the row is not a question of the call.
__device__ __forceinline__ bool asker(const Table& t, const Ask& a, uint32_t row, uint32_t* seq, uint32_t* nth, uint32_t* count) {
  if (a.off) {
    if (row < a.off[0] || row >= a.off[t.seqs]) return false;
    *seq = owner_of(a.off, t.seqs, row);
    *nth = uint32_t(row - a.off[*seq]);
    *count = uint32_t(a.off[*seq + 1] - a.off[*seq]);
  } else {
    if (row >= t.seqs) return false;
    *seq = row;
    *nth = 0;
    *count = 1;
  }
  return true;
}

// q . k of one cached key (a lane each), f32.
template <int D, int FMT>
__device__ __forceinline__ float dot(const float* q, const uint8_t* keys, uint32_t r) {
  float s = 0.0f;
#pragma unroll 4
  for (int b = 0; b < D; b += 4) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(keys + key_at<D>(r, b));
#pragma unroll
    for (int i = 0; i < 4; i++) s = fmaf(q[b + i], decode<FMT>((w >> (8 * i)) & 0xffu), s);
  }
  return s;
}

// One warp a question and head: a cell of 32 keys at a time, a lane a key; the
// running maximum and sum of its softmax; then the cell's values, D / 32
// dimensions a lane.
template <typename T, int D, int FMT>
__global__ __launch_bounds__(kWarps * 32) void k_attend(AttendArg a) {
  constexpr int E = D / 32;
  __shared__ float s_q[kWarps][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t item = uint64_t(blockIdx.x) * kWarps + warp;
  const uint32_t row = uint32_t(item / a.a.heads), head = uint32_t(item % a.a.heads), kv = head / (a.a.heads / a.c.heads);
  uint32_t seq, nth, count;
  if (row >= a.a.questions || !asker(a.t, a.a, row, &seq, &nth, &count)) return;
  for (int i = lane; i < D; i += 32)
    s_q[warp][i] = to_f32(static_cast<const T*>(a.a.q)[row * a.a.pitch + head * uint64_t(D) + i]) * a.scale;
  __syncwarp();
  const uint32_t len = length_of(a.t, seq), n = (len + kPage - 1) / kPage;
  const float* mask = nullptr;
  uint64_t stride = 0;
  if (a.mask) {
    stride = (a.mask_off[seq + 1] - a.mask_off[seq]) / count;
    mask = a.mask + a.mask_off[seq] + nth * stride;
  }
  const uint32_t* list = a.blocks ? a.blocks + (uint64_t(row) * a.c.heads + kv) * a.block_count : nullptr;
  const uint32_t todo = list ? a.block_count : n;
  float m = -INFINITY, l = 0.0f, o[E] = {};
  for (uint32_t i = 0; i < todo; i++) {
    const uint32_t b = list ? list[i] : i;
    if (b >= n) continue;
    const uint32_t page = a.t.table[uint64_t(seq) * a.t.pitch + b];
    if (page >= a.c.pages) continue;
    for (uint32_t half = 0; half < 2; half++) {
      const uint8_t* cell = cell_of<D>(a.c, page, kv, half);
      const float* scales = reinterpret_cast<const float*>(cell + 2 * kCell * D);
      const uint64_t pos = uint64_t(b) * kPage + half * kCell + lane;
      float s = -INFINITY, vs = 0.0f;
      if (pos < len && (!mask || pos < stride)) {
        const float bias = mask ? mask[pos] : 0.0f;
        if (bias > kBlocked) s = dot<D, FMT>(s_q[warp], cell, lane) * scales[lane] + fminf(bias, -kBlocked);
        vs = scales[kCell + lane];
      }
      float top = s;
#pragma unroll
      for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
      if (top == -INFINITY) continue;
      const float next = fmaxf(m, top), keep = expf(m - next), p = expf(s - next);
      float sum = p;
#pragma unroll
      for (int k = 16; k; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
      l = l * keep + sum;
      m = next;
#pragma unroll
      for (int e = 0; e < E; e++) o[e] *= keep;
      for (int j = 0; j < 32; j++) {
        const float w = __shfl_sync(0xffffffffu, p * vs, j);
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = fmaf(w, decode<FMT>(cell[kCell * D + value_at<D>(j, lane + 32 * e)]), o[e]);
      }
    }
  }
  T* out = static_cast<T*>(a.out) + row * a.out_pitch + head * uint64_t(D);
#pragma unroll
  for (int e = 0; e < E; e++) out[lane + 32 * e] = from_f32<T>(l > 0.0f ? o[e] / l : 0.0f);
  if (a.lse && lane == 0) a.lse[uint64_t(row) * a.a.heads + head] = l > 0.0f ? m + logf(l) : -INFINITY;
}

// One warp a question: its scores, a lane a key.
template <typename T, int D, int FMT>
__global__ __launch_bounds__(kWarps * 32) void k_scores(ScoreArg a) {
  __shared__ float s_q[kWarps][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t row = blockIdx.x * kWarps + warp;
  uint32_t seq, nth, count;
  if (row >= a.a.questions || !asker(a.t, a.a, row, &seq, &nth, &count)) return;
  for (int i = lane; i < D; i += 32) s_q[warp][i] = to_f32(static_cast<const T*>(a.a.q)[row * a.a.pitch + i]) * a.scale;
  __syncwarp();
  const uint32_t len = length_of(a.t, seq);
  const uint64_t stride = (a.off[seq + 1] - a.off[seq]) / count, at = a.off[seq] + nth * stride;
  for (uint64_t pos = lane; pos < stride; pos += 32) {
    float s = kShut;
    if (pos < len) {
      const uint32_t page = a.t.table[uint64_t(seq) * a.t.pitch + pos / kPage];
      const float bias = a.mask ? a.mask[at + pos] : 0.0f;
      if (page < a.c.pages && bias > kBlocked) {
        const uint8_t* cell = cell_of<D>(a.c, page, 0, uint32_t(pos % kPage) / kCell);
        const uint32_t r = uint32_t(pos % kCell);
        s = dot<D, FMT>(s_q[warp], cell, r) * reinterpret_cast<const float*>(cell + 2 * kCell * D)[r] + fminf(bias, -kBlocked);
      }
    }
    a.scores[at + pos] = s;
  }
}

template <typename T, int D>
void attend_as(const AttendArg& a, unsigned grid, cudaStream_t s) {
  if (a.c.format == kI8) k_attend<T, D, kI8><<<grid, kWarps * 32, 0, s>>>(a);
  else k_attend<T, D, kE4M3><<<grid, kWarps * 32, 0, s>>>(a);
}
template <typename T, int D>
void scores_as(const ScoreArg& a, unsigned grid, cudaStream_t s) {
  if (a.c.format == kI8) k_scores<T, D, kI8><<<grid, kWarps * 32, 0, s>>>(a);
  else k_scores<T, D, kE4M3><<<grid, kWarps * 32, 0, s>>>(a);
}
template <typename T>
void attend_dim(const AttendArg& a, unsigned grid, cudaStream_t s) {
  a.c.dim == 32 ? attend_as<T, 32>(a, grid, s) : a.c.dim == 64 ? attend_as<T, 64>(a, grid, s) : attend_as<T, 128>(a, grid, s);
}
template <typename T>
void scores_dim(const ScoreArg& a, unsigned grid, cudaStream_t s) {
  a.c.dim == 32 ? scores_as<T, 32>(a, grid, s) : a.c.dim == 64 ? scores_as<T, 64>(a, grid, s) : scores_as<T, 128>(a, grid, s);
}

}  // namespace

uint64_t plan_attend(AttendArg& a, int) {
  a.splits = 1;
  a.chunk = (a.t.max_len + kPage - 1) / kPage;
  return 0;
}

cudaError_t launch_attend(const AttendArg& a, int, cudaStream_t s, uint64_t* launches) {
  if (a.a.questions == 0 || a.t.seqs == 0) return cudaSuccess;
  const unsigned grid = unsigned((uint64_t(a.a.questions) * a.a.heads + kWarps - 1) / kWarps);
  ++*launches;
  a.a.dtype == kF32 ? attend_dim<float>(a, grid, s) : a.a.dtype == kF16 ? attend_dim<__half>(a, grid, s) : attend_dim<__nv_bfloat16>(a, grid, s);
  return cudaGetLastError();
}

cudaError_t launch_scores(const ScoreArg& a, int, cudaStream_t s, uint64_t* launches) {
  if (a.a.questions == 0 || a.t.seqs == 0) return cudaSuccess;
  const unsigned grid = (a.a.questions + kWarps - 1) / kWarps;
  ++*launches;
  a.a.dtype == kF32 ? scores_dim<float>(a, grid, s) : a.a.dtype == kF16 ? scores_dim<__half>(a, grid, s) : scores_dim<__nv_bfloat16>(a, grid, s);
  return cudaGetLastError();
}

}  // namespace cache
}  // namespace kc
