// cache.cuh — what the bank cache's kernels share: where a row's bytes lie in a
// cell, the value of a code, the types of rows and questions.
//
// Quantising. A row of a head x [dim] is stored as 8-bit codes and one f32 scale:
//   scale = max(f32(max |x| / top), 2^-100),  code = round(f32(x / scale)),
// top = 127 for i8 (stored as code + 128) and 448 for e4m3, halves to the even.
// The stored value is f32(code * scale). NaN counts as 0 and magnitudes beyond
// 2^127 as 2^127, so that everything in a cache is finite; the floor of the scale
// keeps its reciprocal and its logarithm finite (rows below 127 * 2^-100 lose
// digits, no others).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cache_args.h"
#include "policy_args.h"

namespace kc {
namespace cache {

constexpr float kTopI8 = 127.0f, kTopE4M3 = 448.0f;
constexpr float kLeastScale = 7.888609052210118e-31f;   // 2^-100
constexpr float kMostValue = 1.7014118346046923e38f;    // 2^127

// Where byte b of row r of a cell's keys lies. Rows are in order; at dim 128 the
// two 64-byte halves of rows 4..7 of every 8 change places, so that the two rows
// (a, a + 4) whose 16-byte pieces a quarter-warp reads together fall on different
// banks. At 32 and 64 dims consecutive lanes read consecutive bytes already.
template <int D>
__device__ __forceinline__ uint32_t key_at(uint32_t r, uint32_t b) {
  return r * D + (D == 128 ? b ^ (((r >> 2) & 1u) << 6) : b);
}

// The same for the values, whose four rows (a .. a + 3) are read together in
// 32-byte pieces: they change places by the row's number.
template <int D>
__device__ __forceinline__ uint32_t value_at(uint32_t r, uint32_t b) {
  return r * D + (D == 128 ? b ^ ((r & 3u) << 5) : D == 64 ? b ^ (((r >> 1) & 1u) << 5) : b);
}

template <int D>
__device__ __forceinline__ uint8_t* cell_of(const Store& c, uint32_t page, uint32_t head, uint32_t half) {
  return c.cells + ((uint64_t(page) * c.heads + head) * 2 + half) * cell_bytes(D);
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ float tame(float x) {
  return x != x ? 0.0f : fminf(fmaxf(x, -kMostValue), kMostValue);
}

constexpr float kPlainScale = 8.673617379884035e-19f;  // 2^-60: remainders of x / scale stay in f32's range above it

// The values over their scale of a word of four codes.
template <int FMT>
__device__ __forceinline__ void values_of(uint32_t w, float (&v)[4]) {
  if (FMT == kI8) {
    // 0x4b000000 + byte is 2^23 + byte
#pragma unroll
    for (int i = 0; i < 4; i++)
      v[i] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + i)) - 8388736.0f;
  } else {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      uint32_t h;
      const unsigned short x = static_cast<unsigned short>(i ? w >> 16 : w);
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(x));
      const __half2 y = *reinterpret_cast<const __half2*>(&h);
      v[2 * i] = __low2float(y);
      v[2 * i + 1] = __high2float(y);
    }
  }
}

// Rows that sequence s holds.
__device__ __forceinline__ uint32_t length_of(const Table& t, uint32_t s) {
  const uint32_t n = t.lengths[s];
  return n < t.max_len ? n : t.max_len;
}

// The last s with off[s] <= i (off ascending, off[0] <= i), by a whole warp: 32
// places are looked at together, so that a thousand sequences take two trips to
// memory, not ten.
__device__ __forceinline__ uint32_t owner_of(const uint64_t* off, uint32_t n, uint64_t i) {
  const uint32_t lane = threadIdx.x & 31;
  uint32_t lo = 0, hi = n;  // off[lo] <= i < off[hi], or hi = n
  while (hi - lo > 1) {
    const uint32_t step = (hi - lo + 32) / 33;  // lane k looks at lo + (k + 1) step
    const uint64_t at = uint64_t(lo) + uint64_t(lane + 1) * step;
    const uint32_t under = __popc(__ballot_sync(0xffffffffu, at < hi && off[at < hi ? at : lo] <= i));
    const uint64_t top = uint64_t(lo) + uint64_t(under + 1) * step;
    if (top < hi) hi = uint32_t(top);
    lo += under * step;
  }
  return lo;
}

}  // namespace cache
}  // namespace kc
