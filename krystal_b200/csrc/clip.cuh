// clip.cuh — the global norm of many gradient tensors, and clipping by it:
// norm = sqrt(sum_t weight_t^2 sum_i g_ti^2), scale = min(1, max_norm / norm)
// (1 where the norm is not finite: what follows sees the gradients as they
// are), out_ti = g_ti * scale: f64 elements by the f64 scale, the others by the
// scale rounded to f32 and the product to the type (two half steps, and no f64
// conversions, which would bound the pass). A scale near f32's smallest numbers
// multiplies in 64 bits.
//
// Two launches: k_norm leaves one partial sum a CTA, k_scale adds the partial
// sums again in every CTA (a few KB from L2) and scales. Lists of more tensors
// than a launch's table holds take several of each, and one CTA (k_join) adds
// the partial sums of them all once. All sums are 64-bit
// and in an order that the sizes alone decide; there are no atomics. The work
// is cut into chunks of one tensor, 8 to 128 KB so that about one falls to each
// CTA of a small list and a large one pays for few searches of its table; CTA b
// takes chunks b, b + grid, ... and k_scale takes them from the last back, so
// that what k_norm read last is still in L2. k_scale is launched while k_norm
// runs and waits for it on the device.
//
// Bound by HBM: 301 mixed tensors of 200 M elements (510 MB in) take 275 us, of
// which k_norm's one read runs at 5.4 TB/s (83 % of the measured copy rate) and
// k_scale's read and write at 5.8. Small lists (25 tensors, 1.7 M elements)
// take 10 us, the host's two launches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "policy_args.h"

namespace kc {
namespace clip {

constexpr int kThreads = 512;
constexpr uint32_t kMinChunk = 8192, kMaxChunk = 131072;  // bytes

template <uint32_t N>
struct Table {
  Tensor t[N];
  uint32_t count, chunks, chunk_bytes;
};

__host__ __device__ constexpr uint32_t dtype_bytes(int d) { return d == kF32 ? 4u : d == kF64 ? 8u : 2u; }

struct Piece {
  const Tensor* t;
  uint64_t first;  // element
  uint32_t n;      // elements
};

template <uint32_t N>
__device__ __forceinline__ Piece piece_of(const Table<N>& tb, uint32_t chunk) {
  uint32_t lo = 0, hi = tb.count;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (tb.t[mid].chunk0 <= chunk) lo = mid; else hi = mid;
  }
  Piece p;
  p.t = &tb.t[lo];
  const uint32_t per = tb.chunk_bytes / dtype_bytes(p.t->dtype);
  p.first = uint64_t(chunk - p.t->chunk0) * per;
  p.n = uint32_t(min(uint64_t(per), p.t->n - p.first));
  return p;
}

__device__ __forceinline__ double wide(float v) { return double(v); }
__device__ __forceinline__ double wide(double v) { return v; }
__device__ __forceinline__ double wide(__half v) { return double(__half2float(v)); }
__device__ __forceinline__ double wide(__nv_bfloat16 v) { return double(__bfloat162float(v)); }
__device__ __forceinline__ float scaled(float v, double s) { return v * float(s); }
__device__ __forceinline__ double scaled(double v, double s) { return v * s; }
__device__ __forceinline__ __half scaled(__half v, double s) { return __float2half_rn(__half2float(v) * float(s)); }
__device__ __forceinline__ __nv_bfloat16 scaled(__nv_bfloat16 v, double s) {
  return __float2bfloat16_rn(__bfloat162float(v) * float(s));
}

// The same by a scale too small for f32.
constexpr double kSmallScale = 1e-30;
__device__ __forceinline__ void scale64(float& v, double s) { v = float(double(v) * s); }
__device__ __forceinline__ void scale64(double& v, double s) { v *= s; }
__device__ __forceinline__ void scale64(__half& v, double s) { v = __double2half(wide(v) * s); }
__device__ __forceinline__ void scale64(__nv_bfloat16& v, double s) { v = __double2bfloat16(wide(v) * s); }

// Elements of a piece ahead of its first 16-byte boundary.
template <typename T>
__device__ __forceinline__ uint32_t head_of(const T* p, uint32_t n) {
  const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(p) & 15);
  return min(n, off ? uint32_t((16 - off) / sizeof(T)) : 0u);
}

template <typename T>
__device__ __forceinline__ double square_sum(const T* in, uint32_t n) {
  constexpr int V = 16 / int(sizeof(T));
  const uint32_t head = head_of(in, n), vecs = (n - head) / V;
  double acc[2] = {0.0, 0.0};
  const uint4* src = reinterpret_cast<const uint4*>(in + head);
#pragma unroll 8
  for (uint32_t i = threadIdx.x; i < vecs; i += kThreads) {
    const uint4 raw = src[i];
    alignas(16) T v[V];
    *reinterpret_cast<uint4*>(v) = raw;
#pragma unroll
    for (int e = 0; e < V; e++) {
      const double d = wide(v[e]);
      acc[e & 1] = fma(d, d, acc[e & 1]);
    }
  }
  const uint32_t loose = n - vecs * V;  // the head, then the tail
  for (uint32_t i = threadIdx.x; i < loose; i += kThreads) {
    const double d = wide(in[i < head ? i : i + vecs * V]);
    acc[0] = fma(d, d, acc[0]);
  }
  return acc[0] + acc[1];
}

template <typename T>
__device__ __forceinline__ void scale_piece(const T* in, T* out, uint32_t n, double scale) {
  constexpr int V = 16 / int(sizeof(T));
  if (scale < kSmallScale && scale > 0.0) {
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      T v = in[i];
      scale64(v, scale);
      out[i] = v;
    }
    return;
  }
  if ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) {
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) out[i] = scaled(in[i], scale);
    return;
  }
  const uint32_t head = head_of(in, n), vecs = (n - head) / V;
  const uint4* src = reinterpret_cast<const uint4*>(in + head);
  uint4* dst = reinterpret_cast<uint4*>(out + head);
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < vecs; i += kThreads) {
    alignas(16) T v[V];
    *reinterpret_cast<uint4*>(v) = src[i];
#pragma unroll
    for (int e = 0; e < V; e++) v[e] = scaled(v[e], scale);
    dst[i] = *reinterpret_cast<uint4*>(v);
  }
  const uint32_t loose = n - vecs * V;
  for (uint32_t i = threadIdx.x; i < loose; i += kThreads) {
    const uint32_t at = i < head ? i : i + vecs * V;
    out[at] = scaled(in[at], scale);
  }
}

// The CTA's sum, in thread order by warps; valid in every thread.
__device__ __forceinline__ double cta_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  v = lane < kThreads / 32 ? red[lane] : 0.0;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <uint32_t N>
__global__ void __launch_bounds__(kThreads) k_norm(const __grid_constant__ Table<N> tb, double* __restrict__ partial) {
  __shared__ double red[kThreads / 32];
  cudaTriggerProgrammaticLaunchCompletion();
  double sum = 0.0;
  for (uint32_t c = blockIdx.x; c < tb.chunks; c += gridDim.x) {
    const Piece p = piece_of(tb, c);
    double s = 0.0;
    switch (p.t->dtype) {
      case kF32: s = square_sum(static_cast<const float*>(p.t->in) + p.first, p.n); break;
      case kF16: s = square_sum(static_cast<const __half*>(p.t->in) + p.first, p.n); break;
      case kBF16: s = square_sum(static_cast<const __nv_bfloat16*>(p.t->in) + p.first, p.n); break;
      default: s = square_sum(static_cast<const double*>(p.t->in) + p.first, p.n); break;
    }
    sum = fma(p.t->weight * p.t->weight, s, sum);
  }
  sum = cta_sum(sum, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// Every thread of the CTA adds the partial sums and gets norm and scale.
struct Clip {
  double norm, scale;
};
__device__ __forceinline__ Clip join(const double* partial, uint32_t partials, double max_norm, double* red) {
  double sum = 0.0;
  // (written while k_scale runs, so neither read-only data nor read ahead of its wait: from L2)
  for (uint32_t i = threadIdx.x; i < partials; i += kThreads) sum += __ldcg(partial + i);
  const double norm = sqrt(cta_sum(sum, red));
  return Clip{norm, norm > max_norm && norm <= 1.7976931348623157e308 ? max_norm / norm : 1.0};
}

// The norm and scale of a list of several launches, whose scaling launches
// would otherwise add up all of the list's partial sums in each of their CTAs.
static __global__ void __launch_bounds__(kThreads) k_join(const double* partial, uint32_t partials, double max_norm,
                                                          double* __restrict__ result) {
  __shared__ double red[kThreads / 32];
  const Clip c = join(partial, partials, max_norm, red);
  if (threadIdx.x == 0) {
    result[0] = c.norm;
    result[1] = c.scale;
  }
}

// partials 0: k_join has written the result.
template <uint32_t N>
__global__ void __launch_bounds__(kThreads) k_scale(const __grid_constant__ Table<N> tb, const double* partial,
                                                    uint32_t partials, double max_norm, double* result) {
  __shared__ double red[kThreads / 32];
  double scale;
  if (partials) {
    cudaGridDependencySynchronize();  // k_norm has ended and its partial sums are here
    const Clip c = join(partial, partials, max_norm, red);
    scale = c.scale;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      result[0] = c.norm;
      result[1] = scale;
    }
  } else {
    scale = result[1];
  }
  const bool cut = scale != 1.0;
  for (uint32_t r = blockIdx.x; r < tb.chunks; r += gridDim.x) {
    const Piece p = piece_of(tb, tb.chunks - 1 - r);
    if (!p.t->out || (!cut && p.t->out == p.t->in)) continue;
    switch (p.t->dtype) {
      case kF32:
        scale_piece(static_cast<const float*>(p.t->in) + p.first, static_cast<float*>(p.t->out) + p.first, p.n, scale);
        break;
      case kF16:
        scale_piece(static_cast<const __half*>(p.t->in) + p.first, static_cast<__half*>(p.t->out) + p.first, p.n,
                    scale);
        break;
      case kBF16:
        scale_piece(static_cast<const __nv_bfloat16*>(p.t->in) + p.first,
                    static_cast<__nv_bfloat16*>(p.t->out) + p.first, p.n, scale);
        break;
      default:
        scale_piece(static_cast<const double*>(p.t->in) + p.first, static_cast<double*>(p.t->out) + p.first, p.n,
                    scale);
        break;
    }
  }
}

}  // namespace clip
}  // namespace kc
