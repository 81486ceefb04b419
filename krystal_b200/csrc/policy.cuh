// policy.cuh — what a host does with the rows of scores or probabilities a
// selection leaves: draw an answer from a tempered and cut distribution, and
// take the loss of drawn answers with its gradient.
// The selector itself draws from the whole softmax (sampleRow, forward/
// sampling.ts:41-57); the cuts have no counterpart in the reference.
//
// One row v_0 .. v_{n-1}. An entry is open unless it is NaN, a score at or
// below -1e29 (f16: also the type's lowest value) or a probability that is
// not above 0. With m the largest open value and T the temperature,
//
//   x_j = (v_j - m) / T          (probabilities: (log v_j - log m) / T)
//   w_j = e^{x_j}                (probabilities at T = 1: v_j itself)
//
// and then, in this order, top-k keeps the k largest, top-p the shortest
// prefix in descending order whose mass reaches top_p of what top-k left,
// min-p the entries with w_j >= min_p * max w (ties always to the lowest
// index); entries with x_j < -700 cannot be drawn and are dropped. pi_j =
// w_j / Z over what is kept.
//
// Which entries are kept, and which one a uniform hits, are decisions: they
// are taken from 64-bit weights summed in a fixed order, so a row's answer
// does not depend on how the row was split, and equals the definition's to
// about n * 1e-15 of probability. No entry is sorted: a cut is the largest
// value t with count(v >= t) >= k, or mass(v >= t) >= top_p * total, found by
// halving the range of values between snapped row entries, or in a short list
// by adding up, for each entry, what lies ahead of it.
//
// This file: layouts, arithmetic and reductions; policy_cut.cuh: the rows with
// cuts and the draws; policy_whole.cuh: the loss where nothing is cut.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "policy_args.h"

namespace kc {
namespace pol {

constexpr double kDropped = -700.0;  // e^x stays a normal number above it

template <typename T> struct Lowest { static constexpr float open_above = -1e29f; };
template <> struct Lowest<__half> { static constexpr float open_above = -65504.0f; };

__device__ __forceinline__ float as_f32(float v) { return v; }
__device__ __forceinline__ float as_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// f32 values as u32 keys in the same order; 0 is kept for "not in the row's
// support" (no finite value maps to it).
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 joins +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}

// The key of a row's value, 0 where it is not open.
template <typename T>
__device__ __forceinline__ uint32_t open_key(float f, int kind) {
  const bool open = kind == kKindP ? f > 0.0f : f > Lowest<T>::open_above;
  return open ? key_of(fminf(f, 3.402823466e38f)) : 0u;
}

// e^x for -700 <= x <= 0 in 64 bits, by a table of 2^{i/32} (Tang, "Table-
// driven implementation of the exponential function", ACM TOMS 15(2), 1989):
// x = (32 q + i) ln2/32 + r, |r| <= ln2/64, and e^r by its Taylor polynomial
// of degree 5 (the first term left out is below 3e-15). Lane i holds 2^{i/32}
// and the lanes fetch each other's by a shuffle, so every lane of the warp
// calls this together.
__device__ __forceinline__ double exp64(double x, double tab) {
  constexpr double kBig = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
  const double t = fma(x, 46.166241308446828384, kBig);  // 32 / ln 2
  const int n = __double2loint(t);
  const double r = fma(t - kBig, -0.021660849392498290195, x);  // ln 2 / 32
  double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
  p = fma(r, p, 1.0 / 6.0);
  p = fma(r, p, 0.5);
  p = fma(r, p, 1.0);
  p = fma(r, p, 1.0);
  const double s = __shfl_sync(0xffffffffu, tab, n & 31) * p;
  return __hiloint2double(__double2hiint(s) + ((n >> 5) << 20), __double2loint(s));
}

// log v in 64 bits for a positive f32 v, by a table of 32 mantissa intervals
// (Tang, "Table-driven implementation of the logarithm function", ACM TOMS
// 16(4), 1990): v = 2^e m, c_i = 1 / (the middle of m's interval), r = m c_i - 1,
// |r| <= 1/65, log v = e ln 2 - log c_i + log(1 + r) by its series to r^8
// (the first term left out is below 6e-18). Lane i holds c_i and -log c_i;
// every lane of the warp calls this together.
__device__ __forceinline__ double log_tab(float v, double c, double neg_log_c) {
  const double d = double(v);
  const int hi = __double2hiint(d);
  const int i = (hi >> 15) & 31;
  const double m = __hiloint2double((hi & 0xfffff) | 0x3ff00000, __double2loint(d));
  const double ci = __shfl_sync(0xffffffffu, c, i), li = __shfl_sync(0xffffffffu, neg_log_c, i);
  const double r = fma(m, ci, -1.0);
  double p = fma(r, -1.0 / 8.0, 1.0 / 7.0);
  p = fma(r, p, -1.0 / 6.0);
  p = fma(r, p, 1.0 / 5.0);
  p = fma(r, p, -1.0 / 4.0);
  p = fma(r, p, 1.0 / 3.0);
  p = fma(r, p, -0.5);
  p = fma(r, p, 1.0);
  return fma(double((hi >> 20) - 1023), 0.69314718055994530942, fma(r, p, li));
}

// A lane's share of the two tables.
struct Tables {
  double e2, c, l;  // 2^{lane/32}; log_tab's c_i and -log c_i (needs_log only)
  __device__ Tables(int lane, bool needs_log);
};

// One logarithm a row or two, out of line.
static __device__ __noinline__ double log64(double v) { return log(v); }

__device__ __forceinline__ Tables::Tables(int lane, bool needs_log)
    : e2(exp2(double(lane) * (1.0 / 32.0))), c(1.0 / (1.0 + (lane + 0.5) * (1.0 / 32.0))), l(0.0) {
  if (needs_log) l = -log64(c);
}

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float log2_fast(float v) {
  float r;
  asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ float rcp_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ double warp_add(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Inclusive prefix over the lanes.
__device__ __forceinline__ double warp_scan(double v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}
__device__ __forceinline__ uint32_t warp_scan(uint32_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// Reductions over a row's group of W warps in each of CL CTAs. Every thread
// of the group calls each of them the same number of times; sums add the
// warps, then the CTAs, in order. The slots alternate between two buffers, so
// one barrier a reduction is enough: a slot is written again only after the
// next reduction's barrier, which every reader of it has passed.
template <int W, int CL>
struct Group {
  struct Shared {
    double d[2][W > 1 ? W : 1];
    uint32_t u[2][3][W > 1 ? W : 1];
    float2 f[2][W > 1 ? W : 1];
    float2 cf[2][CL];
    double cd[2][CL];
    uint32_t cu[2][3][CL];
  };
  Shared* s;
  int lane, warp, rank, buf;

  // One warp shares nothing.
  __device__ explicit Group(int l) : s(nullptr), lane(l), warp(0), rank(0), buf(0) {
    static_assert(W == 1 && CL == 1, "a group of several warps needs shared memory");
  }
  __device__ Group(Shared& sh, int l, int w) : s(&sh), lane(l), warp(w), rank(0), buf(0) {
    if constexpr (CL > 1) {
      rank = int(cooperative_groups::this_cluster().block_rank());
      cooperative_groups::this_cluster().sync();  // a CTA's shared memory is written once it runs
    }
  }
  __device__ int segment() const { return rank * W + warp; }

  // (sum, min, max) of three values at once
  __device__ void counts(uint32_t& add, uint32_t& mn, uint32_t& mx) {
    add = __reduce_add_sync(0xffffffffu, add);
    mn = __reduce_min_sync(0xffffffffu, mn);
    mx = __reduce_max_sync(0xffffffffu, mx);
    if constexpr (W > 1) {
      buf ^= 1;
      if (lane == 0) { s->u[buf][0][warp] = add; s->u[buf][1][warp] = mn; s->u[buf][2][warp] = mx; }
      __syncthreads();
      const bool in = lane < W;
      add = __reduce_add_sync(0xffffffffu, in ? s->u[buf][0][lane] : 0u);
      mn = __reduce_min_sync(0xffffffffu, in ? s->u[buf][1][lane] : 0xffffffffu);
      mx = __reduce_max_sync(0xffffffffu, in ? s->u[buf][2][lane] : 0u);
    }
    if constexpr (CL > 1) {
      namespace cg = cooperative_groups;
      cg::cluster_group cl = cg::this_cluster();
      if (warp == 0 && lane < CL) {
        uint32_t* dst = cl.map_shared_rank(&s->cu[0][0][0], lane) + buf * 3 * CL;
        dst[rank] = add; dst[CL + rank] = mn; dst[2 * CL + rank] = mx;
      }
      cl.sync();
      const bool in = lane < CL;
      add = __reduce_add_sync(0xffffffffu, in ? s->cu[buf][0][lane] : 0u);
      mn = __reduce_min_sync(0xffffffffu, in ? s->cu[buf][1][lane] : 0xffffffffu);
      mx = __reduce_max_sync(0xffffffffu, in ? s->cu[buf][2][lane] : 0u);
    }
  }
  // The group's sum of one value a thread.
  __device__ double sum(double v) {
    v = warp_add(v);
    if constexpr (W > 1) {
      buf ^= 1;
      if (lane == 0) s->d[buf][warp] = v;
      __syncthreads();
      v = __shfl_sync(0xffffffffu, warp_scan(lane < W ? s->d[buf][lane] : 0.0, lane), W - 1);
    }
    if constexpr (CL > 1) {
      namespace cg = cooperative_groups;
      cg::cluster_group cl = cg::this_cluster();
      if (warp == 0 && lane < CL) cl.map_shared_rank(&s->cd[0][0], lane)[buf * CL + rank] = v;
      cl.sync();
      v = __shfl_sync(0xffffffffu, warp_scan(lane < CL ? s->cd[buf][lane] : 0.0, lane), CL - 1);
    }
    return v;
  }
  // The same, with the sums up to this warp's values in bank order and through
  // them. Added one after another, so that one warp's `through` is the next
  // one's `before` to the last bit, and equal to its own `before` where the
  // warp adds nothing: whatever lies below the sum lies in exactly one warp.
  __device__ double prefix(double v, double& before, double& through) {
    v = warp_add(v);
    before = through = 0.0;
    if constexpr (W > 1) {
      buf ^= 1;
      if (lane == 0) s->d[buf][warp] = v;
      __syncthreads();
      v = 0.0;
#pragma unroll
      for (int j = 0; j < W; j++) {
        if (j == warp) before = v;
        v += s->d[buf][j];
        if (j == warp) through = v;
      }
    }
    if constexpr (CL > 1) {
      namespace cg = cooperative_groups;
      cg::cluster_group cl = cg::this_cluster();
      if (warp == 0 && lane < CL) cl.map_shared_rank(&s->cd[0][0], lane)[buf * CL + rank] = v;
      cl.sync();
      double ahead = v = 0.0;
#pragma unroll
      for (int j = 0; j < CL; j++) {
        if (j == rank) ahead = v;
        v += s->cd[buf][j];
      }
      before += ahead;
      through += ahead;
    }
    return v;
  }
  __device__ uint32_t largest(uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    if constexpr (W > 1) {
      buf ^= 1;
      if (lane == 0) s->u[buf][0][warp] = v;
      __syncthreads();
      v = __reduce_max_sync(0xffffffffu, lane < W ? s->u[buf][0][lane] : 0u);
    }
    if constexpr (CL > 1) {
      namespace cg = cooperative_groups;
      cg::cluster_group cl = cg::this_cluster();
      if (warp == 0 && lane < CL) cl.map_shared_rank(&s->cu[0][0][0], lane)[buf * 3 * CL + rank] = v;
      cl.sync();
      v = __reduce_max_sync(0xffffffffu, lane < CL ? s->cu[buf][0][lane] : 0u);
    }
    return v;
  }
  __device__ uint32_t total(uint32_t v) {
    v = __reduce_add_sync(0xffffffffu, v);
    if constexpr (W > 1) {
      buf ^= 1;
      if (lane == 0) s->u[buf][0][warp] = v;
      __syncthreads();
      v = __reduce_add_sync(0xffffffffu, lane < W ? s->u[buf][0][lane] : 0u);
    }
    if constexpr (CL > 1) {
      namespace cg = cooperative_groups;
      cg::cluster_group cl = cg::this_cluster();
      if (warp == 0 && lane < CL) cl.map_shared_rank(&s->cu[0][0][0], lane)[buf * 3 * CL + rank] = v;
      cl.sync();
      v = __reduce_add_sync(0xffffffffu, lane < CL ? s->cu[buf][0][lane] : 0u);
    }
    return v;
  }
  // The group's sums of two f32, by trees of at most 5 levels a step.
  static __device__ float2 warp_pair(float2 v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    return v;
  }
  __device__ float2 pair_sum(float2 v) {
    const float2 nil = make_float2(0.0f, 0.0f);
    v = warp_pair(v);
    if constexpr (W > 1) {
      buf ^= 1;
      if (lane == 0) s->f[buf][warp] = v;
      __syncthreads();
      v = warp_pair(lane < W ? s->f[buf][lane] : nil);
    }
    if constexpr (CL > 1) {
      namespace cg = cooperative_groups;
      cg::cluster_group cl = cg::this_cluster();
      if (warp == 0 && lane < CL) cl.map_shared_rank(&s->cf[0][0], lane)[buf * CL + rank] = v;
      cl.sync();
      v = warp_pair(lane < CL ? s->cf[buf][lane] : nil);
    }
    return v;
  }
  // The group's sum of one u32 a thread whose warp sums stay below 2^32.
  __device__ double sum_u32(uint32_t v) {
    v = __reduce_add_sync(0xffffffffu, v);
    if constexpr (W > 1 || CL > 1) return sum(lane == 0 ? double(v) : 0.0);
    return double(v);
  }
  // The same, with the minimum and maximum of two more.
  __device__ double masses(uint32_t add, uint32_t& mn, uint32_t& mx) {
    if constexpr (W > 1 || CL > 1) {
      const double v = sum_u32(add);
      uint32_t none = 0;
      counts(none, mn, mx);
      return v;
    }
    counts(add, mn, mx);
    return double(add);
  }
  // The sum over the warps ahead of this one of a value the warp agrees on;
  // *all (if asked for) gets the group's sum.
  __device__ uint32_t ahead(uint32_t v, uint32_t* all = nullptr) {
    uint32_t before = 0;
    if constexpr (W > 1) {
      buf ^= 1;
      if (lane == 0) s->u[buf][0][warp] = v;
      __syncthreads();
      const uint32_t sc = warp_scan(lane < W ? s->u[buf][0][lane] : 0u, lane);
      before = warp ? __shfl_sync(0xffffffffu, sc, warp - 1) : 0u;
      v = __shfl_sync(0xffffffffu, sc, W - 1);
    }
    if constexpr (CL > 1) {
      namespace cg = cooperative_groups;
      cg::cluster_group cl = cg::this_cluster();
      if (warp == 0 && lane < CL) cl.map_shared_rank(&s->cu[0][0][0], lane)[buf * 3 * CL + rank] = v;
      cl.sync();
      const uint32_t sc = warp_scan(lane < CL ? s->cu[buf][0][lane] : 0u, lane);
      const uint32_t others = __shfl_sync(0xffffffffu, sc, rank ? rank - 1 : 0);
      if (rank) before += others;
      v = __shfl_sync(0xffffffffu, sc, CL - 1);
    }
    if (all) *all = v;
    return before;
  }
};

// A 16-byte vector as four words: entry e of it, and two results as a word.
template <typename T> __device__ __forceinline__ float entry(const uint32_t* w, int e);
template <> __device__ __forceinline__ float entry<float>(const uint32_t* w, int e) { return __uint_as_float(w[e]); }
template <> __device__ __forceinline__ float entry<__nv_bfloat16>(const uint32_t* w, int e) {
  return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
}
template <> __device__ __forceinline__ float entry<__half>(const uint32_t* w, int e) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu)));
}
template <typename T> __device__ __forceinline__ void set2(uint32_t* w, int e, float x, float y);
template <> __device__ __forceinline__ void set2<float>(uint32_t* w, int e, float x, float y) {
  w[e] = __float_as_uint(x);
  w[e + 1] = __float_as_uint(y);
}
template <> __device__ __forceinline__ void set2<__half>(uint32_t* w, int e, float x, float y) {
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[e / 2]) : "f"(y), "f"(x));
}
template <> __device__ __forceinline__ void set2<__nv_bfloat16>(uint32_t* w, int e, float x, float y) {
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[e / 2]) : "f"(y), "f"(x));
}

// Entry e of a vector set to x (by masks: an index would move the vector to local memory).
template <typename T> __device__ __forceinline__ void set_entry(uint32_t* w, uint32_t e, float x) {
  uint32_t d[2];
  set2<T>(d, 0, x, x);
  const uint32_t part = sizeof(T) == 4 ? 0xffffffffu : e & 1 ? 0xffff0000u : 0xffffu;
#pragma unroll
  for (uint32_t j = 0; j < 4; j++) {
    const uint32_t hit = e * uint32_t(sizeof(T)) / 4 == j ? part : 0u;
    w[j] = (w[j] & ~hit) | (d[0] & hit);
  }
}

// The word w with the first (second) entry of x; an f32 word is one entry.
template <typename T> __device__ __forceinline__ uint32_t first_of(uint32_t x, uint32_t w) {
  return sizeof(T) == 4 ? x : (w & 0xffff0000u) | (x & 0xffffu);
}
template <typename T> __device__ __forceinline__ uint32_t second_of(uint32_t x, uint32_t w) {
  return sizeof(T) == 4 ? x : (w & 0xffffu) | (x & 0xffff0000u);
}

// Writes a row's entries of T, a 16-byte vector a lane and chunk, to an address
// that need not be aligned as the vectors are. With out + i + delta on a
// 16-byte boundary, a lane stores its own entries from delta on and the next
// lane's (lane 31: the next chunk's lane 0) up to delta: whole vectors again,
// for four shuffles and a shift in registers. What the row's and the warp's
// ends leave is written entry by entry. The warp calls put for its chunks in
// order, then finish.
template <typename T>
struct RowWriter {
  static constexpr int V = 16 / int(sizeof(T));
  T* out;
  int n, lane, delta, prev_i;
  uint4 prev;
  bool have;

  __device__ RowWriter(T* o, int len, int l, int i0) : out(o), n(len), lane(l), have(false) {
    delta = int((16 - (reinterpret_cast<uintptr_t>(o + i0) & 15)) & 15) / int(sizeof(T));
  }
  __device__ void some(const uint4& d, int i, int from, int to) {
    const T* e = reinterpret_cast<const T*>(&d);
#pragma unroll
    for (int j = 0; j < V; j++)
      if (j >= from && j < to && i + j >= 0 && i + j < n) out[i + j] = e[j];
  }
  __device__ void whole(const uint4& d, int i) {
    if (i >= 0 && i + V <= n) __stcs(reinterpret_cast<uint4*>(out + i), d);
    else some(d, i, 0, V);
  }
  __device__ void emit(const uint4& next, bool last) {
    const uint4 s = lane == 0 ? next : prev;
    uint32_t a[8] = {prev.x, prev.y, prev.z, prev.w, 0u, 0u, 0u, 0u};
    const int from = (lane + 1) & 31;
    a[4] = __shfl_sync(0xffffffffu, s.x, from);
    a[5] = __shfl_sync(0xffffffffu, s.y, from);
    a[6] = __shfl_sync(0xffffffffu, s.z, from);
    a[7] = __shfl_sync(0xffffffffu, s.w, from);
    const int words = delta * int(sizeof(T)) / 4;
    if (words & 2) {
#pragma unroll
      for (int j = 0; j < 6; j++) a[j] = a[j + 2];
    }
    if (words & 1) {
#pragma unroll
      for (int j = 0; j < 5; j++) a[j] = a[j + 1];
    }
    if (sizeof(T) == 2 && (delta & 1)) {
#pragma unroll
      for (int j = 0; j < 4; j++) a[j] = __byte_perm(a[j], a[j + 1], 0x5432);
    }
    const uint4 d = make_uint4(a[0], a[1], a[2], a[3]);
    if (last && lane == 31) some(d, prev_i + delta, 0, V - delta);
    else whole(d, prev_i + delta);
  }
  __device__ void put(const uint32_t* w, int i) {
    const uint4 d = make_uint4(w[0], w[1], w[2], w[3]);
    if (delta == 0) {
      whole(d, i);
      return;
    }
    if (have) emit(d, false);
    else if (lane == 0) some(d, i, 0, delta);
    prev = d;
    prev_i = i;
    have = true;
  }
  __device__ void finish() {
    if (delta && have) emit(prev, true);
  }
};

// Clears n entries of T by `threads` threads, whole vectors where they are.
template <typename T>
__device__ __forceinline__ void clear_row(T* out, int n, int tid, int threads) {
  constexpr int V = 16 / int(sizeof(T));
  const int shift = int((reinterpret_cast<uintptr_t>(out) & 15) / sizeof(T));
  for (int j = tid; j * V < n + shift; j += threads) {
    const int i = j * V - shift;
    if (i >= 0 && i + V <= n) {
      *reinterpret_cast<uint4*>(out + i) = make_uint4(0u, 0u, 0u, 0u);
    } else {
#pragma unroll
      for (int e = 0; e < V; e++)
        if (i + e >= 0 && i + e < n) out[i + e] = from_f32<T>(0.0f);
    }
  }
}

// Where a row lies. The frame of a ragged row is found by a 32-way search of
// q_off (three probes for 4096 frames). False: the row lies behind the last
// frame's questions, and nothing of it exists.
struct RowAt {
  uint64_t in, out;
  uint64_t n;
};
// Row `before` of frame f, whose block holds count rows.
__device__ __forceinline__ void block(const RowsArg& r, uint32_t f, uint64_t count, uint64_t before, RowAt* at) {
  const uint64_t p0 = r.p_off[f], size = r.p_off[f + 1] - p0;
  uint64_t n;
  if ((size | count) >> 32) n = size / count;
  else n = uint32_t(size) / uint32_t(count);
  at->in = at->out = p0 + before * n;
  at->n = n;
}
__device__ __forceinline__ bool locate(const RowsArg& r, uint64_t out_pitch, uint32_t row, int lane, RowAt* at,
                                       uint32_t* frame = nullptr) {
  if (r.frames == 0) {
    *at = RowAt{row * r.pitch, row * out_pitch, r.row_len};
    return true;
  }
  uint32_t lo = row;
  uint64_t first = row, count = 1;
  if (r.q_off) {
    uint32_t hi = r.frames;
    lo = 0;
    if (row >= r.q_off[hi]) return false;
    while (hi - lo > 1) {
      const uint32_t step = (hi - lo + 31) / 32;
      const uint64_t probe = uint64_t(lo) + uint64_t(lane) * step;
      const uint32_t below = __popc(__ballot_sync(0xffffffffu, probe < hi && r.q_off[probe < hi ? probe : lo] <= row));
      lo += (max(below, 1u) - 1) * step;
      hi = min(hi, lo + step);
    }
    first = r.q_off[lo];
    if (row < first) return false;  // offsets that do not start at 0 have no such row
    count = r.q_off[lo + 1] - first;
  } else if (row >= r.frames) {
    return false;
  }
  if (frame) *frame = lo;
  block(r, lo, count, row - first, at);
  return true;
}

// The rows from one on, in order: the frame is searched for once.
struct Walk {
  RowAt at;
  uint64_t end;    // the row behind the frame's last
  uint32_t frame;

  __device__ __forceinline__ bool start(const RowsArg& r, uint64_t out_pitch, uint32_t row, int lane) {
    if (!locate(r, out_pitch, row, lane, &at, &frame)) return false;
    pitch_out = out_pitch;
    end = r.frames == 0 ? ~0ull : r.q_off ? r.q_off[frame + 1] : uint64_t(row) + 1;
    return true;
  }
  // To the next row; false behind the last frame.
  __device__ __forceinline__ bool step(const RowsArg& r, uint32_t row) {
    if (r.frames == 0) {
      at.in += r.pitch;
      at.out += pitch_out;
      return true;
    }
    if (row < end) {
      at.in += at.n;
      at.out = at.in;
      return true;
    }
    uint64_t count = 1;
    do {  // frames without questions hold no rows
      if (++frame >= r.frames) return false;
      const uint64_t from = end;
      end = r.q_off ? r.q_off[frame + 1] : uint64_t(row) + 1;
      count = r.q_off ? end - from : 1;
    } while (row >= end);
    block(r, frame, count, 0, &at);
    return true;
  }

 private:
  uint64_t pitch_out;
};

struct Cut {
  double inv_t;
  bool greedy;      // a temperature that is not above 0: the first largest entry alone
  uint32_t k;       // 0: off
  double top_p;     // >= 1: off
  double min_p;     // <= 0: off
};
__device__ __forceinline__ Cut cut_of(const CutArg& c, uint32_t row) {
  const float t = c.row_temperature ? c.row_temperature[row] : c.temperature;
  const float p = c.row_top_p ? c.row_top_p[row] : c.top_p;
  const float m = c.row_min_p ? c.row_min_p[row] : c.min_p;
  Cut o;
  o.inv_t = !c.row_temperature ? c.inv_temperature : t > 0.0f ? 1.0 / double(t) : 0.0;
  o.k = c.row_top_k ? c.row_top_k[row] : c.top_k;
  o.top_p = p < 1.0f ? fmax(double(p), 0.0) : 2.0;  // a NaN cuts nothing
  o.min_p = m > 0.0f ? fmin(double(m), 1.0) : 0.0;
  o.greedy = !(t > 0.0f);
  if (o.greedy) o.k = 1;
  return o;
}

}  // namespace pol
}  // namespace kc
