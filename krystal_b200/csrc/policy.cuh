// policy.cuh — what a host does with the rows of scores or probabilities a
// selection leaves: draw an answer from a tempered and cut distribution
// (k_draw), and the loss of drawn answers with its gradient (k_policy_loss).
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
// halving the range of values between snapped row entries.
//
// A row lives in registers: E entries a thread, one warp a row up to 1024
// entries, a CTA to 32768, a cluster of CTAs beyond. Warp g of the row's
// group owns the contiguous segment [32 E g, 32 E (g + 1)), in chunks of one
// 16-byte load a lane, so that bank order is (warp, chunk, lane, entry) and a
// prefix sum needs one warp scan a chunk.
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

// One logarithm a row or two, out of line.
static __device__ __noinline__ double log64(double v) { return log(v); }

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
  Shared& s;
  int lane, warp, rank, buf;

  __device__ Group(Shared& sh, int l, int w) : s(sh), lane(l), warp(w), rank(0), buf(0) {
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
      if (lane == 0) { s.u[buf][0][warp] = add; s.u[buf][1][warp] = mn; s.u[buf][2][warp] = mx; }
      __syncthreads();
      const bool in = lane < W;
      add = __reduce_add_sync(0xffffffffu, in ? s.u[buf][0][lane] : 0u);
      mn = __reduce_min_sync(0xffffffffu, in ? s.u[buf][1][lane] : 0xffffffffu);
      mx = __reduce_max_sync(0xffffffffu, in ? s.u[buf][2][lane] : 0u);
    }
    if constexpr (CL > 1) {
      namespace cg = cooperative_groups;
      cg::cluster_group cl = cg::this_cluster();
      if (warp == 0 && lane < CL) {
        uint32_t* dst = cl.map_shared_rank(&s.cu[0][0][0], lane) + buf * 3 * CL;
        dst[rank] = add; dst[CL + rank] = mn; dst[2 * CL + rank] = mx;
      }
      cl.sync();
      const bool in = lane < CL;
      add = __reduce_add_sync(0xffffffffu, in ? s.cu[buf][0][lane] : 0u);
      mn = __reduce_min_sync(0xffffffffu, in ? s.cu[buf][1][lane] : 0xffffffffu);
      mx = __reduce_max_sync(0xffffffffu, in ? s.cu[buf][2][lane] : 0u);
    }
  }
  // The group's sum of one value a thread; *before (if asked for) gets the
  // sum over the warps ahead of this one in bank order.
  __device__ double sum(double v, double* before = nullptr) {
    v = warp_add(v);
    if constexpr (W > 1) {
      buf ^= 1;
      if (lane == 0) s.d[buf][warp] = v;
      __syncthreads();
      const double sc = warp_scan(lane < W ? s.d[buf][lane] : 0.0, lane);
      if (before) *before = warp ? __shfl_sync(0xffffffffu, sc, warp - 1) : 0.0;
      v = __shfl_sync(0xffffffffu, sc, W - 1);
    } else if (before) {
      *before = 0.0;
    }
    if constexpr (CL > 1) {
      namespace cg = cooperative_groups;
      cg::cluster_group cl = cg::this_cluster();
      if (warp == 0 && lane < CL) cl.map_shared_rank(&s.cd[0][0], lane)[buf * CL + rank] = v;
      cl.sync();
      const double sc = warp_scan(lane < CL ? s.cd[buf][lane] : 0.0, lane);
      const double ahead = __shfl_sync(0xffffffffu, sc, rank ? rank - 1 : 0);
      if (before && rank) *before += ahead;
      v = __shfl_sync(0xffffffffu, sc, CL - 1);
    }
    return v;
  }
  __device__ uint32_t largest(uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    if constexpr (W > 1) {
      buf ^= 1;
      if (lane == 0) s.u[buf][0][warp] = v;
      __syncthreads();
      v = __reduce_max_sync(0xffffffffu, lane < W ? s.u[buf][0][lane] : 0u);
    }
    if constexpr (CL > 1) {
      namespace cg = cooperative_groups;
      cg::cluster_group cl = cg::this_cluster();
      if (warp == 0 && lane < CL) cl.map_shared_rank(&s.cu[0][0][0], lane)[buf * 3 * CL + rank] = v;
      cl.sync();
      v = __reduce_max_sync(0xffffffffu, lane < CL ? s.cu[buf][0][lane] : 0u);
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
      if (lane == 0) s.f[buf][warp] = v;
      __syncthreads();
      v = warp_pair(lane < W ? s.f[buf][lane] : nil);
    }
    if constexpr (CL > 1) {
      namespace cg = cooperative_groups;
      cg::cluster_group cl = cg::this_cluster();
      if (warp == 0 && lane < CL) cl.map_shared_rank(&s.cf[0][0], lane)[buf * CL + rank] = v;
      cl.sync();
      v = warp_pair(lane < CL ? s.cf[buf][lane] : nil);
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
  // The sum over the warps ahead of this one of a value the warp agrees on.
  __device__ uint32_t ahead(uint32_t v) {
    uint32_t before = 0;
    if constexpr (W > 1) {
      buf ^= 1;
      if (lane == 0) s.u[buf][0][warp] = v;
      __syncthreads();
      const uint32_t sc = warp_scan(lane < W ? s.u[buf][0][lane] : 0u, lane);
      before = warp ? __shfl_sync(0xffffffffu, sc, warp - 1) : 0u;
      v = __shfl_sync(0xffffffffu, sc, W - 1);
    }
    if constexpr (CL > 1) {
      namespace cg = cooperative_groups;
      cg::cluster_group cl = cg::this_cluster();
      if (warp == 0 && lane < CL) cl.map_shared_rank(&s.cu[0][0][0], lane)[buf * 3 * CL + rank] = v;
      cl.sync();
      const uint32_t sc = warp_scan(lane < CL ? s.cu[buf][0][lane] : 0u, lane);
      const uint32_t others = __shfl_sync(0xffffffffu, sc, rank ? rank - 1 : 0);
      if (rank) before += others;
    }
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

// Where a row lies. The frame of a ragged row is found by a 32-way search of
// q_off (three probes for 4096 frames). False: the row lies behind the last
// frame's questions, and nothing of it exists.
struct RowAt {
  uint64_t in, out;
  uint64_t n;
};
__device__ __forceinline__ bool locate(const RowsArg& r, uint64_t out_pitch, uint32_t row, int lane, RowAt* at) {
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
      lo += (below - 1) * step;
      hi = min(hi, lo + step);
    }
    first = r.q_off[lo];
    count = r.q_off[lo + 1] - first;
  } else if (row >= r.frames) {
    return false;
  }
  const uint64_t p0 = r.p_off[lo], block = r.p_off[lo + 1] - p0;
  uint64_t n;
  if ((block | count) >> 32) n = block / count;
  else n = uint32_t(block) / uint32_t(count);
  const uint64_t at0 = p0 + (row - first) * n;
  *at = RowAt{at0, at0, n};
  return true;
}

struct Cut {
  double inv_t;     // 0: the largest entry alone
  uint32_t k;       // 0: off
  double top_p;     // >= 1: off
  double min_p;     // <= 0: off
};
__device__ __forceinline__ Cut cut_of(const CutArg& c, uint32_t row) {
  const float t = c.row_temperature ? c.row_temperature[row] : c.temperature;
  const float p = c.row_top_p ? c.row_top_p[row] : c.top_p;
  const float m = c.row_min_p ? c.row_min_p[row] : c.min_p;
  Cut o;
  o.inv_t = t > 0.0f ? 1.0 / double(t) : 0.0;
  o.k = c.row_top_k ? c.row_top_k[row] : c.top_k;
  o.top_p = p < 1.0f ? fmax(double(p), 0.0) : 2.0;  // a NaN cuts nothing
  o.min_p = m > 0.0f ? fmin(double(m), 1.0) : 0.0;
  if (!(t > 0.0f)) o.k = 1;
  return o;
}

// A row's entries in registers, and its cut.
template <typename T, int E, int W, int CL>
struct Row {
  static constexpr int V = 16 / int(sizeof(T));
  static constexpr int kChunks = E / V;
  static constexpr uint32_t kCap = uint32_t(32) * E * W * CL;
  static constexpr bool kCached = E <= 32;  // the registers hold a weight an entry beside the keys
  static_assert(E % V == 0 && kChunks <= 32, "a thread holds whole vectors");

  Group<W, CL> g;
  uint32_t k[E];   // keys; 0: not in the support
  uint32_t live;   // chunks of this warp that hold an entry of the support
  double tab;      // 2^{lane/32}
  double c_tab, l_tab;  // log_tab's table, for tempered probabilities
  double m, log_m, inv_t;
  bool power;      // probabilities at a temperature other than 1: x from logarithms
  bool plain_p;    // probabilities at T = 1: the weights are the values
  int i0;          // index of this lane's first entry of chunk 0

  __device__ Row(typename Group<W, CL>::Shared& sh, int lane, int warp) : g(sh, lane, warp) {
    tab = exp2(double(lane) * (1.0 / 32.0));
    c_tab = 1.0 / (1.0 + (lane + 0.5) * (1.0 / 32.0));
    l_tab = 0.0;
  }

  __device__ int at(int c) const { return i0 + c * 32 * V; }
  __device__ uint32_t index(int e) const { return uint32_t(at(e / V) + e % V); }

  // f(entry) for every entry of the chunks that hold any; the warp together.
  template <typename F>
  __device__ __forceinline__ void each(F f) {
#pragma unroll
    for (int c = 0; c < kChunks; c++)
      if (live >> c & 1u) {
#pragma unroll
        for (int e = 0; e < V; e++) f(c * V + e);
      }
  }
  __device__ void find_live() {
    live = 0;
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      uint32_t any = 0;
#pragma unroll
      for (int e = 0; e < V; e++) any |= k[c * V + e];
      if (__any_sync(0xffffffffu, any != 0u)) live |= 1u << c;
    }
  }

  // Loads n entries from row. A lane's 16-byte loads start on 16-byte
  // boundaries; a vector that reaches past either end of the row is read
  // entry by entry.
  __device__ void load(const T* row, uint32_t n, int kind) {
    const int shift = int((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    i0 = g.segment() * 32 * E + g.lane * V - shift;
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      const int i = at(c);
      alignas(16) T v[V];
      bool in[V];
      if (i >= 0 && i + V <= int(n)) {
        *reinterpret_cast<uint4*>(v) = __ldcs(reinterpret_cast<const uint4*>(row + i));
#pragma unroll
        for (int e = 0; e < V; e++) in[e] = true;
      } else {
#pragma unroll
        for (int e = 0; e < V; e++) {
          in[e] = i + e >= 0 && i + e < int(n);
          v[e] = in[e] ? row[i + e] : from_f32<T>(0.0f);
        }
      }
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float f = as_f32(v[e]);
        const bool open = in[e] && (kind == kKindP ? f > 0.0f : f > Lowest<T>::open_above);
        k[c * V + e] = open ? key_of(fminf(f, 3.402823466e38f)) : 0u;
      }
    }
    find_live();
  }

  // The tempered log weight of a key in the support (a key outside it: some
  // number). Every lane of the warp calls this together.
  __device__ double x_of(uint32_t key) const {
    const float v = value_of(key ? key : 0xbf800000u);
    return power ? (log_tab(v, c_tab, l_tab) - log_m) * inv_t : (double(v) - m) * inv_t;
  }
  // The weight of an x, and of a key; 0 for key 0 and for dropped entries.
  __device__ double weight_of(uint32_t key, double x) const {
    const double w = exp64(fmin(fmax(x, kDropped), 0.0), tab);
    return key && x >= kDropped ? w : 0.0;
  }
  __device__ double weight(uint32_t key) const {
    if (plain_p) return key ? double(value_of(key)) : 0.0;
    return weight_of(key, x_of(key));
  }

  // The pivot between two values of the row: halfway in value for scores,
  // halfway in exponent and mantissa for probabilities (which span decades);
  // after a dozen steps the two alternate, so that no row takes more than
  // about 70 steps whatever its values.
  __device__ static uint32_t pivot(uint32_t lo, uint32_t hi, int step, int kind) {
    const bool by_value = step < 12 ? kind != kKindP : (step & 1);
    uint32_t p = lo + (hi - lo + 1) / 2;
    if (by_value) p = key_of(0.5f * value_of(lo) + 0.5f * value_of(hi));
    return min(max(p, lo + 1), hi);
  }

  // Drops the entries below the cut t and all but the first `ties` of the
  // `all` at it.
  __device__ void apply(uint32_t t, uint32_t ties, uint32_t all) {
    if (ties >= all) {
      each([&](int e) { if (k[e] < t) k[e] = 0u; });
    } else {
      uint32_t mine = 0;
      each([&](int e) { mine += k[e] == t; });
      uint32_t seen = g.ahead(__reduce_add_sync(0xffffffffu, mine));
#pragma unroll
      for (int c = 0; c < kChunks; c++) {
        uint32_t in = 0;
#pragma unroll
        for (int e = 0; e < V; e++) in += k[c * V + e] == t;
        const uint32_t incl = warp_scan(in, g.lane);
        uint32_t r = seen + incl - in;
#pragma unroll
        for (int e = 0; e < V; e++) {
          const uint32_t key = k[c * V + e];
          if (key == t) {
            if (r >= ties) k[c * V + e] = 0u;
            r++;
          } else if (key < t) {
            k[c * V + e] = 0u;
          }
        }
        seen += __shfl_sync(0xffffffffu, incl, 31);
      }
    }
    find_live();
  }

  // top-p's search by approximate weights: f32 exponentials in units of 2^-20
  // of the largest, summed as integers. An entry above half a unit has |x| <=
  // 21 ln 2; three f32 roundings of the exponent and ex2's 2^-22 put its weight
  // within 3e-6, and for probabilities lg2's 2^-22 of log2 v and of log2 m add
  // 3.4e-7 (|log2 m| + 21 T) / T. A mass that clears the goal by `err` of the
  // total and half a unit an entry is on its side for certain; the first pivot
  // that does not leaves [lo, cur] to the 64-bit search. What it usually
  // leaves is one value.
  __device__ void narrow(double top_p, uint32_t open, int kind, uint32_t& lo, uint32_t& cur) {
    uint32_t q[E], all = 0;
    const float mv = float(m), it = float(inv_t) * (kind == kKindP ? 1.0f : 1.44269504f);
    const float mu = kind == kKindP ? log2_fast(mv) : mv;
    each([&](int e) {
      const float v = value_of(k[e] ? k[e] : 0xbf800000u);
      const float u = ((kind == kKindP ? log2_fast(v) : v) - mu) * it;
      q[e] = k[e] ? __float2uint_rn(exp2_fast(fminf(u, 0.0f)) * 1048576.0f) : 0u;
      all += q[e];
    });
    const double total = g.sum_u32(all);
    const double goal = top_p * total;
    const double err = (1e-5 + 1e-5 * inv_t + 4e-7 * fabs(double(mu)) * (kind == kKindP ? inv_t : 0.0)) * total +
                       0.5 * open + 1.0;
    for (int step = 0; cur != lo; step++) {
      const uint32_t p = pivot(lo, cur, step, kind);
      uint32_t mass = 0, mn = 0xffffffffu, mx = 0u;
      each([&](int e) {
        if (k[e] >= p) { mass += q[e]; mn = min(mn, k[e]); }
        else mx = max(mx, k[e]);
      });
      const double a = g.masses(mass, mn, mx);
      if (a >= goal + err) lo = mn;
      else if (a < goal - err) cur = mx;
      else return;
    }
  }

  // The temperature and the cuts; afterwards k[e] != 0 exactly for what top-k
  // and top-p keep (min-p and the dropping are left to the weights' pass).
  // Returns the open entries before the cuts.
  __device__ uint32_t cut(const Cut& c, int kind) {
    uint32_t open = 0, lo = 0xffffffffu, hi = 0u;
    each([&](int e) {
      open += k[e] != 0u;
      if (k[e]) lo = min(lo, k[e]);
      hi = max(hi, k[e]);
    });
    g.counts(open, lo, hi);
    plain_p = kind == kKindP && c.inv_t == 1.0;
    power = kind == kKindP && !plain_p;
    inv_t = c.inv_t;
    if (open == 0) { m = log_m = 0.0; return 0; }
    m = double(value_of(hi));
    log_m = 0.0;
    if (power) {
      l_tab = -log64(c_tab);
      log_m = log_tab(value_of(hi), c_tab, l_tab);
    }
    const uint32_t top = hi;
    uint32_t left = open;
    if (c.k && c.k < open) {
      // the largest t with count(k >= t) >= c.k; `above`: count(k > t's bracket)
      uint32_t cur = top, above = 0, at_lo = open;
      for (int step = 0; cur != lo; step++) {
        const uint32_t p = pivot(lo, cur, step, kind);
        uint32_t n = 0, mn = 0xffffffffu, mx = 0u;
        each([&](int e) {
          if (k[e] >= p) { n++; mn = min(mn, k[e]); }
          else mx = max(mx, k[e]);
        });
        g.counts(n, mn, mx);
        if (n >= c.k) { lo = mn; at_lo = n; }
        else { cur = mx; above = n; }
      }
      apply(lo, c.k - above, at_lo - above);
      left = c.k;
    }
    if (c.top_p < 1.0) {
      // the largest t with mass(k >= t) >= goal
      uint32_t cur = top;
      if constexpr (kCached) narrow(c.top_p, left, kind, lo, cur);
      uint32_t ties = 0, mn = 0xffffffffu, mx = 0u;
      each([&](int e) { ties += k[e] == lo; });
      g.counts(ties, mn, mx);
      if (cur != lo || ties > 1) {
        double part = 0.0, over = 0.0;
        each([&](int e) {
          const double w = weight(k[e]);
          part += w;
          if (k[e] > cur) over += w;
        });
        const double goal = c.top_p * g.sum(part);
        double above = g.sum(over);
        for (int step = 0; cur != lo; step++) {
          const uint32_t p = pivot(lo, cur, step, kind);
          double mass = 0.0;
          uint32_t n = 0;
          mn = 0xffffffffu, mx = 0u;
          each([&](int e) {
            const bool in = k[e] >= p && k[e] <= cur;
            if (__any_sync(0xffffffffu, in)) mass += weight(in ? k[e] : 0u);
            if (k[e] >= p) mn = min(mn, k[e]);
            else mx = max(mx, k[e]);
          });
          mass = above + g.sum(mass);
          g.counts(n, mn, mx);
          if (mass >= goal) lo = mn;
          else { cur = mx; above = mass; }
        }
        ties = 0, mn = 0xffffffffu, mx = 0u;
        each([&](int e) { ties += k[e] == lo; });
        g.counts(ties, mn, mx);
        const double w = weight(lo);
        const double need = w > 0.0 ? ceil((goal - above) / w) : 1.0;
        apply(lo, need < 1.0 ? 1u : need >= double(ties) ? ties : uint32_t(need), ties);
      } else {
        apply(lo, 1u, 1u);
      }
    }
    return open;
  }
};

template <typename T, int E, int W, int CL>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32) k_draw(DrawArg a) {
  using R = Row<T, E, W, CL>;
  constexpr int V = R::V;
  __shared__ typename Group<W, CL>::Shared sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t row = W == 1 ? blockIdx.x * 4 + warp : blockIdx.x / CL;
  if (row >= a.r.rows) return;
  RowAt at;
  if (!locate(a.r, a.out_pitch, row, lane, &at)) return;
  R r(sh, lane, W == 1 ? 0 : warp);
  const bool fits = at.n <= a.r.row_len && at.n + V - 1 <= R::kCap;
  const uint32_t n = fits ? uint32_t(at.n) : 0u;
  const T* in = static_cast<const T*>(a.r.values) + at.in;
  r.load(in, n, a.r.kind);
  const Cut c = cut_of(a.c, row);
  r.cut(c, a.r.kind);
  // the weights, their prefix sums chunk by chunk in bank order
  const double floor_w = c.min_p * (r.plain_p ? r.m : 1.0);
  double incl[R::kChunks], w[R::kCached ? E : 1], run = 0.0;
  uint32_t kept = 0, last = 0u;
#pragma unroll
  for (int ch = 0; ch < R::kChunks; ch++) {
    incl[ch] = run;
    if (!(r.live >> ch & 1u)) continue;
    double s = 0.0;
#pragma unroll
    for (int e = ch * V; e < ch * V + V; e++) {
      double we = r.weight(r.k[e]);
      if (we < floor_w) we = 0.0;
      if (!(we > 0.0)) r.k[e] = 0u;
      if constexpr (R::kCached) w[e] = we;
      s += we;
      if (r.k[e]) {
        kept++;
        last = r.index(e) + 1u;
      }
    }
    const double sc = warp_scan(s, lane);
    incl[ch] = run + sc;
    run += __shfl_sync(0xffffffffu, sc, 31);
  }
  auto weight = [&](int e) {
    if constexpr (R::kCached) return w[e];
    else return r.weight(r.k[e]);
  };
  double before;
  const double z = r.g.sum(lane == 31 ? run : 0.0, &before);
  // the first entry whose prefix passes u z, or (no u) the first largest
  uint32_t hit = 0xffffffffu;
  if (a.uniforms) {
    // cum > u z by the sign of u z - cum, whose one rounding keeps it: u on an
    // entry's edge falls where the reals put it
    const double u = fmin(fmax(a.uniforms[row], 0.0), 1.0);
#pragma unroll
    for (int ch = 0; ch < R::kChunks; ch++) {
      const bool past = (r.live >> ch & 1u) && fma(u, z, -(before + incl[ch])) < 0.0;
      if (hit == 0xffffffffu && __any_sync(0xffffffffu, past)) {
        // the first such lane walks its entries from the prefix ahead of it
        const int who = __ffs(__ballot_sync(0xffffffffu, past)) - 1;
        double ws[V], own = 0.0;
#pragma unroll
        for (int e = 0; e < V; e++) own += ws[e] = weight(ch * V + e);
        double cum = before + (incl[ch] - own);
        uint32_t found = 0xffffffffu;
#pragma unroll
        for (int e = 0; e < V; e++) {
          cum += ws[e];
          if (found == 0xffffffffu && r.k[ch * V + e] && fma(u, z, -cum) < 0.0) found = r.index(ch * V + e);
        }
        if (found == 0xffffffffu) {  // a last bit short: the lane's last kept entry
#pragma unroll
          for (int e = 0; e < V; e++)
            if (r.k[ch * V + e]) found = r.index(ch * V + e);
        }
        hit = __shfl_sync(0xffffffffu, found, who);
      }
    }
  } else {
    const uint32_t top = key_of(float(r.m));
#pragma unroll
    for (int e = E - 1; e >= 0; e--)
      if (r.k[e] == top) hit = r.index(e);
  }
  r.g.counts(kept, hit, last);
  if (kept && hit == 0xffffffffu) hit = last - 1u;
  // the owner of the entry writes the row's answer
  const bool lead = r.g.segment() == 0 && lane == 0;
  if (kept == 0) {
    if (lead) {
      if (a.index) a.index[row] = kNone;
      if (a.logp) a.logp[row] = -INFINITY;
      if (a.kept) a.kept[row] = 0u;
    }
  } else {
    r.each([&](int e) {
      const bool mine = r.index(e) == hit && r.k[e];
      if (__any_sync(0xffffffffu, mine)) {
        const double we = weight(e);
        if (mine) {
          if (a.index) a.index[row] = hit;
          if (a.logp) a.logp[row] = float(log64(we / z));
        }
      }
    });
    if (lead && a.kept) a.kept[row] = kept;
  }
  if (a.p && fits) {
    const double inv = kept ? 1.0 / z : 0.0;
    float* out = a.p + at.out;
#pragma unroll
    for (int ch = 0; ch < R::kChunks; ch++) {
      const int i = r.at(ch);
      alignas(16) float v[V];
#pragma unroll
      for (int e = 0; e < V; e++) {
        v[e] = 0.0f;
        if (r.live >> ch & 1u) v[e] = float(weight(ch * V + e) * inv);
      }
      if (i >= 0 && i + V <= int(n) && (reinterpret_cast<uintptr_t>(out + i) & 15) == 0) {
#pragma unroll
        for (int e = 0; e < V; e += 4) *reinterpret_cast<float4*>(out + i + e) = *reinterpret_cast<float4*>(v + e);
      } else {
#pragma unroll
        for (int e = 0; e < V; e++)
          if (i + e >= 0 && i + e < int(n)) out[i + e] = v[e];
      }
    }
  }
}

// loss = -A log pi(a) - beta H(pi), H = log Z - sum w x / Z, and
// dloss/dv_j = (A (pi_j - [j = a]) + beta pi_j (log pi_j + H)) / T for what is
// kept, 0 elsewhere, times the row's weight.
template <typename T, int E, int W, int CL>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32) k_policy_loss(LossArg a) {
  using R = Row<T, E, W, CL>;
  constexpr int V = R::V;
  __shared__ typename Group<W, CL>::Shared sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t row = W == 1 ? blockIdx.x * 4 + warp : blockIdx.x / CL;
  if (row >= a.r.rows) return;
  RowAt at;
  if (!locate(a.r, a.out_pitch, row, lane, &at)) return;
  R r(sh, lane, W == 1 ? 0 : warp);
  const bool fits = at.n <= a.r.row_len && at.n + V - 1 <= R::kCap;
  const uint32_t n = fits ? uint32_t(at.n) : 0u;
  const T* in = static_cast<const T*>(a.r.values) + at.in;
  r.load(in, n, kKindScores);
  const Cut c = cut_of(a.c, row);
  r.cut(c, kKindScores);
  const uint32_t act = a.actions[row];
  const bool asked = act != kNone;
  double part = 0.0, px = 0.0, xa = 0.0;
  uint32_t kept = 0, live = 0xffffffffu, dummy = 0u;
  double ws[R::kCached ? E : 1];
  r.each([&](int e) {
    uint32_t& key = r.k[e];
    const double x = r.x_of(key);
    double w = r.weight_of(key, x);
    if (w < c.min_p) w = 0.0;
    if (!(w > 0.0)) key = 0u;
    if constexpr (R::kCached) ws[e] = w;
    part += w;
    px = fma(w, key ? x : 0.0, px);
    if (key) {
      kept++;
      if (r.index(e) == act) { live = 0u; xa = x; }
    }
  });
  const double z = r.g.sum(part);
  const double sx = r.g.sum(px);
  xa = r.g.sum(xa);
  r.g.counts(kept, live, dummy);
  const double log_z = kept ? log64(z) : 0.0;
  const double h = kept ? log_z - sx / z : 0.0;
  const double logp = xa - log_z;
  // a temperature that is not positive has one answer and no gradient
  const bool learns = asked && live == 0u && c.inv_t > 0.0;
  const double adv = double(a.advantage[row]), beta = double(a.beta);
  const double rw = a.row_weight ? double(a.row_weight[row]) : 1.0;
  if (r.g.segment() == 0 && lane == 0) {
    if (a.loss) a.loss[row] = learns ? float(-adv * logp - beta * h) : 0.0f;
    if (a.logp) a.logp[row] = !asked ? 0.0f : live == 0u ? float(logp) : -INFINITY;
    if (a.entropy) a.entropy[row] = float(h);
  }
  if (!a.grad || !fits) return;
  T* out = static_cast<T*>(a.grad) + at.out;
  const double g0 = rw * c.inv_t, inv_z = kept ? 1.0 / z : 0.0, base = h - log_z;
  RowWriter<T> writer(out, int(n), lane, r.i0);
#pragma unroll
  for (int ch = 0; ch < R::kChunks; ch++) {
    const int i = r.at(ch);
    float f[V];
    uint32_t v[4];
#pragma unroll
    for (int e = 0; e < V; e++) {
      const uint32_t key = r.k[ch * V + e];
      double d = 0.0;
      if (learns && (r.live >> ch & 1u)) {
        const double x = r.x_of(key);
        double pi;
        if constexpr (R::kCached) pi = ws[ch * V + e] * inv_z;
        else pi = r.weight_of(key, x) * inv_z;
        const double one = uint32_t(i + e) == act ? 1.0 : 0.0;
        if (key) d = g0 * fma(adv, pi - one, beta * pi * (x + base));
      }
      f[e] = float(d);
    }
#pragma unroll
    for (int e = 0; e < V; e += 2) set2<T>(v, e, f[e], f[e + 1]);
    writer.put(v, i);
  }
  writer.finish();
}

// ---------------------------------------------------------------------------
// The policy loss over the whole softmax, nothing cut: no decision hangs on a
// last bit, so the row stays as it was loaded (a warp's registers, NV 16-byte
// vectors a lane; longer rows: k_policy_long) and its exponentials are f32. With u_j = (v_j - m) log2(e) / T, taken as one
// fma of v_j (the rounding of m log2(e) / T is common to all and cancels),
//   Z = sum 2^u, S = sum 2^u u, log pi_j = ln 2 (u_j - log2 Z),
//   H = ln 2 (log2 Z - S / Z), and the gradient is
//   2^u_j (u_j B + C) with B = g beta ln 2 / (T Z), C = g (A + beta (H - ln Z)) / (T Z)
// but for -g A / T more at the action. Sums: eight f32 partial sums of at most
// 16 terms a thread, joined by trees. Arithmetic on pairs (f32x2).
//
// Masked entries need no test where they vanish by themselves: NaN and what
// lies below the mask's floor is raised to it as the row is loaded, and 2^u is
// 0 if (m - floor) log2(e) / T >= 200. A row where that does not hold (a
// largest score near the floor, f16 at a temperature of hundreds), that holds
// +infinity, or whose m log2(e) / T is 1e5 or more (its rounding, 2^-24 of it,
// would not stay far below 1) tests every entry and subtracts m first.
// ---------------------------------------------------------------------------
struct Pair { float x, y; };
__device__ __forceinline__ unsigned long long pack2(float x, float y) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ Pair unpack2(unsigned long long v) {
  Pair p;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(p.x), "=f"(p.y) : "l"(v));
  return p;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// What masked entries are raised to: a value of the type at or below open_above.
template <typename T> struct Floor { static constexpr float value = -1.00025555e30f; };  // a bf16 value
template <> struct Floor<__half> { static constexpr float value = -65504.0f; };


// The largest of a thread's vectors; raise() also raises a vector's entries to
// the floor, a NaN too.
template <typename T> struct Top;
template <> struct Top<float> {
  float top = Floor<float>::value;
  __device__ __forceinline__ void raise(uint32_t* w) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float f = fmaxf(__uint_as_float(w[e]), Floor<float>::value);
      w[e] = __float_as_uint(f);
      top = fmaxf(top, f);
    }
  }
  __device__ __forceinline__ float value() const { return top; }
};
template <typename T2> struct TopPairs {
  T2 low, top;
  __device__ __forceinline__ TopPairs(T2 l) : low(l), top(l) {}
  __device__ __forceinline__ void raise(uint32_t* w) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const T2 f = __hmax2(*reinterpret_cast<T2*>(w + e), low);
      w[e] = *reinterpret_cast<const uint32_t*>(&f);
      top = __hmax2(top, f);
    }
  }
  __device__ __forceinline__ float value() const { return fmaxf(__low2float(top), __high2float(top)); }
};
template <> struct Top<__half> : TopPairs<__half2> {
  __device__ __forceinline__ Top() : TopPairs(__float2half2_rn(Floor<__half>::value)) {}
};
template <> struct Top<__nv_bfloat16> : TopPairs<__nv_bfloat162> {
  __device__ __forceinline__ Top() : TopPairs(__float2bfloat162_rn(Floor<__nv_bfloat16>::value)) {}
};

template <typename T, int NV>
__global__ void __launch_bounds__(128) k_policy_whole(LossArg a) {
  constexpr int W = 1, CL = 1;
  constexpr int V = 16 / int(sizeof(T));
  constexpr uint32_t kCap = uint32_t(32) * V * NV * W * CL;
  __shared__ typename Group<W, CL>::Shared sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t row = W == 1 ? blockIdx.x * 4 + warp : blockIdx.x / CL;
  if (row >= a.r.rows) return;
  RowAt at;
  if (!locate(a.r, a.out_pitch, row, lane, &at)) return;
  Group<W, CL> g(sh, lane, W == 1 ? 0 : warp);
  const bool fits = at.n <= a.r.row_len && at.n + V - 1 <= kCap;
  const int n = fits ? int(at.n) : 0;
  const T* in = static_cast<const T*>(a.r.values) + at.in;
  const int shift = int((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
  const int i0 = g.segment() * 32 * V * NV + lane * V - shift;
  constexpr float floor_v = Floor<T>::value;

  // the row, masked entries raised to the floor; its largest
  uint32_t v[NV][4];
#pragma unroll
  for (int c = 0; c < NV; c++) {
    const int i = i0 + c * 32 * V;
    if (i >= 0 && i + V <= n) {
      const uint4 q = __ldcs(reinterpret_cast<const uint4*>(in + i));
      v[c][0] = q.x; v[c][1] = q.y; v[c][2] = q.z; v[c][3] = q.w;
    } else {
      float f[V];
#pragma unroll
      for (int e = 0; e < V; e++) f[e] = i + e >= 0 && i + e < n ? as_f32(in[i + e]) : floor_v;
#pragma unroll
      for (int e = 0; e < V; e += 2) set2<T>(v[c], e, f[e], f[e + 1]);
    }
  }
  Top<T> highest;
#pragma unroll
  for (int c = 0; c < NV; c++) highest.raise(v[c]);
  const float mx = highest.value();
  // the action's value, before anything is written: grad may lie over values
  const uint32_t act = a.actions[row];
  const bool asked = act != kNone;
  const float va = act < uint32_t(n) ? as_f32(in[act]) : floor_v;
  constexpr float kLn2 = 0.69314718055994530942f, kMost = 3.402823466e38f;
  const uint32_t top = g.largest(key_of(mx));
  const bool endless = top == 0xff800000u;  // the row holds +infinity
  const float m = endless ? kMost : value_of(top);
  const float t_row = a.c.row_temperature ? a.c.row_temperature[row] : a.c.temperature;
  const bool open_t = t_row > 0.0f, any = m > Lowest<T>::open_above;
  const float sc = open_t ? 1.44269504088896340736f / t_row : 0.0f;  // log2(e) / T
  const bool plain = !endless && (m - Lowest<T>::open_above) * sc >= 200.0f && fabsf(m * sc) < 1e5f && sc < 1e6f;
  const float off = -m * sc;
  auto u_of = [&](float f) { return plain ? fmaf(f, sc, off) : (fminf(f, m) - m) * sc; };

  // Z and S
  float2 zs = make_float2(0.0f, 0.0f);
  if (plain) {
    const unsigned long long sc2 = pack2(sc, sc), off2 = pack2(off, off);
    unsigned long long za[4] = {0ull, 0ull, 0ull, 0ull}, sa[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
    for (int c = 0; c < NV; c++)
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const int k = (c * V + e) / 2 & 3;
        const unsigned long long u = fma2(pack2(entry<T>(v[c], e), entry<T>(v[c], e + 1)), sc2, off2);
        const Pair up = unpack2(u);
        const unsigned long long w = pack2(exp2_fast(up.x), exp2_fast(up.y));
        za[k] = add2(za[k], w);
        sa[k] = fma2(w, u, sa[k]);
      }
    const Pair z1 = unpack2(add2(add2(za[0], za[1]), add2(za[2], za[3])));
    const Pair s1 = unpack2(add2(add2(sa[0], sa[1]), add2(sa[2], sa[3])));
    zs = make_float2(z1.x + z1.y, s1.x + s1.y);
  } else if (any) {
    double z = 0.0, s = 0.0;
#pragma unroll
    for (int c = 0; c < NV; c++)
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float f = entry<T>(v[c], e);
        if (f > Lowest<T>::open_above) {
          const float u = fmaxf(u_of(f), -2000.0f), w = exp2_fast(u);
          z += double(w);
          s += double(w) * double(u);
        }
      }
    zs = make_float2(float(z), float(s));
  }
  zs = g.pair_sum(zs);
  // the widened entries are made again below, not kept: 16-bit rows would take
  // twice the registers
#pragma unroll
  for (int c = 0; c < NV; c++) asm volatile("" : "+r"(v[c][0]), "+r"(v[c][1]), "+r"(v[c][2]), "+r"(v[c][3]));

  // the row's answer
  const float ua = u_of(fminf(va, kMost));
  bool live = asked && va > Lowest<T>::open_above && ua * kLn2 >= float(kDropped);
  if (!open_t) {  // temperature 0: the first largest entry alone
    uint32_t first = 0xffffffffu;
#pragma unroll
    for (int c = 0; c < NV; c++)
#pragma unroll
      for (int e = 0; e < V; e++)
        if (fminf(entry<T>(v[c], e), kMost) == m) first = min(first, uint32_t(i0 + c * 32 * V + e));
    uint32_t zero = 0, none = 0;
    g.counts(none, first, zero);
    live = asked && any && first == act;
  }
  const float lg_z = any ? log2f(zs.x) : 0.0f, inv_z = any ? 1.0f / zs.x : 0.0f;
  const float h = any && open_t ? kLn2 * (lg_z - zs.y * inv_z) : 0.0f;
  const float logp = open_t ? kLn2 * (ua - lg_z) : 0.0f;
  const bool learns = asked && live && open_t;
  const float adv = a.advantage[row], beta = a.beta;
  if (g.segment() == 0 && lane == 0) {
    if (a.loss) a.loss[row] = learns ? fmaf(-adv, logp, -beta * h) : 0.0f;
    if (a.logp) a.logp[row] = !asked ? 0.0f : live ? logp : -INFINITY;
    if (a.entropy) a.entropy[row] = h;
  }
  if (!a.grad || !fits) return;
  T* out = static_cast<T*>(a.grad) + at.out;
  const float gt = learns ? (a.row_weight ? a.row_weight[row] : 1.0f) / t_row : 0.0f;
  const float over = gt * inv_z;
  const float B = over * beta * kLn2, C = over * fmaf(beta, h - kLn2 * lg_z, adv);
  const bool quick = plain && fabsf(B) < 10.0f;
  RowWriter<T> writer(out, n, lane, i0);
  const unsigned long long sc2 = pack2(sc, sc), off2 = pack2(off, off), B2 = pack2(B, B), C2 = pack2(C, C);
#pragma unroll
  for (int c = 0; c < NV; c++) {
    const int i = i0 + c * 32 * V;
    uint32_t d[4];
    if (quick) {
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const unsigned long long u = fma2(pack2(entry<T>(v[c], e), entry<T>(v[c], e + 1)), sc2, off2);
        const Pair up = unpack2(u);
        const Pair r = unpack2(mul2(pack2(exp2_fast(up.x), exp2_fast(up.y)), fma2(u, B2, C2)));
        set2<T>(d, e, r.x, r.y);
      }
    } else {
      float f[V];
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float x = entry<T>(v[c], e), u = fmaxf(u_of(x), -2000.0f);
        f[e] = learns && x > Lowest<T>::open_above ? exp2_fast(u) * fmaf(u, B, C) : 0.0f;
      }
#pragma unroll
      for (int e = 0; e < V; e += 2) set2<T>(d, e, f[e], f[e + 1]);
    }
    // the action's entry, and its lane's alone, gets the rest
    if (learns && act - uint32_t(i) < uint32_t(V)) {
      // (in 64 bits: pi - 1 is the row's largest gradient)
      const double pi = double(exp2_fast(ua)) / double(zs.x), scale = double(a.row_weight ? a.row_weight[row] : 1.0f) / t_row;
      const float x = float(scale * fma(double(adv), pi - 1.0, double(beta) * pi * (double(logp) + h)));
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        uint32_t w[4];
        set2<T>(w, e, x, x);
        if (uint32_t(i + e) == act) d[e * int(sizeof(T)) / 4] = first_of<T>(w[e * int(sizeof(T)) / 4], d[e * int(sizeof(T)) / 4]);
        if (uint32_t(i + e + 1) == act) d[(e + 1) * int(sizeof(T)) / 4] = second_of<T>(w[(e + 1) * int(sizeof(T)) / 4], d[(e + 1) * int(sizeof(T)) / 4]);
      }
    }
    writer.put(d, i);
  }
  writer.finish();
}


// The same for longer rows, which stay in shared memory as they were loaded:
// CL CTAs of NT threads a row, each with its segment of 16-byte vectors. The
// loops are rolled (a row in registers would unroll them over its whole length,
// and the instruction cache then bounds them), three CTAs an SM overlap one
// row's loads with another's arithmetic, and the last pass reads the row at the
// gradient's alignment, so that every store is a whole vector.
struct WholeRow {
  float sc, off, m;
  bool plain;
  __device__ float u_of(float f) const { return plain ? fmaf(f, sc, off) : (fminf(f, m) - m) * sc; }
};

// The vector that starts O entries behind w[0]: O of the next one's. O = 0: w itself.
template <typename T, int WORDS>
__device__ __forceinline__ void shifted(const uint4& x, const uint4& y, bool odd, uint32_t* d) {
  const uint32_t a[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
  for (int j = 0; j < 4; j++)
    d[j] = sizeof(T) == 2 && odd ? __byte_perm(a[j + WORDS], a[j + WORDS + 1], 0x5432) : a[j + WORDS];
}

template <typename T, int NT, int CL>
__global__ void __launch_bounds__(NT) k_policy_long(LossArg a, uint32_t seg_vecs) {
  constexpr int V = 16 / int(sizeof(T)), W = NT / 32;
  extern __shared__ uint4 sm_all[];
  uint4* sm = sm_all + 1;  // one vector ahead of the segment and two behind it may be read
  __shared__ typename Group<W, CL>::Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t row = blockIdx.x / CL;
  RowAt at;
  if (!locate(a.r, a.out_pitch, row, lane, &at)) return;
  Group<W, CL> g(sh, lane, warp);
  constexpr float kLn2 = 0.69314718055994530942f, kMost = 3.402823466e38f, floor_v = Floor<T>::value;
  const bool fits = at.n <= a.r.row_len && at.n + V - 1 <= uint64_t(seg_vecs) * V * CL;
  const int n = fits ? int(at.n) : 0;
  const T* in = static_cast<const T*>(a.r.values) + at.in;
  const int shift = int((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
  const int vecs = (n + shift + V - 1) / V;  // of the row, its misaligned ends included
  const int v0 = g.rank * int(seg_vecs);     // this CTA's first
  // one more is loaded where another CTA's segment follows
  const int mine = max(0, min(int(seg_vecs), vecs - v0)), have = max(0, min(int(seg_vecs) + 1, vecs - v0));
  const int i0 = v0 * V - shift;

  // the row, by asynchronous copies that are all in flight at once
  for (int j = tid; j < have; j += NT) {
    const int i = i0 + j * V;
    if (i >= 0 && i + V <= n) {
      cp_async16(sm + j, in + i);
    } else {
      float f[V];
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < V; e++) f[e] = i + e >= 0 && i + e < n ? as_f32(in[i + e]) : floor_v;
#pragma unroll
      for (int e = 0; e < V; e += 2) set2<T>(w, e, f[e], f[e + 1]);
      sm[j] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  // masked entries raised to the floor (a thread's own vectors: no barrier); the largest
  Top<T> highest;
#pragma unroll 4
  for (int j = tid; j < have; j += NT) {
    const uint4 q = sm[j];
    uint32_t w[4] = {q.x, q.y, q.z, q.w};
    highest.raise(w);
    sm[j] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  const float mx = highest.value();
  // the action's value, before anything is written: grad may lie over values
  const uint32_t act = a.actions[row];
  const bool asked = act != kNone;
  const float va = act < uint32_t(n) ? as_f32(in[act]) : floor_v;
  const uint32_t top = g.largest(key_of(fmaxf(mx, floor_v)));
  const bool endless = top == 0xff800000u;  // the row holds +infinity
  const float m = endless ? kMost : value_of(top);
  const float t_row = a.c.row_temperature ? a.c.row_temperature[row] : a.c.temperature;
  const bool open_t = t_row > 0.0f, any = m > Lowest<T>::open_above;
  const float sc = open_t ? 1.44269504088896340736f / t_row : 0.0f;  // log2(e) / T
  const bool plain = !endless && (m - Lowest<T>::open_above) * sc >= 200.0f && fabsf(m * sc) < 1e5f && sc < 1e6f;
  const WholeRow wr{sc, -m * sc, m, plain};
  const unsigned long long sc2 = pack2(sc, sc), off2 = pack2(wr.off, wr.off);

  // Z and S
  float2 zs = make_float2(0.0f, 0.0f);
  if (plain) {
    unsigned long long za[4] = {0ull, 0ull, 0ull, 0ull}, sa[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll 2
    for (int j = tid; j < mine; j += NT) {
      const uint4 q = sm[j];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const unsigned long long u = fma2(pack2(entry<T>(w, e), entry<T>(w, e + 1)), sc2, off2);
        const Pair up = unpack2(u);
        const unsigned long long x = pack2(exp2_fast(up.x), exp2_fast(up.y));
        za[e / 2 & 3] = add2(za[e / 2 & 3], x);
        sa[e / 2 & 3] = fma2(x, u, sa[e / 2 & 3]);
      }
    }
    const Pair z1 = unpack2(add2(add2(za[0], za[1]), add2(za[2], za[3])));
    const Pair s1 = unpack2(add2(add2(sa[0], sa[1]), add2(sa[2], sa[3])));
    zs = make_float2(z1.x + z1.y, s1.x + s1.y);
  } else if (any) {
    double z = 0.0, s = 0.0;
    for (int j = tid; j < mine; j += NT) {
      const uint4 q = sm[j];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float f = entry<T>(w, e);
        if (f > Lowest<T>::open_above) {
          const float u = fmaxf(wr.u_of(f), -2000.0f), x = exp2_fast(u);
          z += double(x);
          s += double(x) * double(u);
        }
      }
    }
    zs = make_float2(float(z), float(s));
  }
  zs = g.pair_sum(zs);

  // the row's answer
  const float ua = wr.u_of(fminf(va, kMost));
  bool live = asked && va > Lowest<T>::open_above && ua * kLn2 >= float(kDropped);
  if (!open_t) {  // temperature 0: the first largest entry alone
    uint32_t first = 0xffffffffu, zero = 0, none = 0;
    for (int j = tid; j < mine; j += NT) {
      const uint4 q = sm[j];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < V; e++)
        if (fminf(entry<T>(w, e), kMost) == m) first = min(first, uint32_t(i0 + j * V + e));
    }
    g.counts(none, first, zero);
    live = asked && any && first == act;
  }
  const float lg_z = any ? log2f(zs.x) : 0.0f, inv_z = any ? 1.0f / zs.x : 0.0f;
  const float h = any && open_t ? kLn2 * (lg_z - zs.y * inv_z) : 0.0f;
  const float logp = open_t ? kLn2 * (ua - lg_z) : 0.0f;
  const bool learns = asked && live && open_t;
  const float adv = a.advantage[row], beta = a.beta;
  if (g.rank == 0 && tid == 0) {
    if (a.loss) a.loss[row] = learns ? fmaf(-adv, logp, -beta * h) : 0.0f;
    if (a.logp) a.logp[row] = !asked ? 0.0f : live ? logp : -INFINITY;
    if (a.entropy) a.entropy[row] = h;
  }
  if (!a.grad || !fits) return;
  T* out = static_cast<T*>(a.grad) + at.out;
  const float rw = a.row_weight ? a.row_weight[row] : 1.0f, gt = learns ? rw / t_row : 0.0f, over = gt * inv_z;
  const float B = over * beta * kLn2, C = over * fmaf(beta, h - kLn2 * lg_z, adv);
  const bool quick = plain && fabsf(B) < 10.0f;
  const unsigned long long B2 = pack2(B, B), C2 = pack2(C, C);
  // Group j of the gradient starts at entry q = i0 + j V + skew of the row, on a
  // 16-byte boundary of out: entries skew.. of vector j and those of j + 1
  // ahead of skew. Groups belong to the CTA that holds their first vector;
  // the first CTA has the one that starts ahead of the row, too.
  const int skew = int((16 - (reinterpret_cast<uintptr_t>(out + i0) & 15)) & 15) / int(sizeof(T));
  const int words = skew * int(sizeof(T)) / 4;
  const bool odd = sizeof(T) == 2 && (skew & 1);
  auto groups = [&](auto w_) {
    constexpr int WORDS = decltype(w_)::value;
#pragma unroll 2
    for (int j = tid - (skew && g.rank == 0 ? 1 : 0); j < mine; j += NT) {
      const int i = i0 + j * V + skew;
      uint32_t w[4], d[4];
      const uint4 x = sm[j];
      shifted<T, WORDS>(x, WORDS || odd ? sm[j + 1] : x, odd, w);
      if (quick) {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const unsigned long long u = fma2(pack2(entry<T>(w, e), entry<T>(w, e + 1)), sc2, off2);
          const Pair up = unpack2(u);
          const Pair r = unpack2(mul2(pack2(exp2_fast(up.x), exp2_fast(up.y)), fma2(u, B2, C2)));
          set2<T>(d, e, r.x, r.y);
        }
      } else {
        float f[V];
#pragma unroll
        for (int e = 0; e < V; e++) {
          const float x = entry<T>(w, e), u = fmaxf(wr.u_of(x), -2000.0f);
          f[e] = learns && x > Lowest<T>::open_above ? exp2_fast(u) * fmaf(u, B, C) : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < V; e += 2) set2<T>(d, e, f[e], f[e + 1]);
      }
      // the action's entry gets the rest, in 64 bits: pi - 1 is the row's largest gradient
      if (learns && act - uint32_t(i) < uint32_t(V)) {
        const double pi = double(exp2_fast(ua)) / double(zs.x), scale = double(rw) / t_row;
        const float x = float(scale * fma(double(adv), pi - 1.0, double(beta) * pi * (double(logp) + h)));
        uint32_t y[4];
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          set2<T>(y, e, x, x);
          constexpr int S = int(sizeof(T));
          if (uint32_t(i + e) == act) d[e * S / 4] = first_of<T>(y[e * S / 4], d[e * S / 4]);
          if (uint32_t(i + e + 1) == act) d[(e + 1) * S / 4] = second_of<T>(y[(e + 1) * S / 4], d[(e + 1) * S / 4]);
        }
      }
      if (i >= 0 && i + V <= n) {
        __stcs(reinterpret_cast<uint4*>(out + i), make_uint4(d[0], d[1], d[2], d[3]));
      } else {
#pragma unroll
        for (int e = 0; e < V; e++)
          if (i + e >= 0 && i + e < n) out[i + e] = from_f32<T>(entry<T>(d, e));
      }
    }
  };
  switch (words) {
    case 0: groups(std::integral_constant<int, 0>{}); break;
    case 1: groups(std::integral_constant<int, 1>{}); break;
    case 2: groups(std::integral_constant<int, 2>{}); break;
    default: groups(std::integral_constant<int, 3>{}); break;
  }
}

}  // namespace pol
}  // namespace kc
