// policy_whole.cuh — the policy loss where nothing is cut (k_policy_whole,
// k_policy_long); the rows with cuts are policy_cut.cuh's.
#pragma once
#include "policy.cuh"

namespace kc {
namespace pol {

// ---------------------------------------------------------------------------
// The policy loss over the whole softmax, nothing cut: no decision hangs on a
// last bit, so the row stays as it was loaded (a warp's registers, NV 16-byte
// vectors a lane; longer rows: k_policy_long) and its exponentials are f32. With
// u_j = (v_j - m) log2(e) / T, taken as one fma of v_j (the rounding of
// m log2(e) / T is common to all and cancels),
//   Z = sum 2^u, S = sum 2^u u, log pi_j = ln 2 (u_j - log2 Z),
//   H = ln 2 (log2 Z - S / Z), and the gradient is
//   2^u_j (u_j B + C) with B = g beta ln 2 / (T Z), C = g (A + beta (H - ln Z)) / (T Z)
// but for -g A / T more at the action. Sums: four or eight f32 partial sums
// of at most 18 terms a thread, joined by trees. Arithmetic on pairs (f32x2).
// The sums are taken without the action's entry (raised to the masks' floor in
// its place) and its terms added last: with O the others' sum of weights, a
// confident row's log pi(a) = -log1p(O / w_a) and its gradient's pi - 1 = -O / Z
// at the action come without cancellation, to the weights' own accuracy.
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

struct WholeRow {
  float sc, off, m;
  bool plain;
  __device__ float u_of(float f) const { return plain ? fmaf(f, sc, off) : (fminf(f, m) - m) * sc; }
};

// The row's scalars from the others' sums O and S and the action's u (0 weight
// without one): Z, its logarithm and inverse, log pi(a) and H. Where the action
// has half of the mass or more both come from terms that do not cancel,
// H = -pi_a log pi_a - ln 2 (S - O log2 Z) / Z.
struct WholeSums {
  float others, w, lg_z, inv_z, logp, h;
  __device__ __forceinline__ float z() const { return others + w; }
  __device__ __forceinline__ WholeSums(float2 zs, float ua, bool apart, bool any, bool open_t) {
    constexpr float kLn2 = 0.69314718055994530942f;
    others = zs.x;
    ua = apart ? fmaxf(ua, -2000.0f) : 0.0f;  // (a masked action's u is anything)
    w = apart ? exp2_fast(ua) : 0.0f;
    lg_z = any ? log2f(z()) : 0.0f;
    inv_z = any ? rcp_fast(z()) : 0.0f;
    logp = open_t ? kLn2 * (ua - lg_z) : 0.0f;
    h = any && open_t ? kLn2 * (lg_z - fmaf(w, ua, zs.y) * inv_z) : 0.0f;
    if (apart && others <= w) {
      logp = -log1pf(others * rcp_fast(w));
      h = fmaf(kLn2 * inv_z, fmaf(others, lg_z, -zs.y), -w * inv_z * logp);
    }
  }
};

// log2(e) / T; a T below 5e-39 keeps it finite, so that the largest entry's u is 0.
__device__ __forceinline__ float scale_of(float t) { return fminf(1.44269504088896340736f / t, 3.402823466e38f); }

// The gradient entry by entry in 64 bits: where a factor of the quick form
// could overflow before the product does, and at the action.
struct WholeSlope {
  float rw, t, adv, beta;
  const WholeSums& s;
  __device__ __forceinline__ float of(float u) const {
    const double w = double(exp2_fast(u)), e = 0.69314718055994530942 * (double(u) - double(s.lg_z)) + double(s.h);
    return float(double(rw) / double(t) * (w / double(s.z()) * fma(double(beta), e, double(adv))));
  }
  __device__ __forceinline__ float of_action() const {
    const double w = double(s.w), o = double(s.others);
    return float(double(rw) * (double(beta) * w * (double(s.logp) + double(s.h)) - double(adv) * o) / (double(t) * (o + w)));
  }
};

template <typename T, int NV>
__global__ void __launch_bounds__(128) k_policy_whole(LossArg a) {
  constexpr int V = 16 / int(sizeof(T));
  constexpr uint32_t kCap = uint32_t(32) * V * NV;
  const int lane = threadIdx.x & 31;
  const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= a.r.rows) return;
  RowAt at;
  if (!locate(a.r, a.out_pitch, row, lane, &at)) return;
  Group<1, 1> g(lane);
  const bool fits = at.n <= a.r.row_len && at.n + V - 1 <= kCap;
  const int n = fits ? int(at.n) : 0;
  const T* in = static_cast<const T*>(a.r.values) + at.in;
  const int shift = int((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
  const int i0 = lane * V - shift;
  constexpr float floor_v = Floor<T>::value;
  const uint32_t act = a.actions[row];

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
  // the action is summed apart
#pragma unroll
  for (int c = 0; c < NV; c++) {
    const uint32_t e = act - uint32_t(i0 + c * 32 * V);
    if (e < uint32_t(V)) set_entry<T>(v[c], e, floor_v);
  }
  // the action's value, before anything is written: grad may lie over values
  const bool asked = act != kNone;
  const float va = act < uint32_t(n) ? as_f32(in[act]) : floor_v;
  constexpr float kLn2 = 0.69314718055994530942f, kMost = 3.402823466e38f;
  const uint32_t top = g.largest(key_of(mx));
  const bool endless = top == 0xff800000u;  // the row holds +infinity
  const float m = endless ? kMost : value_of(top);
  const float t_row = a.c.row_temperature ? a.c.row_temperature[row] : a.c.temperature;
  const bool open_t = t_row > 0.0f, any = m > Lowest<T>::open_above;
  const float sc = open_t ? scale_of(t_row) : 0.0f;
  const bool plain = !endless && (m - Lowest<T>::open_above) * sc >= 200.0f && fabsf(m * sc) < 1e5f && sc < 1e6f;
  const float off = -m * sc;
  const WholeRow row_of{sc, off, m, plain};
  // Z and S of the others
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
          const float u = fmaxf(row_of.u_of(f), -2000.0f), w = exp2_fast(u);
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
  const float ua = row_of.u_of(fminf(va, kMost));
  const WholeSums sums(zs, ua, va > Lowest<T>::open_above, any, open_t);
  bool live = asked && va > Lowest<T>::open_above && ua * kLn2 >= float(kDropped);
  if (!open_t) {  // temperature 0: the first largest entry alone
    uint32_t first = va > Lowest<T>::open_above && fminf(va, kMost) == m ? act : 0xffffffffu;
#pragma unroll
    for (int c = 0; c < NV; c++)
#pragma unroll
      for (int e = 0; e < V; e++)
        if (fminf(entry<T>(v[c], e), kMost) == m) first = min(first, uint32_t(i0 + c * 32 * V + e));
    uint32_t zero = 0, none = 0;
    g.counts(none, first, zero);
    live = asked && any && first == act;
  }
  const float lg_z = sums.lg_z, inv_z = sums.inv_z, h = sums.h, logp = sums.logp;
  const bool learns = asked && live && open_t;
  const float adv = a.advantage[row], beta = a.beta;
  if (lane == 0) {
    if (a.loss) a.loss[row] = learns ? fmaf(-adv, logp, -beta * h) : 0.0f;
    if (a.logp) a.logp[row] = !asked ? 0.0f : live ? logp : -INFINITY;
    if (a.entropy) a.entropy[row] = h;
  }
  if (!a.grad || !fits) return;
  T* out = static_cast<T*>(a.grad) + at.out;
  const float rw = a.row_weight ? a.row_weight[row] : 1.0f;
  const float over = learns ? rw * (kLn2 * sc) * inv_z : 0.0f;  // rw / (T Z), for the quick form alone
  const WholeSlope slope{rw, t_row, adv, beta, sums};
  const float B = over * beta * kLn2, C = learns ? over * fmaf(beta, h - kLn2 * lg_z, adv) : 0.0f;  // (adv may be NaN)
  const bool quick = plain && fabsf(B) < 10.0f && fabsf(C) < 1e30f;  // (a vanished weight times infinity)
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
        const float x = entry<T>(v[c], e);
        f[e] = learns && x > Lowest<T>::open_above ? slope.of(fmaxf(row_of.u_of(x), -2000.0f)) : 0.0f;
      }
#pragma unroll
      for (int e = 0; e < V; e += 2) set2<T>(d, e, f[e], f[e + 1]);
    }
    // the action's entry, and its lane's alone, gets the rest
    if (learns && act - uint32_t(i) < uint32_t(V)) {
      const float x = slope.of_action();
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

// The vector that starts O entries behind w[0]: O of the next one's. O = 0: w itself.
template <typename T, int WORDS>
__device__ __forceinline__ void shifted(const uint4& x, const uint4& y, bool odd, uint32_t* d) {
  const uint32_t a[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
  for (int j = 0; j < 4; j++)
    d[j] = sizeof(T) == 2 && odd ? __byte_perm(a[j + WORDS], a[j + WORDS + 1], 0x5432) : a[j + WORDS];
}

// The same for longer rows, which stay in shared memory as they were loaded:
// CL CTAs of NT threads a row, each with its segment of 16-byte vectors. The
// loops are rolled (a row in registers would unroll them over its whole length,
// and the instruction cache then bounds them), three CTAs an SM overlap one
// row's loads with another's arithmetic, and the last pass reads the row at the
// gradient's alignment, so that every store is a whole vector. 4096 bf16 rows of
// 32001 take 112 to 124 us, 4.2 to 4.7 TB/s, two thirds of the measured copy
// rate: two exponentials an entry keep their pipe busy half the time, and a
// CTA's own load, arithmetic and store follow each other.
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
  const uint32_t act = a.actions[row];

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
  // the action is summed apart
  const int at_act = act < uint32_t(n) ? int(act) - i0 : -1;
  if (at_act >= 0 && at_act < mine * V && at_act / V % NT == tid) {
    const uint4 q = sm[at_act / V];
    uint32_t w[4] = {q.x, q.y, q.z, q.w};
    set_entry<T>(w, uint32_t(at_act % V), floor_v);
    sm[at_act / V] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  // the action's value, before anything is written: grad may lie over values
  const bool asked = act != kNone;
  const float va = act < uint32_t(n) ? as_f32(in[act]) : floor_v;
  const uint32_t top = g.largest(key_of(fmaxf(mx, floor_v)));
  const bool endless = top == 0xff800000u;  // the row holds +infinity
  const float m = endless ? kMost : value_of(top);
  const float t_row = a.c.row_temperature ? a.c.row_temperature[row] : a.c.temperature;
  const bool open_t = t_row > 0.0f, any = m > Lowest<T>::open_above;
  const float sc = open_t ? scale_of(t_row) : 0.0f;
  const bool plain = !endless && (m - Lowest<T>::open_above) * sc >= 200.0f && fabsf(m * sc) < 1e5f && sc < 1e6f;
  const WholeRow wr{sc, -m * sc, m, plain};
  const unsigned long long sc2 = pack2(sc, sc), off2 = pack2(wr.off, wr.off);

  // Z and S of the others
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
  const WholeSums sums(zs, ua, va > Lowest<T>::open_above, any, open_t);
  bool live = asked && va > Lowest<T>::open_above && ua * kLn2 >= float(kDropped);
  if (!open_t) {  // temperature 0: the first largest entry alone
    uint32_t first = va > Lowest<T>::open_above && fminf(va, kMost) == m ? act : 0xffffffffu, zero = 0, none = 0;
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
  const float lg_z = sums.lg_z, inv_z = sums.inv_z, h = sums.h, logp = sums.logp;
  const bool learns = asked && live && open_t;
  const float adv = a.advantage[row], beta = a.beta;
  if (g.rank == 0 && tid == 0) {
    if (a.loss) a.loss[row] = learns ? fmaf(-adv, logp, -beta * h) : 0.0f;
    if (a.logp) a.logp[row] = !asked ? 0.0f : live ? logp : -INFINITY;
    if (a.entropy) a.entropy[row] = h;
  }
  if (!a.grad || !fits) return;
  T* out = static_cast<T*>(a.grad) + at.out;
  const float rw = a.row_weight ? a.row_weight[row] : 1.0f;
  const float over = learns ? rw * (kLn2 * sc) * inv_z : 0.0f;  // rw / (T Z), for the quick form alone
  const WholeSlope slope{rw, t_row, adv, beta, sums};
  const float B = over * beta * kLn2, C = learns ? over * fmaf(beta, h - kLn2 * lg_z, adv) : 0.0f;  // (adv may be NaN)
  const bool quick = plain && fabsf(B) < 10.0f && fabsf(C) < 1e30f;  // (a vanished weight times infinity)
  const unsigned long long B2 = pack2(B, B), C2 = pack2(C, C);
  // Group j of the gradient starts at entry q = i0 + j V + skew of the row, on a
  // 16-byte boundary of out: entries skew.. of vector j and those of j + 1
  // ahead of skew. Groups belong to the CTA that holds their first vector;
  // the first CTA has the one that starts ahead of the row, too.
  const int skew = int((16 - (reinterpret_cast<uintptr_t>(out + i0) & 15)) & 15) / int(sizeof(T));
  const int words = skew * int(sizeof(T)) / 4;
  const bool odd = sizeof(T) == 2 && (skew & 1);
  const int ahead = skew && g.rank == 0 ? 1 : 0;
  auto groups = [&](auto w_, auto quick_) {
    constexpr int WORDS = decltype(w_)::value;
#pragma unroll 2
    for (int j = tid - ahead; j < mine; j += NT) {
      const int i = i0 + j * V + skew;
      uint32_t w[4], d[4];
      const uint4 x = sm[j];
      shifted<T, WORDS>(x, WORDS || odd ? sm[j + 1] : x, odd, w);
      if constexpr (decltype(quick_)::value) {
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
          const float x = entry<T>(w, e);
          f[e] = learns && x > Lowest<T>::open_above ? slope.of(fmaxf(wr.u_of(x), -2000.0f)) : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < V; e += 2) set2<T>(d, e, f[e], f[e + 1]);
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
  auto pass = [&](auto quick_) {  // (two loops: one with the test inside would hold what both need)
    switch (words) {
      case 0: groups(std::integral_constant<int, 0>{}, quick_); break;
      case 1: groups(std::integral_constant<int, 1>{}, quick_); break;
      case 2: groups(std::integral_constant<int, 2>{}, quick_); break;
      default: groups(std::integral_constant<int, 3>{}, quick_); break;
    }
  };
  if (quick) pass(std::true_type{});
  else pass(std::false_type{});
  // the action's entry gets the rest, from the thread that wrote its group
  if (learns) {
    const int to_act = int(act) - i0 - skew + V, j = to_act / V - 1;
    if (to_act >= 0 && j >= -ahead && j < mine && (j + ahead) % NT == tid)
      out[act] = from_f32<T>(slope.of_action());
  }
}

}  // namespace pol
}  // namespace kc
