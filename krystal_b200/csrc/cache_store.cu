// cache_store.cu — rows quantised into the bank cache, rows read back, and the
// selection of the blocks whose keys can score highest.
#include <cooperative_groups.h>

#include <algorithm>

#include "cache.cuh"

namespace cg = cooperative_groups;

namespace kc {
namespace cache {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr uint32_t kRowsMost = 64;  // source rows a CTA of k_write or k_read looks after

// Where the rows of a chunk lie. Called by a whole CTA, for `chunk` rows from
// `first` on; the first warps fill in the places of a row each.
struct Place {
  uint32_t seq;
  int64_t pos;           // in the sequence
  uint64_t nth, count;   // the row's number among its sequence's rows of the call, and their number
  bool mine, inside;     // a row of the call; at a position that the table has a page for
};
__device__ __forceinline__ Place place_of(const Table& t, const Rows& r, uint64_t first, uint32_t chunk) {
  Place p{};
  const uint64_t i = first + threadIdx.x;
  p.mine = threadIdx.x < chunk && i < r.rows && (r.off ? i >= r.off[0] && i < r.off[t.seqs] : i < t.seqs);
  if (r.off) {
    // the warp's first row by a search, the others among the 32 sequences behind
    // its owner where these reach far enough
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t who = __ballot_sync(0xffffffffu, p.mine);
    if (!who) return p;
    const uint32_t base = owner_of(r.off, t.seqs, __shfl_sync(0xffffffffu, i, __ffs(who) - 1));
    const uint64_t ends = base + 1 + lane <= t.seqs ? r.off[base + 1 + lane] : ~0ull;  // of sequence base + lane
    const bool near = __shfl_sync(0xffffffffu, ends, 31) > __shfl_sync(0xffffffffu, i, 31 - __clz(who));
    uint32_t over = 0;  // sequences of the window that end at or before the row
    if (near) {
#pragma unroll
      for (int k = 16; k; k >>= 1) {
        const uint64_t e = __shfl_sync(0xffffffffu, ends, over + k - 1);
        if (e <= i) over += k;
      }
      p.seq = base + over;
    } else {
      for (int k = 0; k < 32; k++) {
        const uint64_t row = __shfl_sync(0xffffffffu, i, k);
        if (!(who >> k & 1)) continue;
        const uint32_t s = owner_of(r.off, t.seqs, row);
        if (lane == uint32_t(k)) p.seq = s;
      }
    }
    if (p.mine) {
      const uint64_t from = r.off[p.seq];
      p.nth = i - from;
      p.count = r.off[p.seq + 1] - from;
    }
  } else {
    p.seq = uint32_t(i);
    p.count = 1;
  }
  if (p.mine) {
    p.pos = (r.starts ? int64_t(r.starts[p.seq]) : int64_t(t.lengths[p.seq]) - int64_t(p.count)) + int64_t(p.nth);
    p.inside = p.pos >= 0 && p.pos < int64_t(uint64_t(t.pitch) * kPage);
  }
  return p;
}

// Eight elements as they lie, by 16-byte loads (WIDE: aligned to them) or one by one.
template <typename T>
struct Eight {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ float at(int i) const { return to_f32(reinterpret_cast<const T*>(v)[i]); }
};
template <typename T, bool WIDE>
__device__ __forceinline__ Eight<T> load8(const T* p) {
  Eight<T> x;
  if (WIDE) {
#pragma unroll
    for (int i = 0; i < int(sizeof(T) / 2); i++) x.v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) reinterpret_cast<T*>(x.v)[i] = p[i];
  }
  return x;
}

// The largest of N magnitudes; NaN if one is.
__device__ __forceinline__ float most_of(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(fabsf(b)));
  return y;
}

// x / top rounded to f32: q + (x - q top) / top with q = x / top nearly (Markstein).
// Where the remainder would leave f32's range the scale's floor holds anyway.
template <int FMT>
__device__ __forceinline__ float scale_of(float x) {
  constexpr float kTop = FMT == kI8 ? kTopI8 : kTopE4M3, kOver = 1.0f / kTop;
  const float q = x * kOver;
  return fmaxf(fmaf(fmaf(-q, kTop, x), kOver, q), kLeastScale);
}

// N codes of a row, 4 a word. The quotient is
// formed the same way from the rounded reciprocal; for scales so small that the
// remainder could leave f32's range it is the division itself (not for rows of
// zeros, which are common).
template <int FMT, int N>
__device__ __forceinline__ void codes_of(float (&x)[N], float scale, bool zero, uint32_t (&w)[N / 4]) {
  float y[N] = {};
  if (scale > kPlainScale || zero) {
    const float r = __frcp_rn(scale);
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float q = x[i] * r;
      y[i] = fmaf(fmaf(-q, scale, x[i]), r, q);
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < N; i++) {  // the division stands here once, the registers move on past it
      const float q = __fdiv_rn(x[0], scale);
#pragma unroll
      for (int k = 0; k + 1 < N; k++) {
        x[k] = x[k + 1];
        y[k] = y[k + 1];
      }
      y[N - 1] = q;
    }
  }
  if (FMT == kI8) {
    // adding 1.5 * 2^23 leaves the nearest integer, halves to the even, in the low bits
    uint32_t b[N];
#pragma unroll
    for (int i = 0; i < N; i++) b[i] = __float_as_uint(y[i] + (12582912.0f + 128.0f));
#pragma unroll
    for (int p = 0; p < N / 4; p++)
      w[p] = __byte_perm(__byte_perm(b[4 * p], b[4 * p + 1], 0x0040), __byte_perm(b[4 * p + 2], b[4 * p + 3], 0x0040), 0x5410);
  } else {
#pragma unroll
    for (int p = 0; p < N / 4; p++) {
      uint32_t lo, hi;
      asm("{.reg .b16 t; cvt.rn.satfinite.e4m3x2.f32 t, %2, %1; cvt.u32.u16 %0, t;}" : "=r"(lo) : "f"(y[4 * p]), "f"(y[4 * p + 1]));
      asm("{.reg .b16 t; cvt.rn.satfinite.e4m3x2.f32 t, %2, %1; cvt.u32.u16 %0, t;}"
          : "=r"(hi) : "f"(y[4 * p + 2]), "f"(y[4 * p + 3]));
      w[p] = __byte_perm(lo, hi, 0x5410);
    }
  }
}

// Bounds that take in the 8 keys' dimensions of two words of codes.
template <int FMT>
__device__ __forceinline__ void widen_bounds(const uint32_t (&w)[2], float scale, float (&lo)[8], float (&hi)[8]) {
#pragma unroll
  for (int p = 0; p < 2; p++) {
    float v[4];
    values_of<FMT>(w[p], v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      lo[4 * p + i] = fminf(lo[4 * p + i], v[i] * scale);
      hi[4 * p + i] = fmaxf(hi[4 * p + i], v[i] * scale);
    }
  }
}

// One warp the keys or the values of a page and head: the call's rows of that page
// quantised into its cells and, with the keys, the bounds of all the rows the page
// holds. A CTA looks at `chunk` source rows and takes the pages whose first new row
// is among them, so that every page has one writer and the pages need not be listed
// beforehand; where pages are few, several CTAs share them, each some of the heads.
// kAhead passes of 8 elements a lane are on their way together (4 a lane took twice
// the instructions for f32), and no code of the call's rows is read again.
// 507 000 f32 rows of 4 heads of 32: 159 us, 4.2 TB/s; 250 000 bf16 rows of 8 heads
// of 128 to e4m3: 481 us, 3.2 TB/s. About 20 instructions an element (the quotient, the
// code, its value again for the bounds) take half of that; the warps wait for memory
// first, and the registers leave room for 38 % of them.
constexpr int kWriteThreads = 128;

template <typename T, int D, int FMT, bool WIDE>
__global__ __launch_bounds__(kWriteThreads, 7) void k_write(Store c, Table t, Rows r, uint32_t chunk) {
  constexpr int V = 8, L = D / V, RP = 32 / L;  // elements a lane, lanes a row, rows a pass
  constexpr int kAhead = sizeof(T) == 4 ? 2 : 4;
  __shared__ uint32_t s_count, s_seq[kRowsMost], s_pos[kRowsMost], s_new[kRowsMost];
  __shared__ uint64_t s_row[kRowsMost];
  if (threadIdx.x == 0) s_count = 0;
  __syncthreads();
  if (threadIdx.x < (chunk + 31) / 32 * 32) {
    const uint64_t i0 = uint64_t(blockIdx.x) * chunk;
    const Place p = place_of(t, r, i0, chunk);
    const uint32_t at = uint32_t(p.pos % kPage);
    if (p.inside && (at == 0 || p.nth == 0)) {
      const uint32_t k = atomicAdd(&s_count, 1u);
      s_seq[k] = p.seq;
      s_pos[k] = uint32_t(p.pos);
      s_new[k] = uint32_t(min(uint64_t(kPage - at), min(p.count, r.rows - (i0 + threadIdx.x - p.nth)) - p.nth));
      s_row[k] = i0 + threadIdx.x;
    }
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t b = (lane % L) * V, sub = lane / L, items = s_count * c.heads * 2;
  for (uint32_t item = warp * gridDim.y + blockIdx.y; item < items; item += kWriteThreads / 32 * gridDim.y) {
    const uint32_t which = item & 1u, k = item / 2 / c.heads, head = item / 2 - k * c.heads;
    const uint32_t page = t.table[uint64_t(s_seq[k]) * t.pitch + s_pos[k] / kPage];
    if (page >= c.pages) continue;
    const uint32_t first = s_pos[k] % kPage, n = s_new[k];
    uint8_t* cells = cell_of<D>(c, page, head, 0);
    const T* from = static_cast<const T*>(which ? r.values : r.keys) + s_row[k] * r.pitch + head * D + b;
    float lo[V], hi[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
      lo[i] = __int_as_float(0x7f800000);
      hi[i] = -lo[i];
    }
    for (uint32_t j0 = 0; j0 < n; j0 += RP * kAhead) {
      Eight<T> raw[kAhead];
#pragma unroll
      for (int x = 0; x < kAhead; x++) {
        const uint32_t j = j0 + x * RP + sub;
        raw[x] = j < n ? load8<T, WIDE>(from + j * r.pitch) : Eight<T>{};
      }
#pragma unroll
      for (int x = 0; x < kAhead; x++) {
        if (j0 + x * RP >= n) break;
        const uint32_t j = j0 + x * RP + sub, row = first + j, rc = row % kCell;
        float y[V], top = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++) {
          y[i] = raw[x].at(i);
          top = most_of(top, y[i]);
        }
        if (!(top <= kMostValue)) {
          top = 0.0f;
#pragma unroll
          for (int i = 0; i < V; i++) {
            y[i] = tame(y[i]);
            top = fmaxf(top, fabsf(y[i]));
          }
        }
#pragma unroll
        for (int o = 1; o < L; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float scale = scale_of<FMT>(top);
        uint32_t w[V / 4];
        codes_of<FMT, V>(y, scale, top == 0.0f, w);
        if (j < n) {
          uint8_t* cell = cells + (row / kCell) * cell_bytes(D);
          uint8_t* dst = cell + (which ? kCell * D + value_at<D>(rc, b) : key_at<D>(rc, b));
          *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
          if (lane % L == 0) reinterpret_cast<float*>(cell + 2 * kCell * D)[which * kCell + rc] = scale;
          if (!which) widen_bounds<FMT>(w, scale, lo, hi);
        }
      }
    }
    if (which) continue;
    // rows that the page held before
    constexpr int kBack = 8;
    for (uint32_t r0 = 0; r0 < first; r0 += RP * kBack) {
      uint32_t w[kBack][V / 4];
      float scale[kBack];
#pragma unroll
      for (int x = 0; x < kBack; x++) {
        const uint32_t row = min(r0 + x * RP + sub, first - 1);  // the last one again where there is none
        const uint8_t* cell = cells + (row / kCell) * cell_bytes(D);
        const uint2 v = *reinterpret_cast<const uint2*>(cell + key_at<D>(row % kCell, b));
        w[x][0] = v.x;
        w[x][1] = v.y;
        scale[x] = reinterpret_cast<const float*>(cell + 2 * kCell * D)[row % kCell];
      }
#pragma unroll
      for (int x = 0; x < kBack; x++) widen_bounds<FMT>(w[x], scale[x], lo, hi);
    }
    float* bounds = c.bounds + (uint64_t(page) * c.heads + head) * 2 * D;
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
      for (int o = L; o < 32; o <<= 1) {
        lo[i] = fminf(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], o));
        hi[i] = fmaxf(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], o));
      }
    if (lane < L) {
#pragma unroll
      for (int p = 0; p < V / 4; p++) {
        *reinterpret_cast<float4*>(bounds + b + 4 * p) = make_float4(lo[4 * p], lo[4 * p + 1], lo[4 * p + 2], lo[4 * p + 3]);
        *reinterpret_cast<float4*>(bounds + D + b + 4 * p) = make_float4(hi[4 * p], hi[4 * p + 1], hi[4 * p + 2], hi[4 * p + 3]);
      }
    }
  }
}

// Rows read back: a CTA looks up where `chunk` rows lie, then its threads copy 16
// bytes of output each, of kAhead places at a time; rows that the sequence does
// not hold are 0. Memory bounds it: the rows above come back at 4.9 and 6.1 TB/s.
template <typename T, int D, int FMT, bool WIDE>
__global__ __launch_bounds__(kThreads) void k_read(Store c, Table t, Rows r, uint32_t chunk) {
  constexpr int V = 16 / sizeof(T), L = D / V, kAhead = 4;
  __shared__ uint64_t s_cell[kRowsMost];  // the cell of the row's first head
  __shared__ uint32_t s_at[kRowsMost];    // its row there; kNone: zeros, kNone - 1: not a row of the call
  const uint64_t row0 = uint64_t(blockIdx.x) * chunk;
  if (threadIdx.x < (chunk + 31) / 32 * 32) {
    const Place p = place_of(t, r, row0, chunk);
    uint32_t at = p.mine ? kNone : kNone - 1;
    uint64_t cell = 0;
    if (p.inside && p.pos < int64_t(t.lengths[p.seq])) {
      const uint32_t page = t.table[uint64_t(p.seq) * t.pitch + uint64_t(p.pos) / kPage];
      if (page < c.pages) {
        at = uint32_t(p.pos % kCell);
        cell = uint64_t(page) * c.heads * 2 + uint32_t(p.pos % kPage) / kCell;
      }
    }
    s_at[threadIdx.x] = at;
    s_cell[threadIdx.x] = cell;
  }
  __syncthreads();
  // a warp takes 32 / L heads or rows at a time: a place is (row, head), L lanes each
  const uint32_t b = threadIdx.x % L * V, lanes = kThreads / L, places = chunk * c.heads;
  for (uint32_t p0 = threadIdx.x / L; p0 < places; p0 += lanes * kAhead) {
    uint32_t w[kAhead][2][V / 4];
    float scale[kAhead][2];
    T* to[kAhead][2];
#pragma unroll
    for (int x = 0; x < kAhead; x++) {
      const uint32_t p = p0 + x * lanes, j = p / c.heads, head = p - j * c.heads;
      const uint32_t at = p < places ? s_at[j] : kNone - 1;
      const uint64_t dst = (row0 + j) * r.pitch + head * D + b;
      to[x][0] = at == kNone - 1 || !r.keys ? nullptr : static_cast<T*>(r.keys) + dst;
      to[x][1] = at == kNone - 1 || !r.values ? nullptr : static_cast<T*>(r.values) + dst;
      const uint8_t* cell = c.cells + (at < kCell ? s_cell[j] + head * 2 : 0) * cell_bytes(D);
#pragma unroll
      for (int which = 0; which < 2; which++) {
        scale[x][which] = 0.0f;
#pragma unroll
        for (int i = 0; i < V / 4; i++) w[x][which][i] = FMT == kI8 ? 0x80808080u : 0u;
        if (at < kCell && to[x][which]) {
          const uint8_t* src = cell + which * kCell * D + (which ? value_at<D>(at, b) : key_at<D>(at, b));
          if constexpr (V == 4) {
            w[x][which][0] = __ldcs(reinterpret_cast<const uint32_t*>(src));
          } else {
            const uint2 v = __ldcs(reinterpret_cast<const uint2*>(src));
            w[x][which][0] = v.x;
            w[x][which][V / 4 - 1] = v.y;
          }
          scale[x][which] = reinterpret_cast<const float*>(cell + 2 * kCell * D)[which * kCell + at];
        }
      }
    }
#pragma unroll
    for (int x = 0; x < kAhead; x++)
#pragma unroll
      for (int which = 0; which < 2; which++) {
        if (!to[x][which]) continue;
        alignas(16) T out[V];
#pragma unroll
        for (int i = 0; i < V / 4; i++) {
          float value[4];
          values_of<FMT>(w[x][which][i], value);
#pragma unroll
          for (int e = 0; e < 4; e++) out[4 * i + e] = from_f32<T>(value[e] * scale[x][which]);
        }
        if (WIDE) {
          __stcs(reinterpret_cast<uint4*>(to[x][which]), *reinterpret_cast<const uint4*>(out));
        } else {
#pragma unroll
          for (int i = 0; i < V; i++) to[x][which][i] = out[i];
        }
      }
  }
}

// A f64 score as a key that orders as it does; NaN below every number.
__device__ __forceinline__ unsigned long long order_key(double s) {
  if (s != s) return 0;
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(s + 0.0));
  return b >> 63 ? ~b : b | (1ull << 63);
}

constexpr uint32_t kAsk = 8;  // questions of a sequence that a cluster scores at once

// A group of `warps` warps of a CTA that selects for one question: warp `nth` of
// it, lane `lane`, meeting at the named barrier `id`.
struct Group {
  uint32_t id, warps, nth, lane;
  __device__ __forceinline__ void meet() const {
    if (warps == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(warps * 32) : "memory");
  }
};
// What the group shares.
struct Pick {
  uint32_t bin[256];
  unsigned long long both[kWarps], any[kWarps];
  uint32_t more[kWarps], ties[kWarps];
};

// The `left` largest of n keys (left < n) of one question: a radix select, 8 bits a
// pass from the highest bit in which two keys differ, until a bin is taken whole.
// An entry is taken if its key's known bits lie above limit's, or equal them and it
// is among the first `ties` that do.
struct Cut {
  unsigned long long known, limit;
  uint32_t ties;
};
__device__ __forceinline__ Cut cut_of(const unsigned long long* key, uint32_t n, uint32_t left, Pick& p, const Group& g) {
  unsigned long long both = ~0ull, any = 0;
  const uint32_t thread = g.nth * 32 + g.lane, step = g.warps * 32;
  for (uint32_t b = thread; b < n; b += step) {
    both &= key[b];
    any |= key[b];
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    both &= __shfl_xor_sync(0xffffffffu, both, o);
    any |= __shfl_xor_sync(0xffffffffu, any, o);
  }
  if (g.lane == 0) {
    p.both[g.nth] = both;
    p.any[g.nth] = any;
  }
  for (uint32_t i = thread; i < 256; i += step) p.bin[i] = 0;
  g.meet();
  for (uint32_t w = 0; w < g.warps; w++) {
    both &= p.both[w];
    any |= p.any[w];
  }
  if (both == any) return Cut{~0ull, any, left};  // all are equal
  int shift = 64 - __clzll(static_cast<long long>(both ^ any)) - 8;  // of the 8 bits that begin with the first that differs
  if (shift < 0) shift = 0;
  Cut c{shift + 8 < 64 ? ~0ull << (shift + 8) : 0ull, 0, left};
  c.limit = any & c.known;
  for (;;) {
    for (uint32_t b = thread; b < n; b += step)
      if ((key[b] & c.known) == c.limit) atomicAdd(&p.bin[uint32_t(key[b] >> shift) & 255u], 1u);
    g.meet();
    uint32_t own[8], sum = 0;  // lane 0 has the highest bins
#pragma unroll
    for (int i = 0; i < 8; i++) sum += own[i] = p.bin[255 - (g.lane * 8 + i)];
    uint32_t upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
      if (g.lane >= uint32_t(o)) upto += y;
    }
    const uint32_t who = __ffs(__ballot_sync(0xffffffffu, upto >= c.ties)) - 1;
    uint32_t above = upto - sum, pick = 0, held = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (!found && above + own[i] >= c.ties) {
        found = true;
        pick = 255 - (g.lane * 8 + i);
        held = own[i];
      }
      if (!found) above += own[i];
    }
    above = __shfl_sync(0xffffffffu, above, who);
    pick = __shfl_sync(0xffffffffu, pick, who);
    held = __shfl_sync(0xffffffffu, held, who);
    c.ties -= above;
    c.limit = (c.limit & c.known) | (static_cast<unsigned long long>(pick) << shift);
    c.known |= 255ull << shift;
    c.limit &= c.known;
    if (held == c.ties || shift == 0) return c;
    shift = shift > 8 ? shift - 8 : 0;
    g.meet();  // the bins are read
    for (uint32_t i = thread; i < 256; i += step) p.bin[i] = 0;
    g.meet();
  }
}

// The blocks that a question's group of heads looks at: with q+ and q- the sums
// of the heads' positive and negative parts,
//   score_b = sum_d q+_d hi_bd + q-_d lo_bd  >=  sum over heads of any q . k in b.
// Products of two f32 are exact in f64 and the sums differ from the definition's
// by about 1e-15 of their terms, so that the choice is the definition's.
//
// A cluster of CTAs takes up to kAsk questions of a sequence and a key head and
// reads each block's bounds once for them: 4 lanes a block, 16 bytes of the
// smallest and of the largest keys a lane and step, so that 8 blocks of a warp are
// on their way at once. The scores go, as keys that order alike, to the shared
// memory of the CTA that selects for the question, with as many of its warps as the
// other questions leave (64 banks of 4096 with 16 questions: 21 us; 8 histories of
// 131072 with 4 questions on 8 key heads of 128, clusters of 4: 58 us, of which the
// bounds' bytes need 20 and the f64 sums about 15). The newest
// blocks are the sequence's last, so they follow whatever is selected.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void k_blocks(BlockArg a, uint32_t ask, uint32_t chunks, uint32_t most) {
  extern __shared__ unsigned long long s_key[];  // [questions of this CTA][most]
  __shared__ double s_q[kAsk][2][D];
  __shared__ Pick s_pick[kWarps];
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t rank = cluster.block_rank(), ctas = cluster.num_blocks();
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t unit = blockIdx.x / ctas, head = unit % a.c.heads, group = a.a.heads / a.c.heads;
  const uint32_t chunk = unit / a.c.heads % chunks, seq = unit / a.c.heads / chunks;
  const uint64_t q0 = a.a.off ? a.a.off[seq] : seq, q1 = a.a.off ? a.a.off[seq + 1] : seq + 1;
  const uint64_t end = min(min(q0 + a.a.max_q, q1), uint64_t(a.a.questions)), row0 = q0 + chunk * ask;
  if (row0 >= end) return;  // the whole cluster
  const uint32_t nq = uint32_t(min(uint64_t(ask), end - row0));
  const uint32_t n = (length_of(a.t, seq) + kPage - 1) / kPage;
  const uint32_t last = min(a.recent, n), scored = n > a.count ? n - last : 0;  // blocks that have to be scored
  for (uint32_t i = threadIdx.x; i < nq * D; i += kThreads) {
    double up = 0.0, down = 0.0;
    const T* q = static_cast<const T*>(a.a.q) + (row0 + i / D) * a.a.pitch + head * group * uint64_t(D) + i % D;
    for (uint32_t g = 0; g < group; g++) {
      const double x = to_f32(q[g * D]);
      up += x > 0.0 ? x : 0.0;
      down += x > 0.0 ? 0.0 : x;
    }
    s_q[i / D][0][i % D] = up;
    s_q[i / D][1][i % D] = down;
  }
  cluster.sync();
  const uint32_t part = lane & 3, stride = ctas * kWarps * 8;
  const uint32_t* table = a.t.table + uint64_t(seq) * a.t.pitch;
  uint32_t b = (rank * kWarps + warp) * 8 + lane / 4;
  uint32_t ahead = b < scored ? table[b] : kNone;
  for (uint32_t b0 = (rank * kWarps + warp) * 8; b0 < scored; b0 += stride, b += stride) {
    const uint32_t page = ahead;
    ahead = b + stride < scored ? table[b + stride] : kNone;
    const bool there = page < a.c.pages;
    constexpr int F = D / 16;
    float4 lo[F], hi[F];
    const float4* bounds = reinterpret_cast<const float4*>(a.c.bounds + (uint64_t(there ? page : 0) * a.c.heads + head) * 2 * D);
#pragma unroll
    for (int i = 0; i < F; i++) {
      lo[i] = bounds[part + 4 * i];
      hi[i] = bounds[D / 4 + part + 4 * i];
    }
    double score[kAsk] = {};
#pragma unroll
    for (int i = 0; i < F; i++) {
      const double l[4] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w}, h[4] = {hi[i].x, hi[i].y, hi[i].z, hi[i].w};
#pragma unroll
      for (uint32_t k = 0; k < kAsk; k++) {
        if (k >= nq) break;
        const double2* up = reinterpret_cast<const double2*>(&s_q[k][0][4 * (part + 4 * i)]);
        const double2* down = reinterpret_cast<const double2*>(&s_q[k][1][4 * (part + 4 * i)]);
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const double2 u = up[j], w = down[j];
          score[k] = fma(u.x, h[2 * j], fma(w.x, l[2 * j], score[k]));
          score[k] = fma(u.y, h[2 * j + 1], fma(w.y, l[2 * j + 1], score[k]));
        }
      }
    }
#pragma unroll
    for (uint32_t k = 0; k < kAsk; k++) {
      if (k >= nq) break;
      double s = score[k];
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      if (part == k % 4 && b < scored) {
        unsigned long long* to = cluster.map_shared_rank(s_key, k % ctas);
        to[uint64_t(k / ctas) * most + b] = order_key(there ? s : -INFINITY);
      }
    }
  }
  cluster.sync();
  const uint32_t here = rank < nq ? (nq - rank + ctas - 1) / ctas : 0;  // questions of this CTA
  if (here == 0) return;
  Group g{0, here == 1 ? 8u : here == 2 ? 4u : here <= 4 ? 2u : 1u, 0, lane};
  const uint32_t local = warp / g.warps, k = rank + ctas * local;
  if (local >= here) return;
  g.id = 1 + local;
  g.nth = warp % g.warps;
  const unsigned long long* key = s_key + uint64_t(local) * most;
  uint32_t* out = a.blocks + ((row0 + k) * a.c.heads + head) * a.count;
  const uint32_t under = (1u << lane) - 1, thread = g.nth * 32 + lane, step = g.warps * 32;
  uint32_t total = 0;
  if (scored == 0) {  // all that there are
    for (uint32_t x = thread; x < n; x += step) out[x] = x;
    total = n;
  } else {
    total = a.count - last;
    if (total) {
      Pick& p = s_pick[local];
      const Cut c = cut_of(key, scored, total, p, g);
      // each warp takes a run of the blocks; it begins behind what the warps before it take
      const uint32_t run = ((scored + 31) / 32 + g.warps - 1) / g.warps * 32, from = g.nth * run, to = min(from + run, scored);
      uint32_t at = 0, even = 0;
      if (g.warps > 1) {
        uint32_t more = 0, ties = 0;
        for (uint32_t x0 = from; x0 < to; x0 += 32) {
          const unsigned long long x = x0 + lane < to ? key[x0 + lane] & c.known : 0;
          more += __popc(__ballot_sync(0xffffffffu, x0 + lane < to && x > c.limit));
          ties += __popc(__ballot_sync(0xffffffffu, x0 + lane < to && x == c.limit));
        }
        if (lane == 0) {
          p.more[g.nth] = more;
          p.ties[g.nth] = ties;
        }
        g.meet();
        for (uint32_t w = 0; w < g.nth; w++) {
          at += p.more[w];
          even += p.ties[w];
        }
        at += min(even, c.ties);
      }
      for (uint32_t x0 = from; x0 < to; x0 += 32) {
        const unsigned long long x = x0 + lane < to ? key[x0 + lane] & c.known : 0;
        const bool tie = x0 + lane < to && x == c.limit, over = x0 + lane < to && x > c.limit;
        const uint32_t mask = __ballot_sync(0xffffffffu, tie);
        const bool take = over || (tie && even + __popc(mask & under) < c.ties);
        const uint32_t took = __ballot_sync(0xffffffffu, take);
        if (take) out[at + __popc(took & under)] = x0 + lane;
        at += __popc(took);
        even += __popc(mask);
      }
    }
    for (uint32_t x = scored + thread; x < n; x += step) out[total + x - scored] = x;
    total += n - scored;
  }
  for (uint32_t x = total + thread; x < a.count; x += step) out[x] = kNone;
}

template <typename T, int D, int FMT>
cudaError_t store_as(bool write, const Store& c, const Table& t, const Rows& r, int sms, cudaStream_t s) {
  const uint64_t step = 16 / sizeof(T);
  const bool wide = (reinterpret_cast<uintptr_t>(r.keys) | reinterpret_cast<uintptr_t>(r.values)) % 16 == 0 && r.pitch % step == 0;
  // few rows go to many CTAs, many rows 64 to a CTA (a page's worth)
  const uint64_t even = (r.rows + uint64_t(sms) * 8 - 1) / (uint64_t(sms) * 8);
  const uint32_t chunk = uint32_t(std::min<uint64_t>(kRowsMost, std::max<uint64_t>(1, even)));
  const uint64_t grid = (r.rows + chunk - 1) / chunk;
  if (grid > 0x7fffffffull) return cudaErrorInvalidConfiguration;
  if (write) {
    // CTAs that share a chunk's pages: until about 6 an SM have one to write, while
    // each of their 4 warps has something of every page (6700 f16 rows of 8 heads of
    // 64 written and read: 47 us, 66 with one)
    const uint64_t pages = r.rows / kPage + std::min<uint64_t>(t.seqs, r.rows);
    unsigned share = 1;
    while (share * 2 * (kWriteThreads / 32) <= c.heads * 2 && pages * share < uint64_t(sms) * 6) share *= 2;
    if (wide) k_write<T, D, FMT, true><<<dim3(unsigned(grid), share), kWriteThreads, 0, s>>>(c, t, r, chunk);
    else k_write<T, D, FMT, false><<<dim3(unsigned(grid), share), kWriteThreads, 0, s>>>(c, t, r, chunk);
  } else {
    if (wide) k_read<T, D, FMT, true><<<unsigned(grid), kThreads, 0, s>>>(c, t, r, chunk);
    else k_read<T, D, FMT, false><<<unsigned(grid), kThreads, 0, s>>>(c, t, r, chunk);
  }
  return cudaGetLastError();
}

template <typename T, int D>
cudaError_t store_fmt(bool write, const Store& c, const Table& t, const Rows& r, int sms, cudaStream_t s) {
  return c.format == kI8 ? store_as<T, D, kI8>(write, c, t, r, sms, s) : store_as<T, D, kE4M3>(write, c, t, r, sms, s);
}

template <typename T>
cudaError_t store_dim(bool write, const Store& c, const Table& t, const Rows& r, int sms, cudaStream_t s) {
  return c.dim == 32 ? store_fmt<T, 32>(write, c, t, r, sms, s)
       : c.dim == 64 ? store_fmt<T, 64>(write, c, t, r, sms, s) : store_fmt<T, 128>(write, c, t, r, sms, s);
}

cudaError_t store(bool write, const Store& c, const Table& t, const Rows& r, int sms, cudaStream_t s, uint64_t* launches) {
  if (r.rows == 0 || t.seqs == 0) return cudaSuccess;
  ++*launches;
  return r.dtype == kF32 ? store_dim<float>(write, c, t, r, sms, s)
       : r.dtype == kF16 ? store_dim<__half>(write, c, t, r, sms, s) : store_dim<__nv_bfloat16>(write, c, t, r, sms, s);
}

}  // namespace

cudaError_t launch_write(const Store& c, const Table& t, const Rows& r, int sms, cudaStream_t s, uint64_t* launches) {
  return store(true, c, t, r, sms, s, launches);
}

cudaError_t launch_read(const Store& c, const Table& t, const Rows& r, int sms, cudaStream_t s, uint64_t* launches) {
  return store(false, c, t, r, sms, s, launches);
}

namespace {

template <typename T, int D>
cudaError_t blocks_as(const BlockArg& a, int sms, cudaStream_t s) {
  const uint32_t most = std::max(1u, (a.t.max_len + kPage - 1) / kPage);
  uint32_t ask = std::min(kAsk, a.a.max_q);
  while (ask > 1 && uint64_t(ask) * most > kMaxBlocks) ask--;
  const uint32_t chunks = (a.a.max_q + ask - 1) / ask;
  const uint64_t units = uint64_t(a.t.seqs) * chunks * a.c.heads;
  // few units of long sequences: clusters share a unit's blocks, while each CTA
  // has a few rounds of its warps' 8 and there is room for two CTAs an SM
  uint32_t ctas = 1;
  while (ctas < 8 && units * ctas * 2 <= uint64_t(sms) * 2 && most >= ctas * 2 * kWarps * 8 * 2) ctas *= 2;
  if (units * ctas > 0x7fffffffull) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(units * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = size_t((ask + ctas - 1) / ctas) * most * 8;
  cfg.stream = s;
  cudaLaunchAttribute cluster[1];
  cluster[0].id = cudaLaunchAttributeClusterDimension;
  cluster[0].val.clusterDim.x = ctas;
  cluster[0].val.clusterDim.y = cluster[0].val.clusterDim.z = 1;
  cfg.attrs = cluster;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_blocks<T, D>, a, ask, chunks, most);
}

template <typename T>
cudaError_t blocks_dim(const BlockArg& a, int sms, cudaStream_t s) {
  return a.c.dim == 32 ? blocks_as<T, 32>(a, sms, s) : a.c.dim == 64 ? blocks_as<T, 64>(a, sms, s) : blocks_as<T, 128>(a, sms, s);
}

template <typename T>
cudaError_t prepare_blocks() {
  const int most = int(kMaxBlocks) * 8;
  cudaError_t e;
  if ((e = cudaFuncSetAttribute(k_blocks<T, 32>, cudaFuncAttributeMaxDynamicSharedMemorySize, most)) ||
      (e = cudaFuncSetAttribute(k_blocks<T, 64>, cudaFuncAttributeMaxDynamicSharedMemorySize, most)) ||
      (e = cudaFuncSetAttribute(k_blocks<T, 128>, cudaFuncAttributeMaxDynamicSharedMemorySize, most)))
    return e;
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_blocks(const BlockArg& a, int sms, cudaStream_t s, uint64_t* launches) {
  if (a.a.questions == 0 || a.t.seqs == 0) return cudaSuccess;
  ++*launches;
  return a.a.dtype == kF32 ? blocks_dim<float>(a, sms, s)
       : a.a.dtype == kF16 ? blocks_dim<__half>(a, sms, s) : blocks_dim<__nv_bfloat16>(a, sms, s);
}

cudaError_t prepare_store() {
  cudaError_t e;
  if ((e = prepare_blocks<float>()) || (e = prepare_blocks<__half>()) || (e = prepare_blocks<__nv_bfloat16>())) return e;
  return cudaSuccess;
}

}  // namespace cache
}  // namespace kc
