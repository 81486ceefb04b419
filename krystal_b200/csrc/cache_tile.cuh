// cache_tile.cuh — a warp's question rows, 8 a tile, against a cell of 32 cached
// keys on the tensor cores: fragments of questions and codes, and the walk over a
// sequence's cells. (mma.sync m16n8k16: a serving call has few question rows a
// key, so that the cache's bytes bound it, and 8-bit codes become f16 in
// registers, where these instructions take their operands; 5th-generation ones
// would need them written back to shared memory, for tiles of 64 or 128 rows that
// are mostly empty.)
//
// Keys and values are the 16-row operand A, the questions and the weights the
// 8-column operand B: S^T = K Q^T, O^T = V^T P^T. A single token's few heads then
// fill the tile that 16 rows of questions would leave empty; every code is widened
// once for all of the warp's tiles.
//
// Exactness. Codes are exact in f16. A question row is divided by a power of two
// that brings its largest element into [1, 2); 16-bit questions are then exact
// (bits 2^-25 below the largest aside), f32 ones are the sum of two f16 (22 bits,
// two products). Products accumulate in f32, below 2^17. They are multiplied by the
// row's unit, then by the key's scale; where the unit lies outside 2^-126 .. 2^108
// the exponents of both are added as whole numbers first (times_pow2).
#pragma once
#include "cache.cuh"

namespace kc {
namespace cache {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// D = A B + D, A [16][16] and B [16][8] f16, D f32. Lane (g, c) = (lane / 4,
// lane % 4) holds A's (g, 2c..), (g + 8, 2c..), (g, 2c + 8..), (g + 8, 2c + 8..),
// B's (2c.., g), (2c + 8.., g) and D's (g, 2c), (g, 2c + 1), (g + 8, 2c), (g + 8, 2c + 1).
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Bytes 0 and 1 (HIGH: 2 and 3) of a word of codes as two f16. i8: 0x6400 + byte
// is 1024 + byte, less 1152. e4m3: the instruction for it.
template <int FMT, bool HIGH>
__device__ __forceinline__ uint32_t widen(uint32_t w) {
  if (FMT == kI8) {
    const uint32_t x = __byte_perm(w, 0x64646464u, HIGH ? 0x4342 : 0x4140);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2{__ushort_as_half(0x6480), __ushort_as_half(0x6480)});
    return *reinterpret_cast<const uint32_t*>(&y);
  }
  uint32_t y;
  const unsigned short x = static_cast<unsigned short>(HIGH ? w >> 16 : w);
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(y) : "h"(x));
  return y;
}

// 2^x, x an integer in [-126, 127] given as its biased exponent.
__device__ __forceinline__ float pow2_biased(uint32_t e) { return __uint_as_float(e << 23); }

// x 2^n where the product is in f32's range, though 2^n may not be.
__device__ __forceinline__ float times_pow2(float x, int n) {
  n = min(max(n, -252), 252);
  const int half = n >> 1;
  return x * pow2_biased(uint32_t(127 + half)) * pow2_biased(uint32_t(127 + n - half));
}

// s: a product of a row whose unit is m 2^power, key: the key's scale.
__device__ __forceinline__ float far_score(float s, float m, int power, float key) {
  const uint32_t bits = __float_as_uint(key);
  return times_pow2(s * m * __uint_as_float((bits & 0x007fffffu) | 0x3f800000u), power + int(bits >> 23) - 127);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// An 8 x 8 matrix of f16 transposed over the warp: lane (g, c) gives (g, 2c..),
// and gets (2c.., g).
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// The key of a 16-key group that lane row g (the A operand's row g, or 8 + g less
// 8) stands for: neighbouring rows (2c, 2c + 1) are the keys (c, c + 4), so that
// the four value rows a lane reads with another's are neighbours, and a
// quarter-warp's key rows fall on different banks.
__device__ __forceinline__ uint32_t key_of(int g) { return uint32_t(g >> 1) + (uint32_t(g & 1) << 2); }

// Two f32 in one register pair, and the instructions that take two at once.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves(Pair p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// The B fragments of a warp's question rows, 8 a tile. The dimensions' order
// within a fragment is the keys': lane c's bytes of a key row, 4 a fragment.
template <typename T, int D, int NT>
struct QTile {
  static constexpr bool kTwo = sizeof(T) == 4;  // f32: two f16 a value
  static constexpr int kSteps = D / 16;
  uint32_t hi[NT][kSteps][2], lo[kTwo ? NT : 1][kTwo ? kSteps : 1][2];
  float unit[NT][2];  // what a product of rows 2c and 2c + 1 of a tile is multiplied by
  static constexpr int kLeastPower = -125, kMostPower = 108;  // of two that a unit may hold

  // Dimension of the first of the 4 elements of lane c's piece of fragment s.
  static __device__ __forceinline__ int dim(int s, int c) {
    return D == 32 ? 8 * c + 4 * s : D == 64 ? 16 * c + 4 * s : s < 4 ? 16 * c + 4 * s : 64 + 16 * c + 4 * (s - 4);
  }

  // row: row g of tile t, null where there is none; wide: it begins at 16 bytes, and
  // is read 4 elements at once (515 sequences of 20 questions, 8 heads of 128 in f16
  // over 2: 121 us, 5 more one by one). m 2^e multiplies every score. power: the units
  // are m 2^power; true where a unit does not hold one of the tile's.
  __device__ __forceinline__ bool load(int t, const T* row, bool wide, int c, float m, int e, int (&power)[2]) {
    float x[kSteps][4], top = 0.0f;
#pragma unroll
    for (int s = 0; s < kSteps; s++) {
      alignas(16) T y[4] = {};
      if (row) {
        const T* at = row + dim(s, c);
        if (wide) {
          if constexpr (kTwo) *reinterpret_cast<uint4*>(y) = *reinterpret_cast<const uint4*>(at);
          else *reinterpret_cast<uint2*>(y) = *reinterpret_cast<const uint2*>(at);
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++) y[i] = at[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        x[s][i] = to_f32(y[i]);
        top = fmaxf(top, fabsf(x[s][i]));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t biased = top == 0.0f ? 127u : min(max(__float_as_uint(top) >> 23, 1u), 253u);
    const float down = pow2_biased(254u - biased);
    const int own = int(biased) - 127 + e;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      power[h] = __shfl_sync(0xffffffffu, own, 8 * c + 4 * h);
      unit[t][h] = m * pow2_biased(uint32_t(127 + min(max(power[h], kLeastPower), 127)));
    }
#pragma unroll
    for (int s = 0; s < kSteps; s++)
#pragma unroll
      for (int p = 0; p < 2; p++) {
        const float y0 = x[s][2 * p] * down, y1 = x[s][2 * p + 1] * down;
        hi[t][s][p] = pack(y0, y1);
        if (kTwo) {
          const __half2 h = *reinterpret_cast<const __half2*>(&hi[t][s][p]);
          lo[kTwo ? t : 0][kTwo ? s : 0][p] = pack(y0 - __low2float(h), y1 - __high2float(h));
        }
      }
    return __any_sync(0xffffffffu, own < kLeastPower || own > kMostPower);
  }
};

// The words of one key row that lane c multiplies, a word a fragment.
template <int D>
__device__ __forceinline__ void key_words(const uint8_t* keys, uint32_t row, int c, uint32_t (&w)[D / 16]) {
  if constexpr (D == 32) {
    const uint2 v = *reinterpret_cast<const uint2*>(keys + key_at<D>(row, 8 * c));
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int p = 0; p < D / 64; p++) {
      const uint4 v = *reinterpret_cast<const uint4*>(keys + key_at<D>(row, 64 * p + 16 * c));
      w[4 * p] = v.x; w[4 * p + 1] = v.y; w[4 * p + 2] = v.z; w[4 * p + 3] = v.w;
    }
  }
}

// s[t][u] = keys of 16-key group u of the cell at `keys` times the rows of tile t:
// (key g, rows 2c, 2c + 1), (key g + 8, rows 2c, 2c + 1), keys by key_of.
template <typename T, int D, int FMT, int NT>
__device__ __forceinline__ void key_products(const QTile<T, D, NT>& q, const uint8_t* keys, int g, int c, float (&s)[NT][2][4]) {
#pragma unroll
  for (int u = 0; u < 2; u++) {
    uint32_t w0[D / 16], w1[D / 16];
    key_words<D>(keys, 16 * u + key_of(g), c, w0);
    key_words<D>(keys, 16 * u + 8 + key_of(g), c, w1);
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) s[t][u][i] = 0.0f;
#pragma unroll
    for (int k = 0; k < D / 16; k++) {
      const uint32_t a[4] = {widen<FMT, false>(w0[k]), widen<FMT, false>(w1[k]), widen<FMT, true>(w0[k]), widen<FMT, true>(w1[k])};
#pragma unroll
      for (int t = 0; t < NT; t++) {
        mma(s[t][u], a, q.hi[t][k][0], q.hi[t][k][1]);
        if constexpr (QTile<T, D, NT>::kTwo) mma(s[t][u], a, q.lo[t][k][0], q.lo[t][k][1]);
      }
    }
  }
}

// o += the values of 16-key group u times the weights of the warp's rows (B
// fragments, hi and for f32 questions lo). Rows g and g + 8 of tile m of o stand
// for dimensions (D / 8) g + 2 m and the next.
template <int D, int FMT, int NT, bool TWO>
__device__ __forceinline__ void value_products(const uint32_t (&hi)[NT][2], const uint32_t (&lo)[TWO ? NT : 1][2],
                                               const uint8_t* values, int u, int g, int c, float (&o)[NT][D / 16][4]) {
  constexpr int W = D / 32;  // words of 4 dimensions that a lane reads of each of its keys
  uint32_t w[4][W];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint8_t* p = values + value_at<D>(16 * u + c + 4 * i, 4 * W * g);
    if constexpr (W == 1) {
      w[i][0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (W == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[i][0] = v.x; w[i][1] = v.y;
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
    }
  }
#pragma unroll
  for (int x = 0; x < W; x++)
#pragma unroll
    for (int y = 0; y < 2; y++) {  // bytes 2 y and 2 y + 1 of the word
      const uint32_t p0 = __byte_perm(w[0][x], w[1][x], y ? 0x7362 : 0x5140);
      const uint32_t p1 = __byte_perm(w[2][x], w[3][x], y ? 0x7362 : 0x5140);
      const uint32_t a[4] = {widen<FMT, false>(p0), widen<FMT, true>(p0), widen<FMT, false>(p1), widen<FMT, true>(p1)};
#pragma unroll
      for (int t = 0; t < NT; t++) {
        mma(o[t][2 * x + y], a, hi[t][0], hi[t][1]);
        if constexpr (TWO) mma(o[t][2 * x + y], a, lo[t][0], lo[t][1]);
      }
    }
}

// 16 bytes, global to shared, asynchronous.
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
               ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;"
               ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The warps of a team meet (named barriers 1..8; a team of one needs none).
__device__ __forceinline__ void meet(uint32_t team, uint32_t warps) {
  if (warps == 1) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(warps * 32) : "memory");
}

// The cells a team walks over: cell first + step * i of the blocks from b0 on,
// 32 at a time in the lanes' registers and 32 ahead, so that no copy waits for a
// page number.
struct Walk {
  const uint32_t* table;  // the sequence's pages
  const uint32_t* list;   // the question's blocks, or null: every block in turn
  uint32_t blocks, pages; // of the sequence; of the cache
  uint32_t b0, cells, first, step;
  uint32_t block[2], page[2];

  __device__ __forceinline__ uint32_t count() const { return cells > first ? (cells - first + step - 1) / step : 0; }
  __device__ __forceinline__ uint32_t half(uint32_t i) const { return (first + step * i) & 1u; }
  __device__ __forceinline__ void fetch(uint32_t batch, int which) {
    const uint32_t cell = first + step * (batch * 32 + (threadIdx.x & 31));
    uint32_t b = kNone, p = kNone;
    if (cell < cells) {
      b = b0 + (cell >> 1);
      if (list) b = list[b];
      if (b < blocks) p = table[b];
      if (p >= pages) p = kNone;
    }
    block[which] = b;
    page[which] = p;
  }
  __device__ __forceinline__ void begin() {
    fetch(0, 0);
    fetch(1, 1);
  }
  // At the start of step i: the registers move on with it.
  __device__ __forceinline__ void advance(uint32_t i) {
    if (i && (i & 31u) == 0) {
      block[0] = block[1];
      page[0] = page[1];
      fetch(i / 32 + 1, 1);
    }
  }
  // The page of step i + ahead (kNone: none), where step i is the current one.
  __device__ __forceinline__ uint32_t page_of(uint32_t i, uint32_t ahead) const {
    const uint32_t j = (i & 31u) + ahead;
    return __shfl_sync(0xffffffffu, j < 32 ? page[0] : page[1], j & 31u);
  }
  __device__ __forceinline__ uint32_t block_of(uint32_t i, uint32_t ahead) const {
    const uint32_t j = (i & 31u) + ahead;
    return __shfl_sync(0xffffffffu, j < 32 ? block[0] : block[1], j & 31u);
  }
};

}  // namespace cache
}  // namespace kc
