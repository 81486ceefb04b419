// cache_attend.cuh — attention and pointer scores of questions over the bank
// cache, on the tiles of cache_tile.cuh; instantiated by question type
// (cache_attend_f32.cu, _f16.cu, _bf16.cu).
//
// Attention. With s_j the scores in units of log 2, b_j their mask entries and
// vs_j = f_j 2^e_j the value scales,
//   t_j = (b_j - B) + s_j + e_j,  B the largest b_j,  M the largest t_j,
//   x_j = 2^(t_j - M + 8),  l = sum x_j 2^-e_j,  o = sum (x_j f_j) code_j,  out = o / l.
// The value scales' exponents are in the maximum, so that the weights x_j f_j that
// are rounded to f16 lie below 2^15 whatever the scales are, and a large scale
// that the mask or its score puts out of the running does not push the others
// below f16's range. Subtracting B first keeps the digits of masks far from 0.
// B, M, l and o run over a warp's cells, then over the warps that share a row, then
// over the parts that a long sequence is cut into. Within a warp M is left alone
// while no score lies more than 6 binary orders above it, and B within 32, so that
// most cells take a vote in place of the rows' maxima.
//
// The general form. x_j leaves f32 where t_j lies more than 134 below M. While all
// e_j lie in -40 .. 24 (rows whose largest value is 1e-10 to 2e9) a row whose x_j is
// lost has less than 2^-70 of the sum; rows of zeros count as -40, any exponent is
// theirs. From the first cell with another scale on (the vote on M finds it), or for
// questions whose scores two multiplications do not give (cache_tile.cuh), a warp
// takes its cells in a form of two exponentials a score: rows of zeros are left out
// of M, and the sums have a maximum of their own,
//   l = sum 2^((b_j - B) + s_j - L),  L the largest exponent.
// Sums that meet, of warps or parts, bring their L (M - 8 where there is none).
//
// Small weights. The least step of f16's pieces is 2^-24, so that x_j f_j is rounded
// to 2^-33 of 2^M at the finest. (The general form with weights brought up cell by
// cell, from 8192 rows a warp on, took 3.9 ms where this takes 2.2: 200 banks of
// 30000 rows, 64 f32 questions.)
//
// A cell's bytes are read once by the team of warps that needs them, by 16-byte
// asynchronous copies two cells ahead (one in masked calls of wide heads).
//
// Measured (B200, whole calls): few question rows are bound by memory: single bf16
// tokens of 32 sequences of up to 16384 rows (8 key heads of 128, e4m3) take 115 us,
// 4.9 TB/s; one f16 token over 400003 rows 55 us, of which the parts 42 (5.2 TB/s).
// Many are bound by their instructions, 400 to 900 a cell and warp, and the few
// warps that hide their latency (2.3 to 2.4 of 4 a cycle with 4 warps a scheduler;
// most stalls wait for the instruction before): 64 f32 questions over 64 masked
// banks of 4096 (4 heads of 32) take 183 us, of which the exponentials need 15, the
// tensor cores 30 and the join of the parts takes 14; 4096 banks of 8 to 240 rows
// with 1 to 16 questions 86 us, 2.1 TB/s.
#pragma once
#include <algorithm>
#include <type_traits>

#include "cache_tile.cuh"

namespace kc {
namespace cache {
namespace {

constexpr int kThreads = 256, kWarps = 8;
constexpr float kLift = 8.0f, kSlack = 6.0f, kFar = 32.0f;
constexpr uint32_t kLeastExp = 127 - 40, kMostExp = 127 + 24;  // biased, of the usual value scales

// Cells a ring holds; a masked call's has the mask entries of each warp's rows
// beside them, 36 floats apart so that what a warp reads at once lies on different banks.
constexpr int kMaskPitch = 36;
__host__ __device__ constexpr int mask_bytes(int tiles) { return 8 * tiles * kMaskPitch * 4; }
__host__ __device__ constexpr int stages(int dim, bool masked) { return masked && dim > 32 ? 2 : 3; }

// What a warp needs of one key of a cell: score = product * unit * a + e.
struct KeyInfo {
  float a;   // key scale
  float e;   // exponent of the value scale; -infinity: not attended, or (general form) a row of zeros
  float f;   // value scale / 2^e
  float re;  // 2^-e; 0: not attended
};

// The unit of work a team looks at: a sequence's questions (or one question, with
// a list of its own) against one key head.
struct Unit {
  uint32_t seq, q0, rows, len, blocks, kv, row0;  // row0: the team's first row
  uint64_t stride;                                // of the mask
  const float* mask;                              // of the unit's first question
};

// How a launch's warps are shared out: teams of `mg` warps (8 `tiles` rows each) read
// the same cells, `kg` teams share a unit's cells, a CTA of `warps` warps has hg units.
struct Shape {
  uint32_t tiles, mg, kg, hg, warps, chunks;  // chunks: of 8 tiles mg rows, that a unit may have
  uint64_t items;
};

// Row r of a unit: its question (from the unit's first) and its head of the group.
struct RowId {
  uint32_t question, head;
};
__device__ __forceinline__ RowId row_id(uint32_t r, uint32_t group) {
  if (group == 1) return RowId{r, 0};  // the same for all: no division
  const uint32_t q = r / group;
  return RowId{q, r - q * group};
}

__device__ __forceinline__ bool unit_of(const AttendArg& a, const Shape& sh, uint32_t item, Unit* u) {
  if (item >= sh.items) return false;
  const uint32_t group = a.a.heads / a.c.heads, rest = item / a.c.heads;
  u->kv = item - rest * a.c.heads;
  const uint32_t which = sh.chunks == 1 ? rest : rest / sh.chunks, chunk = rest - which * sh.chunks;
  uint32_t first, count;
  if (a.blocks) {  // a question
    if (a.a.off) {
      if (which < a.a.off[0] || which >= a.a.off[a.t.seqs]) return false;
      u->seq = owner_of(a.a.off, a.t.seqs, which);
      first = uint32_t(a.a.off[u->seq]);
      count = uint32_t(a.a.off[u->seq + 1]) - first;
    } else {
      if (which >= a.t.seqs) return false;
      u->seq = first = which;
      count = 1;
    }
    if (which - first >= a.a.max_q) return false;
    u->q0 = which;
    u->rows = group;
  } else {  // a sequence
    u->seq = which;
    first = a.a.off ? uint32_t(a.a.off[which]) : which;
    const uint64_t end = a.a.off ? a.a.off[which + 1] : which + 1;
    count = uint32_t(end - first);
    u->q0 = first;
    u->rows = min(count, a.a.max_q) * group;
  }
  if (first >= a.a.questions) return false;
  u->rows = min(u->rows, (a.a.questions - u->q0) * group);
  u->row0 = chunk * 8 * sh.tiles * sh.mg;
  if (u->row0 >= u->rows) return false;
  u->len = length_of(a.t, u->seq);
  u->blocks = (u->len + kPage - 1) / kPage;
  u->stride = 0;
  u->mask = nullptr;
  if (a.mask) {
    u->stride = (a.mask_off[u->seq + 1] - a.mask_off[u->seq]) / count;
    u->mask = a.mask + a.mask_off[u->seq] + (u->q0 - first) * u->stride;
  }
  return true;
}

// What is known of a row's scores, as the warps of a row, or the parts of a
// sequence, are joined: [B, M, l, L] and o. The sum of the exponentials is
// l 2^(B + L), what they weigh o 2^(B + M - 8).
struct Stat {
  float b, m, l, low;
};
__device__ __forceinline__ Stat nothing() { return Stat{-INFINITY, -INFINITY, 0.0f, -INFINITY}; }
__device__ __forceinline__ Stat stat_at(const float* p) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  return v.z > 0.0f ? Stat{v.x, v.y, v.z, v.w} : nothing();
}
__device__ __forceinline__ float4 packed(const Stat& s) { return make_float4(s.b, s.m, s.l, s.low); }
// x 2^d where the product is in f32's range, though 2^d may not be.
__device__ __forceinline__ float times_ex2(float x, float d) {
  const float y = ex2(0.5f * d);
  return x * y * y;
}

// The Stats of `width` neighbouring lanes (a power of two) as one, and what this
// lane's o is multiplied by. The largest L does for the joined sum: the largest sum
// is at least 2^(L - 16), since M - 8 lies 16 above its sum's logarithm at most.
__device__ __forceinline__ Stat joined(const Stat& s, uint32_t width, float* weight) {
  Stat all = s;
  for (uint32_t o = width / 2; o; o >>= 1) all.b = fmaxf(all.b, __shfl_xor_sync(0xffffffffu, all.b, o));
  const bool some = s.l > 0.0f;
  const float up = some ? s.b - all.b : 0.0f;
  all.m = up + s.m;
  all.low = up + s.low;
  for (uint32_t o = width / 2; o; o >>= 1) {
    all.m = fmaxf(all.m, __shfl_xor_sync(0xffffffffu, all.m, o));
    all.low = fmaxf(all.low, __shfl_xor_sync(0xffffffffu, all.low, o));
  }
  *weight = s.m == -INFINITY ? 0.0f : ex2(up + (s.m - all.m));
  all.l = some ? times_ex2(s.l, up + (s.low - all.low)) : 0.0f;
  for (uint32_t o = width / 2; o; o >>= 1) all.l += __shfl_xor_sync(0xffffffffu, all.l, o);
  return all;
}

template <typename T, int FMT>
__device__ __forceinline__ void put(const AttendArg& a, uint64_t question, uint32_t head, uint32_t dim, float o, const Stat& s) {
  static_cast<T*>(a.out)[question * a.out_pitch + uint64_t(head) * a.c.dim + dim] =
      from_f32<T>(s.l > 0.0f ? times_ex2(o * (1.0f / s.l), s.m - kLift - s.low) : 0.0f);
}
__device__ __forceinline__ void put_lse(const AttendArg& a, uint64_t question, uint32_t head, const Stat& s) {
  if (a.lse) a.lse[question * a.a.heads + head] = s.l > 0.0f ? (s.b + s.low) * kLn2 + logf(s.l) : -INFINITY;
}

// Part `part` of a row's results in the workspace: o [dim], then B, M, l, L.
__device__ __forceinline__ float* part_of(const AttendArg& a, uint64_t question, uint32_t head, uint32_t part) {
  return a.work + ((question * a.a.heads + head) * a.splits + part) * (a.c.dim + 4);
}

// The largest of a tile row's values: over the lanes of one c.
__device__ __forceinline__ float row_most(float x) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

// N values of a row, one after another; wide: the place is 16-byte aligned.
template <typename T, int N>
__device__ __forceinline__ void put_run(T* dst, const float (&x)[N], bool wide) {
  constexpr int bytes = N * int(sizeof(T));
  if (wide) {
    alignas(16) T y[N];
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = from_f32<T>(x[i]);
    if constexpr (bytes % 16 == 0) {
#pragma unroll
      for (int i = 0; i < bytes / 16; i++) reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(y)[i];
    } else {
      *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) dst[i] = from_f32<T>(x[i]);
  }
}

// The cell's bytes, shared out among the MG warps of a team.
template <int CB, int MG>
__device__ __forceinline__ void copy_cell(uint8_t* dst, const uint8_t* src, uint32_t thread) {
#pragma unroll
  for (int k = 0; k < (CB / 16 + MG * 32 - 1) / (MG * 32); k++) {
    const uint32_t at = thread + k * MG * 32;
    if ((k + 1) * MG * 32 <= CB / 16 || at < CB / 16) copy16(dst + 16 * at, src + 16 * at);
  }
}

// Whether a row of D codes is one of zeros.
template <int D, int FMT>
__device__ __forceinline__ bool zero_row(const uint8_t* codes) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < D / 16; i++) {
    const uint4 w = reinterpret_cast<const uint4*>(codes)[i];
    if (FMT == kI8) any |= (w.x ^ 0x80808080u) | (w.y ^ 0x80808080u) | (w.z ^ 0x80808080u) | (w.w ^ 0x80808080u);
    else any |= (w.x | w.y | w.z | w.w) & 0x7f7f7f7fu;  // 0 and -0
  }
  return any == 0;
}

// f16 pieces of a weight: two for f32 questions (22 bits) and for f16 ones, whose
// output one piece's rounding would reach; bf16 outputs round 8 times more. (With one,
// 7 % of bf16 outputs lie a step from those of f32 weights, with two 0.2 %, both as far
// from the exact ones; two take single tokens from 115 to 119 us, 20 questions of 64
// dims from 109 to 166.)
template <typename T>
__host__ __device__ constexpr int parts_of_weights() { return std::is_same<T, __nv_bfloat16>::value ? 1 : 2; }

// CTAs of 256 threads that an SM should hold at once: what their rings leave room
// for. The registers of most forms then spill: 4 to 76 bytes a thread, 72 to 192 in
// the masked two-tile f32 ones of 32 dims, the masked f32 ones of 64 and the two-tile
// bf16 ones of 64. One CTA less, which spills nothing, is slower all the same: 64
// masked banks of 4096 236 us against 183, 300 banks with 20 bf16 questions of 64
// dims 146 against 109, 512 banks with 8 f32 questions 68 against 60.
__host__ __device__ constexpr int resident(int dim, int tiles, bool masked, int weights) {
  return dim == 128 || (dim == 64 && tiles == 2 && (masked || weights == 2)) ? 1 : dim == 32 && tiles == 1 && !masked ? 3 : 2;
}

template <typename T, int D, int FMT, int NT, bool MASKED>
__global__ __launch_bounds__(kThreads, resident(D, NT, MASKED, parts_of_weights<T>())) void k_attend(AttendArg a, Shape sh) {
  constexpr int S = stages(D, MASKED), CB = int(cell_bytes(D)), MT = D / 16, NB = D / 8, R = 8 * NT;
  constexpr bool kTwo = parts_of_weights<T>() == 2, kApart = sizeof(T) == 4;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ KeyInfo s_info[kWarps][kCell];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const uint32_t team = warp / sh.mg, mi = warp % sh.mg;
  const uint32_t part = blockIdx.y, group = a.a.heads / a.c.heads;
  Unit u{};
  const bool live = unit_of(a, sh, blockIdx.x * sh.hg + (sh.kg == 1 ? team : team / sh.kg), &u);

  Walk w{};
  uint32_t parts = 1;
  if (live) {
    const uint32_t all = a.blocks ? a.block_count : u.blocks;
    parts = max(1u, (all + a.chunk - 1) / a.chunk);
    w.table = a.t.table + uint64_t(u.seq) * a.t.pitch;
    w.list = a.blocks ? a.blocks + (uint64_t(u.q0) * a.c.heads + u.kv) * a.block_count : nullptr;
    w.blocks = u.blocks;
    w.pages = a.c.pages;
    w.b0 = part * a.chunk;
    w.cells = w.b0 < all ? 2 * min(a.chunk, all - w.b0) : 0;
    if (!a.blocks && w.cells)  // a page's second cell may be empty
      w.cells = min(w.cells, (u.len - w.b0 * kPage + kCell - 1) / kCell);
    w.first = team % sh.kg;
    w.step = sh.kg;
  }
  const bool mine = live && part < parts;
  uint32_t n = mine ? w.count() : 0;
  if (n) w.begin();
  // A list ends with its last block that is there (81 sequences of 3 to 32 rows, lists
  // of 32 and 8 heads, a CTA each: 55 us, 67 with the empty entries gone through).
  if (a.blocks && n && n <= 64) {
    const uint32_t late = __ballot_sync(0xffffffffu, w.page[1] != kNone), early = __ballot_sync(0xffffffffu, w.page[0] != kNone);
    n = late ? 64 - __clz(late) : 32 - __clz(early);
  }
  const uint32_t row0 = u.row0 + mi * R;  // the warp's first row
  const uint32_t n_rows = mine && row0 < u.rows ? min(uint32_t(R), u.rows - row0) : 0;

  uint8_t* ring = smem + team * (S * CB);
  uint8_t* biases = smem + sh.warps / sh.mg * (S * CB) + warp * (S * mask_bytes(NT));  // a masked call's
  __shared__ uint64_t s_mask[MASKED ? kWarps : 1][R];  // where the rows' masks begin
  const uint32_t open_end = MASKED ? uint32_t(min(uint64_t(u.len), u.stride)) : u.len;
  bool aligned = false;  // whether every row's mask begins at 16 bytes
  if (MASKED) {
    if (lane < R) s_mask[warp][lane] = uint64_t(row_id(row0 + lane, group).question) * u.stride;
    aligned = (reinterpret_cast<uintptr_t>(u.mask) | u.stride * 4) % 16 == 0;
    // rows that are not there are shut: what a vote sees of them must not change from call to call
    for (uint32_t r = n_rows; r < uint32_t(R); r++)
      for (int k = 0; k < S; k++) reinterpret_cast<float*>(biases + k * mask_bytes(NT))[r * kMaskPitch + lane] = kShut;
    __syncwarp();
  }
  auto issue = [&](uint32_t i, uint32_t page, uint32_t block) {
    if (page != kNone) {
      const uint8_t* src = cell_of<D>(a.c, page, u.kv, w.half(i));
      uint8_t* dst = ring + (i % S) * CB;
      const uint32_t thread = mi * 32 + lane;
      if (sh.mg == 1) copy_cell<CB, 1>(dst, src, thread);
      else if (sh.mg == 2) copy_cell<CB, 2>(dst, src, thread);
      else if (sh.mg == 4) copy_cell<CB, 4>(dst, src, thread);
      else copy_cell<CB, 8>(dst, src, thread);
      if (MASKED) {
        const uint32_t pos = block * kPage + w.half(i) * kCell;  // below 2^32: the length is
        uint8_t* to = biases + (i % S) * mask_bytes(NT);
        if (aligned && pos + kCell <= open_end) {  // 4 rows at a time
#pragma unroll
          for (int r = 0; r < R; r += 4)
            if (uint32_t(r + lane / 8) < n_rows)
              copy16(to + (r + lane / 8) * (4 * kMaskPitch) + 16 * (lane % 8),
                     u.mask + s_mask[warp][r + lane / 8] + pos + 4 * (lane % 8));
        } else {
          const bool in = pos + lane < open_end;
          for (uint32_t r = 0; r < n_rows; r++) {
            uint8_t* dst = to + r * (4 * kMaskPitch) + 4 * lane;
            if (in) copy4(dst, u.mask + s_mask[warp][r] + pos + lane);
            else *reinterpret_cast<float*>(dst) = kShut;
          }
        }
      }
    }
    copy_commit();
  };
  uint32_t ahead[S - 1];  // the pages of the cells that are on their way
  if (n) {
#pragma unroll
    for (uint32_t i = 0; i + 1 < S; i++) {
      ahead[i] = w.page_of(0, i);
      issue(i, ahead[i], w.block_of(0, i));
    }
  }
  QTile<T, D, NT> q;
  bool general = false;  // the form of the cells
  volatile int powers[NT][2];  // of the units; in local memory, the general form's alone
  const bool wide_q = (reinterpret_cast<uintptr_t>(a.a.q) | a.a.pitch * sizeof(T)) % 16 == 0;
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const RowId r = row_id(row0 + 8 * t + g, group);
    const T* at = static_cast<const T*>(a.a.q) + (u.q0 + r.question) * a.a.pitch + (u.kv * group + r.head) * uint64_t(D);
    int power[2];
    general |= q.load(t, uint32_t(8 * t + g) < n_rows ? at : nullptr, wide_q, c, a.scale.m * kLog2e, a.scale.e, power);
    powers[t][0] = power[0];
    powers[t][1] = power[1];
  }

  float o[NT][MT][4], top[NT][2], high[NT][2], sum[NT][2];
#pragma unroll
  for (int t = 0; t < NT; t++) {
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int i = 0; i < 4; i++) o[t][m][i] = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      top[t][h] = MASKED ? -INFINITY : 0.0f;
      high[t][h] = -INFINITY;
      sum[t][h] = 0.0f;
    }
  }
  KeyInfo* info = s_info[warp];
  float low[NT][2];  // L, of the general form
  // Cell i, which has arrived, in the usual form or the general one. False: the
  // usual form does not do for it, and has left it.
  auto take = [&](auto general, uint32_t i, uint32_t page, uint32_t block) -> bool {
    constexpr bool kGeneral = decltype(general)::value;
    if (!n_rows || page == kNone) return true;
    uint8_t* cell = ring + (i % S) * CB;
    const uint64_t pos = uint64_t(block) * kPage + w.half(i) * kCell;
    if (pos >= u.len) return true;
    if (FMT == kE4M3 && pos + kCell > u.len) {
      // bytes behind the sequence's last row may be e4m3's NaN, which no weight of
      // 0 takes away; every warp of a team writes the zeros that it will read
      const uint32_t held = uint32_t(u.len - pos), n16 = (kCell - held) * D / 16;
      for (uint32_t k = lane; k < n16; k += 32) {
        reinterpret_cast<uint4*>(cell + held * D)[k] = uint4{};
        reinterpret_cast<uint4*>(cell + (kCell + held) * D)[k] = uint4{};
      }
      __syncwarp();
    }
    const float* scales = reinterpret_cast<const float*>(cell + 2 * kCell * D);
    bool apart;  // the lane's row has an unusual scale, or is one of zeros
    {
      const float vs = scales[kCell + lane];
      const uint32_t raw = __float_as_uint(vs) >> 23, e = min(max(raw, kGeneral ? 27u : kLeastExp), kGeneral ? 253u : kMostExp);
      const bool open = pos + lane < open_end;
      KeyInfo k;
      k.re = pow2_biased(254u - e);
      k.f = vs * k.re;
      k.a = scales[lane];
      k.e = float(int(e) - 127);
      if (kGeneral && vs == kLeastScale && zero_row<D, FMT>(cell + (kCell + lane) * D)) k.e = -INFINITY;
      apart = open && raw != e;
      if (!open) k = KeyInfo{0.0f, -INFINITY, 0.0f, 0.0f};
      info[lane] = k;
    }
    float s[NT][2][4];
    key_products<T, D, FMT, NT>(q, cell, g, c, s);
    __syncwarp();
    KeyInfo key[4];  // of keys key_of(g) + 8 j
#pragma unroll
    for (int j = 0; j < 4; j++) {
      key[j] = info[8 * j + key_of(g)];
      const Pair ka = pair(key[j].a, key[j].a), ke = pair(key[j].e, key[j].e);
#pragma unroll
      for (int t = 0; t < NT; t++) {
        float* x = &s[t][j / 2][2 * (j % 2)];
        if (kGeneral) {
#pragma unroll
          for (int h = 0; h < 2; h++)
            x[h] = key[j].re == 0.0f ? -INFINITY : far_score(x[h], a.scale.m * kLog2e, powers[t][h], key[j].a);
        } else {
          const float2 y = halves(fma2(mul2(pair(x[0], x[1]), pair(q.unit[t][0], q.unit[t][1])), ka, ke));
          x[0] = y.x;
          x[1] = y.y;
        }
      }
    }
    if (MASKED) {
      const float* bias = reinterpret_cast<const float*>(biases + (i % S) * mask_bytes(NT)) + 2 * c * kMaskPitch + key_of(g);
#pragma unroll
      for (int t = 0; t < NT; t++) {
        float x[4][2], most[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
          for (int j = 0; j < 4; j++) x[j][h] = bias[(8 * t + h) * kMaskPitch + 8 * j];
          // a maximum passes NaN over, where it is not the only one: hence kShut
          most[h] = fminf(fmaxf(fmaxf(fmaxf(kShut, x[0][h]), x[1][h]), fmaxf(x[2][h], x[3][h])), -kBlocked) * kLog2e;
          if (!(most[h] > kBlocked * kLog2e)) most[h] = -INFINITY;
        }
        if (__any_sync(0xffffffffu, most[0] > top[t][0] + kFar || most[1] > top[t][1] + kFar)) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const float was = top[t][h];
            top[t][h] = fmaxf(was, row_most(most[h]));
            if (was != top[t][h]) {  // M is measured from the new one, and L
              high[t][h] = was == -INFINITY ? -INFINITY : high[t][h] + (was - top[t][h]);
              if (kGeneral) low[t][h] = was == -INFINITY ? -INFINITY : low[t][h] + (was - top[t][h]);
            }
          }
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const float from = top[t][h] == -INFINITY ? 0.0f : -top[t][h];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            float& y = s[t][j / 2][2 * (j % 2) + h];
            y = x[j][h] > kBlocked ? y + (fminf(x[j][h], -kBlocked) * kLog2e + from) : -INFINITY;  // rounded as top is
          }
        }
      }
    }
    if (kGeneral) {
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          float now = low[t][h];
          now = fmaxf(now, row_most(fmaxf(fmaxf(s[t][0][h], s[t][0][2 + h]), fmaxf(s[t][1][h], s[t][1][2 + h]))));
          if (now > -INFINITY) {
            sum[t][h] *= ex2(low[t][h] - now);
            low[t][h] = now;
          }
#pragma unroll
          for (int j = 0; j < 4; j++) {
            float& y = s[t][j / 2][2 * (j % 2) + h];
            if (y > -INFINITY) sum[t][h] += ex2(y - now);
            y += key[j].e;
          }
        }
    }
    float most[NT][2];
    bool above = apart && !kGeneral;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        most[t][h] = fmaxf(fmaxf(s[t][0][h], s[t][0][2 + h]), fmaxf(s[t][1][h], s[t][1][2 + h]));
        above |= most[t][h] > high[t][h] + kSlack;
      }
    if (__any_sync(0xffffffffu, above)) {
      if (!kGeneral) {  // rows of zeros are taken as they are
        if (apart && scales[kCell + lane] == kLeastScale) apart = !zero_row<D, FMT>(cell + (kCell + lane) * D);
        if (__any_sync(0xffffffffu, apart)) return false;
      }
#pragma unroll
      for (int t = 0; t < NT; t++) {
        float keep[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const float now = fmaxf(high[t][h], row_most(most[t][h]));
          keep[h] = now == high[t][h] ? 1.0f : ex2(high[t][h] - now);
          high[t][h] = now;
          if (!kGeneral) sum[t][h] *= keep[h];
        }
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int k = 0; k < 4; k++) o[t][m][k] *= keep[k % 2];
      }
    }
    // f32 outputs: a cell's products are summed by themselves. The tensor cores'
    // sums truncate, and one sum over 16 cells was off by 1.2e-6, this by 4e-7.
    [[maybe_unused]] float part_o[kApart ? NT : 1][kApart ? MT : 1][4] = {};
#pragma unroll
    for (int v = 0; v < 2; v++) {
      uint32_t hi[NT][2], lo[kTwo ? NT : 1][2];
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const Pair less = pair(high[t][0] == -INFINITY ? 0.0f : kLift - high[t][0],
                               high[t][1] == -INFINITY ? 0.0f : kLift - high[t][1]);
        Pair l = pair(sum[t][0], sum[t][1]);
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const KeyInfo& k = key[2 * v + j];
          const float2 y = halves(add2(pair(s[t][v][2 * j], s[t][v][2 * j + 1]), less));
          const Pair x = pair(ex2(y.x), ex2(y.y));
          if (!kGeneral) l = fma2(x, pair(k.re, k.re), l);
          const Pair w = mul2(x, pair(k.f, k.f));
          const float2 wf = halves(w);
          const uint32_t h = pack(wf.x, wf.y);
          hi[t][j] = transposed(h);
          if (kTwo) {
            const __half2 z = *reinterpret_cast<const __half2*>(&h);
            const float2 rest = halves(fma2(pair(__low2float(z), __high2float(z)), pair(-1.0f, -1.0f), w));
            lo[kTwo ? t : 0][j] = transposed(pack(rest.x, rest.y));
          }
        }
        sum[t][0] = halves(l).x;
        sum[t][1] = halves(l).y;
      }
      if constexpr (kApart) value_products<D, FMT, NT, kTwo>(hi, lo, cell + kCell * D, v, g, c, part_o);
      else value_products<D, FMT, NT, kTwo>(hi, lo, cell + kCell * D, v, g, c, o);
    }
    if constexpr (kApart) {
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            const float2 y = halves(add2(pair(o[t][m][k], o[t][m][k + 1]), pair(part_o[t][m][k], part_o[t][m][k + 1])));
            o[t][m][k] = y.x;
            o[t][m][k + 1] = y.y;
          }
    }
    __syncwarp();
    return true;
  };
  auto arrive = [&](uint32_t i) {  // of the team; cell i + S - 1 is sent for
    w.advance(i);
    copy_wait<S - 2>();
    meet(team, sh.mg);
    const uint32_t page = ahead[0];
#pragma unroll
    for (int k = 0; k + 2 < S; k++) ahead[k] = ahead[k + 1];
    ahead[S - 2] = w.page_of(i, S - 1);  // none behind the last
    issue(i + S - 1, ahead[S - 2], MASKED ? w.block_of(i, S - 1) : 0);
    return page;
  };
  uint32_t i = 0;
  if (general && n) arrive(0);
  for (; i < n && !general; i += !general) {
    const uint32_t page = arrive(i);
    general = !take(std::false_type{}, i, page, w.block_of(i, 0));
  }
  if (general && n) {
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        low[t][h] = high[t][h] - kLift;
        bool some = false;
#pragma unroll
        for (int m = 0; m < MT; m++) some |= o[t][m][h] != 0.0f || o[t][m][2 + h] != 0.0f;
        // a row that has seen rows of zeros alone has no M
        if (!(__ballot_sync(0xffffffffu, some) & (0x11111111u << c))) high[t][h] = -INFINITY;
      }
    for (uint32_t page = w.page_of(i, 0);; page = arrive(i)) {  // the first has arrived
      take(std::true_type{}, i, page, w.block_of(i, 0));
      if (++i == n) break;
    }
  }
  copy_wait<0>();
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) sum[t][h] += __shfl_xor_sync(0xffffffffu, sum[t][h], x);

  auto stat_of = [&](int t, int h) {
    return Stat{top[t][h], high[t][h], sum[t][h], general ? low[t][h] : high[t][h] - kLift};
  };
  if (sh.kg == 1) {  // a row has one warp
    const bool wide = (reinterpret_cast<uintptr_t>(a.out) | a.out_pitch * sizeof(T)) % 16 == 0;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t r = 8 * t + 2 * c + h;
        if (r >= n_rows) continue;
        const RowId id = row_id(row0 + r, group);
        const uint64_t question = u.q0 + id.question;
        const uint32_t head = u.kv * group + id.head;
        const Stat st = stat_of(t, h);
        const float unit = parts > 1 ? 1.0f : st.l > 0.0f ? 1.0f / st.l : 0.0f;
        float run[NB];
#pragma unroll
        for (int k = 0; k < NB; k++) run[k] = o[t][k / 2][2 * (k % 2) + h] * unit;
        if (general && parts == 1) {
#pragma unroll
          for (int k = 0; k < NB; k++) run[k] = st.l > 0.0f ? times_ex2(run[k], st.m - kLift - st.low) : 0.0f;
        }
        if (parts == 1) {
          put_run(static_cast<T*>(a.out) + question * a.out_pitch + head * uint64_t(D) + g * NB, run, wide);
          if (g == 0) put_lse(a, question, head, st);
        } else {
          float* p = part_of(a, question, head, part);
          put_run(p + g * NB, run, true);
          if (g == 0) *reinterpret_cast<float4*>(p + D) = packed(st);
        }
      }
    return;
  }
  // the warps of a row meet in shared memory: [warp][rows][D + 4]
  __syncthreads();
  float* join = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint32_t r = 8 * t + 2 * c + h;
      if (r >= n_rows) continue;
      float* p = join + (warp * R + r) * (D + 4);
      float run[NB];
#pragma unroll
      for (int k = 0; k < NB; k++) run[k] = o[t][k / 2][2 * (k % 2) + h];
      put_run(p + g * NB, run, true);
      if (g == 0) *reinterpret_cast<float4*>(p + D) = packed(stat_of(t, h));
    }
  __syncthreads();
  // the team kgi of a unit's kg takes every kg-th row of its warps'
  const uint32_t kgi = team % sh.kg, base = (team - kgi) * sh.mg + mi;
  for (uint32_t r = kgi; r < n_rows; r += sh.kg) {
    auto at = [&](uint32_t k) { return join + ((base + k * sh.mg) * R + r) * (D + 4); };
    float weight;
    const Stat all = joined(stat_at(at(lane & (sh.kg - 1)) + D), sh.kg, &weight);
    float acc[D / 32] = {};
    for (uint32_t k = 0; k < sh.kg; k++) {
      const float x = __shfl_sync(0xffffffffu, weight, k);
#pragma unroll
      for (int e = 0; e < D / 32; e++) acc[e] = fmaf(x, at(k)[lane + 32 * e], acc[e]);
    }
    const RowId id = row_id(row0 + r, group);
    const uint64_t question = u.q0 + id.question;
    const uint32_t head = u.kv * group + id.head;
    if (parts == 1) {
#pragma unroll
      for (int e = 0; e < D / 32; e++) put<T, FMT>(a, question, head, lane + 32 * e, acc[e], all);
      if (lane == 0) put_lse(a, question, head, all);
    } else {
      float* p = part_of(a, question, head, part);
#pragma unroll
      for (int e = 0; e < D / 32; e++) p[lane + 32 * e] = acc[e];
      if (lane == 0) *reinterpret_cast<float4*>(p + D) = packed(all);
    }
  }
}

// The parts of every row of a cut sequence, joined (16384 rows of 4 parts: 14 us,
// launch and latency): `per` warps a question and head, each over its share of the
// parts, 32 at a time (a lane a part for the weights, then a lane a dimension), then
// the warps' sums in their order. It may be launched while the last of k_attend's
// CTAs run, and begins when they have ended.
template <typename T, int D, int FMT>
__global__ __launch_bounds__(kThreads) void k_join(AttendArg a, uint32_t per) {
  __shared__ float s_o[kWarps][D];
  __shared__ Stat s_stat[kWarps];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // before any return: what follows this kernel follows the parts
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t item = blockIdx.x * (kWarps / per) + warp / per, share = warp % per;
  const uint32_t question = item / a.a.heads, head = item % a.a.heads;
  uint32_t seq = question, nth = 0;
  bool live = question < a.a.questions;
  if (a.a.off) {
    live = live && question >= a.a.off[0] && question < a.a.off[a.t.seqs];
    if (live) {
      seq = owner_of(a.a.off, a.t.seqs, question);
      nth = uint32_t(question - a.a.off[seq]);
    }
  }
  live = live && seq < a.t.seqs && nth < a.a.max_q;
  const uint32_t all = !live ? 0 : a.blocks ? a.block_count : (length_of(a.t, seq) + kPage - 1) / kPage;
  const uint32_t parts = (all + a.chunk - 1) / a.chunk;
  live = live && parts > 1;
  // lanes that the parts fill; the others hold them again
  const uint32_t width = a.splits > 16 ? 32 : a.splits > 8 ? 16 : a.splits > 4 ? 8 : a.splits > 2 ? 4 : 2;
  Stat st = nothing();
  float acc[D / 32] = {};
  if (live) {
    const float* p = part_of(a, question, head, 0);
    for (uint32_t k0 = share * 32; k0 < parts; k0 += per * 32) {
      const uint32_t mine = k0 + (lane & (width - 1));
      float add, keep;
      const Stat other = joined(mine < parts ? stat_at(p + uint64_t(mine) * (D + 4) + D) : nothing(), width, &add);
      if (k0 == share * 32) {
        st = other;
      } else {  // lane by lane what is held and what comes
        const bool come = lane & 1;
        st = joined(come ? other : st, 2, &keep);
        add *= __shfl_sync(0xffffffffu, keep, 1);
        keep = __shfl_sync(0xffffffffu, keep, 0);
#pragma unroll
        for (int e = 0; e < D / 32; e++) acc[e] *= keep;
      }
      const uint32_t n = min(32u, parts - k0);
      const float* x = p + uint64_t(k0) * (D + 4) + lane;
#pragma unroll 8
      for (uint32_t k = 0; k < n; k++) {
        const float y = __shfl_sync(0xffffffffu, add, k);
#pragma unroll
        for (int e = 0; e < D / 32; e++) acc[e] = fmaf(y, x[k * (D + 4) + 32 * e], acc[e]);
      }
    }
  }
  if (per > 1) {
#pragma unroll
    for (int e = 0; e < D / 32; e++) s_o[warp][lane + 32 * e] = acc[e];
    if (lane == 0) s_stat[warp] = st;
    __syncthreads();
    if (share) return;
    float weight;
    st = joined(s_stat[warp + (lane & (per - 1))], per, &weight);
#pragma unroll
    for (int e = 0; e < D / 32; e++) acc[e] = 0.0f;
    for (uint32_t k = 0; k < per; k++) {
      const float x = __shfl_sync(0xffffffffu, weight, k);
#pragma unroll
      for (int e = 0; e < D / 32; e++) acc[e] = fmaf(x, s_o[warp + k][lane + 32 * e], acc[e]);
    }
  }
  if (!live) return;
#pragma unroll
  for (int e = 0; e < D / 32; e++) put<T, FMT>(a, question, head, lane + 32 * e, acc[e], st);
  if (lane == 0) put_lse(a, question, head, st);
}

// Tiles of 8 rows a warp has at most: two of wide f32 rows would not fit the registers.
template <typename T, int D>
__host__ __device__ constexpr int most_tiles() { return D > 32 && sizeof(T) == 4 ? 1 : 2; }

inline Shape shape_of(const AttendArg& a, int sms) {
  const uint32_t group = a.a.heads / a.c.heads;
  const uint64_t rows = a.blocks || a.block_count ? group : uint64_t(a.a.max_q) * group;
  const uint64_t units = a.blocks || a.block_count ? a.a.questions : a.t.seqs;
  const uint32_t pages = (a.t.max_len + kPage - 1) / kPage;
  // a short sequence's list is mostly empty (81 of 3 to 32 rows, lists of 32, 8 heads
  // of 32: 21 us, 55 with a CTA for each)
  const uint32_t blocks = a.block_count ? std::min(a.block_count, pages) : pages;
  Shape sh{};
  sh.tiles = rows <= 8 || (a.c.dim > 32 && a.a.dtype == kF32) ? 1 : 2;  // most_tiles
  const uint64_t warps = (rows + 8 * sh.tiles - 1) / (8 * sh.tiles);
  sh.mg = warps <= 1 ? 1 : warps <= 2 ? 2 : warps <= 4 ? 4 : 8;
  sh.chunks = uint32_t((warps + sh.mg - 1) / sh.mg);
  sh.items = units * sh.chunks * a.c.heads;
  // short sequences of many units: a team a unit, in CTAs of 4 warps, which units
  // of one length leave together; else the CTA's teams share one
  const bool small = blocks <= 8 && sh.items * sh.mg >= uint64_t(sms) * 16;
  sh.warps = small && sh.mg <= 4 ? 4 : kWarps;
  sh.kg = small ? 1 : kWarps / sh.mg;
  sh.hg = sh.warps / (sh.mg * sh.kg);
  return sh;
}

__host__ __device__ constexpr size_t attend_smem(int dim, int tiles, bool masked, uint32_t warps, uint32_t teams, bool joins) {
  const size_t ring = size_t(stages(dim, masked)) * (teams * cell_bytes(dim) + (masked ? warps * mask_bytes(tiles) : 0));
  const size_t join = joins ? size_t(kWarps) * 8 * tiles * (dim + 4) * 4 : 0;
  return ring > join ? ring : join;
}

template <typename T, int D, int FMT, int NT>
void attend_rows(const AttendArg& a, const Shape& sh, dim3 grid, cudaStream_t s) {
  const size_t smem = attend_smem(D, NT, a.mask != nullptr, sh.warps, sh.warps / sh.mg, sh.kg > 1);
  if (a.mask) k_attend<T, D, FMT, NT, true><<<grid, sh.warps * 32, smem, s>>>(a, sh);
  else k_attend<T, D, FMT, NT, false><<<grid, sh.warps * 32, smem, s>>>(a, sh);
}

template <typename T, int D, int FMT>
cudaError_t attend_tile(const AttendArg& a, int sms, cudaStream_t s, uint64_t* launches) {
  const Shape sh = shape_of(a, sms);
  const uint64_t ctas = (sh.items + sh.hg - 1) / sh.hg;
  if (ctas == 0) return cudaSuccess;
  if (sh.items > 0x7fffffffull || a.splits > 65535) return cudaErrorInvalidConfiguration;
  const dim3 grid(unsigned(ctas), a.splits);
  constexpr int most = most_tiles<T, D>();
  if (sh.tiles == 1) attend_rows<T, D, FMT, 1>(a, sh, grid, s);
  else attend_rows<T, D, FMT, most>(a, sh, grid, s);
  ++*launches;
  cudaError_t e = cudaGetLastError();
  if (e || a.splits == 1) return e;
  cudaLaunchConfig_t cfg{};
  const uint32_t per = a.splits <= 32 ? 1 : kWarps, rows = kWarps / per;
  cfg.gridDim = dim3((a.a.questions * a.a.heads + rows - 1) / rows);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = early;
  cfg.numAttrs = 1;
  ++*launches;
  return cudaLaunchKernelEx(&cfg, k_join<T, D, FMT>, a, per);
}

// --- pointer scores --------------------------------------------------------------

// 8 questions a warp, a cell at a time; `mg` warps with as many questions more
// share the cells that their team brings, kg teams take turns at a sequence's cells
// (64 f32 questions of 128 a bank of 4096: 8 warps a team; with the cells read once for
// every 16 questions before, 110 us against 81; 72 since the questions are read 4
// elements at once). The products pass through shared
// memory so that masks are read and scores written 32 to a row; the mask's entries
// are on their way while the cell is multiplied. Bound by 540 instructions a cell and
// warp, a quarter of them widening i8 keys, at 2.0 of 4 a cycle.
template <typename T, int D, int FMT>
__global__ __launch_bounds__(kThreads, 2) void k_scores(ScoreArg a, uint32_t mg, uint32_t chunks, uint32_t cells) {
  constexpr int S = 3, KB = int(kCell) * D, CB = KB + int(kCell) * 4;  // keys and their scales
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_tile[kWarps][8][kCell + 1];
  __shared__ int s_power[kWarps][8];  // of the rows' units, where they are far from 1
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const uint32_t team = warp / mg, mi = warp % mg, kg = kWarps / mg;
  const uint32_t seq = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const uint64_t q0 = a.a.off ? a.a.off[seq] : seq, q1 = a.a.off ? a.a.off[seq + 1] : seq + 1;
  const uint32_t count = uint32_t(q1 - q0);
  const uint32_t rows = uint32_t(min(uint64_t(min(count, a.a.max_q)), a.a.questions > q0 ? a.a.questions - q0 : 0));
  if (chunk * 8 * mg >= rows) return;  // the whole CTA
  const uint32_t row0 = (chunk * mg + mi) * 8, n_rows = row0 < rows ? min(8u, rows - row0) : 0;
  const uint64_t stride = (a.off[seq + 1] - a.off[seq]) / count;
  const uint32_t len = uint32_t(min(uint64_t(length_of(a.t, seq)), stride));
  const uint64_t end = (stride + kCell - 1) / kCell;  // cells of the row, those behind the bank's end included
  const uint64_t c0 = uint64_t(blockIdx.y) * cells;
  if (c0 >= end) return;

  Walk w{};
  w.table = a.t.table + uint64_t(seq) * a.t.pitch;
  w.blocks = (len + kPage - 1) / kPage;
  w.pages = a.c.pages;
  w.b0 = uint32_t(c0 / 2);
  // the last part takes what the table does not bound
  w.cells = uint32_t(blockIdx.y + 1 == gridDim.y ? end - c0 : min(uint64_t(cells), end - c0));
  w.first = team;
  w.step = kg;
  const uint32_t n = w.count();
  if (n == 0) return;  // the whole team
  uint8_t* ring = smem + team * (S * CB);
  auto issue = [&](uint32_t i, uint32_t page) {
    if (page != kNone) {
      const uint8_t* src = cell_of<D>(a.c, page, 0, w.half(i));
      uint8_t* dst = ring + (i % S) * CB;
      for (uint32_t k = mi * 32 + lane; k < CB / 16; k += mg * 32) copy16(dst + 16 * k, src + 16 * k + (k < KB / 16 ? 0 : KB));
    }
    copy_commit();
  };
  w.begin();
  uint32_t ahead[S - 1];
#pragma unroll
  for (uint32_t i = 0; i + 1 < S; i++) {
    ahead[i] = w.page_of(0, i);
    issue(i, ahead[i]);
  }
  QTile<T, D, 1> q;
  int power[2];
  const bool far = q.load(0, uint32_t(g) < n_rows ? static_cast<const T*>(a.a.q) + (q0 + row0 + g) * a.a.pitch : nullptr,
                          (reinterpret_cast<uintptr_t>(a.a.q) | a.a.pitch * sizeof(T)) % 16 == 0, c, a.scale.m, a.scale.e, power);
  if (far) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      s_power[warp][2 * c + h] = power[h];
      q.unit[0][h] = 1.0f;
    }
  }
  float (*tile)[kCell + 1] = s_tile[warp];
  const uint64_t at0 = a.off[seq] + row0 * stride;
  for (uint32_t i = 0; i < n; i++) {
    w.advance(i);
    copy_wait<S - 2>();
    meet(team, mg);
    const uint32_t page = ahead[0];
    ahead[0] = ahead[1];
    ahead[1] = w.page_of(i, S - 1);
    issue(i + S - 1, ahead[1]);
    const uint64_t pos = (c0 + w.first + uint64_t(w.step) * i) * kCell + lane;
    const bool there = pos < stride;
    float bias[8];
    if (a.mask) {
      const float* m = a.mask + at0 + pos;
#pragma unroll
      for (int r = 0; r < 8; r++) {
        bias[r] = there && uint32_t(r) < n_rows ? *m : 0.0f;
        m += stride;
      }
    }
    float unit = 0.0f;
    if (page != kNone && n_rows) {
      const uint8_t* cell = ring + (i % S) * CB;
      float s[1][2][4];
      key_products<T, D, FMT, 1>(q, cell, g, c, s);
      unit = reinterpret_cast<const float*>(cell + KB)[lane];
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int h = 0; h < 2; h++) tile[2 * c + h][8 * j + key_of(g)] = s[0][j / 2][2 * (j % 2) + h] * q.unit[0][h];
    }
    __syncwarp();
    if (far) {
      for (int r = 0; r < 8; r++) tile[r][lane] = far_score(tile[r][lane], a.scale.m, s_power[warp][r], unit);
      unit = 1.0f;
    }
    if (there) {
      const bool held = page != kNone && pos < len;
      float* out = a.scores + at0 + pos;
#pragma unroll
      for (int r = 0; r < 8; r++) {
        if (uint32_t(r) < n_rows) {
          float x = kShut;
          if (held && (!a.mask || bias[r] > kBlocked)) x = fmaf(tile[r][lane], unit, a.mask ? fminf(bias[r], -kBlocked) : 0.0f);
          *out = x;
        }
        out += stride;
      }
    }
    __syncwarp();
  }
  copy_wait<0>();
}

template <typename T, int D, int FMT>
cudaError_t scores_tile(const ScoreArg& a, int sms, cudaStream_t s, uint64_t* launches) {
  const uint32_t warps = (a.a.max_q + 7) / 8, mg = warps <= 1 ? 1 : warps <= 2 ? 2 : warps <= 4 ? 4 : 8, kg = kWarps / mg;
  const uint32_t chunks = (warps + mg - 1) / mg;
  const uint64_t ctas = uint64_t(a.t.seqs) * chunks;
  if (ctas > 0x7fffffffull) return cudaErrorInvalidConfiguration;
  // parts of at least a cell a team (two for the pair of a block), for about 8 CTAs
  // an SM; rows may be longer than their bank: the table bounds the parts
  const uint64_t all = uint64_t(a.t.pitch) * 2, least = std::max(2u, kg);
  const uint64_t want = std::max<uint64_t>(1, uint64_t(sms) * 8 / std::max<uint64_t>(1, ctas));
  const uint64_t cells = (std::max<uint64_t>(least, (all + want - 1) / want) + least - 1) / least * least;
  const uint64_t parts = std::max<uint64_t>(1, (all + cells - 1) / cells);
  if (parts > 65535 || cells > 0x7fffffffull) return cudaErrorInvalidConfiguration;
  const size_t smem = size_t(kg) * 3 * (kCell * D + kCell * 4);
  k_scores<T, D, FMT><<<dim3(unsigned(ctas), unsigned(parts)), kThreads, smem, s>>>(a, mg, chunks, uint32_t(cells));
  ++*launches;
  return cudaGetLastError();
}

// --- by type -----------------------------------------------------------------------

template <typename T, int D, int FMT>
cudaError_t prepare_tile() {
  constexpr int most = most_tiles<T, D>();
  auto allow = [](auto kernel, int tiles, bool masked) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                int(attend_smem(D, tiles, masked, kWarps, kWarps, true)));
  };
  cudaError_t e;
  if ((e = allow(k_attend<T, D, FMT, 1, false>, 1, false)) || (e = allow(k_attend<T, D, FMT, 1, true>, 1, true)) ||
      (e = allow(k_attend<T, D, FMT, most, false>, most, false)) || (e = allow(k_attend<T, D, FMT, most, true>, most, true)))
    return e;
  return cudaFuncSetAttribute(k_scores<T, D, FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              int(kWarps * 3 * (kCell * D + kCell * 4)));
}

template <typename T>
cudaError_t prepare_as() {
  cudaError_t e;
  if ((e = prepare_tile<T, 32, kI8>()) || (e = prepare_tile<T, 32, kE4M3>()) || (e = prepare_tile<T, 64, kI8>()) ||
      (e = prepare_tile<T, 64, kE4M3>()) || (e = prepare_tile<T, 128, kI8>()) || (e = prepare_tile<T, 128, kE4M3>()))
    return e;
  return cudaSuccess;
}

template <typename T>
cudaError_t attend_as(const AttendArg& a, int sms, cudaStream_t s, uint64_t* launches) {
  const bool i8 = a.c.format == kI8;
  if (a.c.dim == 32) return i8 ? attend_tile<T, 32, kI8>(a, sms, s, launches) : attend_tile<T, 32, kE4M3>(a, sms, s, launches);
  if (a.c.dim == 64) return i8 ? attend_tile<T, 64, kI8>(a, sms, s, launches) : attend_tile<T, 64, kE4M3>(a, sms, s, launches);
  return i8 ? attend_tile<T, 128, kI8>(a, sms, s, launches) : attend_tile<T, 128, kE4M3>(a, sms, s, launches);
}

template <typename T>
cudaError_t scores_as(const ScoreArg& a, int sms, cudaStream_t s, uint64_t* launches) {
  const bool i8 = a.c.format == kI8;
  if (a.c.dim == 32) return i8 ? scores_tile<T, 32, kI8>(a, sms, s, launches) : scores_tile<T, 32, kE4M3>(a, sms, s, launches);
  if (a.c.dim == 64) return i8 ? scores_tile<T, 64, kI8>(a, sms, s, launches) : scores_tile<T, 64, kE4M3>(a, sms, s, launches);
  return i8 ? scores_tile<T, 128, kI8>(a, sms, s, launches) : scores_tile<T, 128, kE4M3>(a, sms, s, launches);
}

}  // namespace
}  // namespace cache
}  // namespace kc
