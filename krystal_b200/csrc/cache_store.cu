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

// Row i of a Rows: its sequence and position there; false where there is none.
struct Place {
  uint32_t seq;
  int64_t pos;
  uint64_t nth, count;  // the row's number among its sequence's rows of the call, and their number
};
__device__ __forceinline__ bool place_of(const Table& t, const Rows& r, uint64_t i, Place* p) {
  if (i >= r.rows) return false;
  if (r.off) {
    if (i < r.off[0] || i >= r.off[t.seqs]) return false;
    p->seq = owner_of(r.off, t.seqs, i);
    const uint64_t first = r.off[p->seq];
    p->nth = i - first;
    p->count = r.off[p->seq + 1] - first;
  } else {
    if (i >= t.seqs) return false;
    p->seq = uint32_t(i);
    p->nth = 0;
    p->count = 1;
  }
  p->pos = (r.starts ? int64_t(r.starts[p->seq]) : int64_t(t.lengths[p->seq]) - int64_t(p->count)) + int64_t(p->nth);
  return p->pos >= 0 && p->pos < int64_t(uint64_t(t.pitch) * kPage);
}

// N elements from p as one or two 16-byte loads (WIDE: p is aligned to them), or one by one.
template <typename T, int N, bool WIDE>
__device__ __forceinline__ void load(const T* p, float (&x)[N]) {
  if (WIDE) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = to_f32(p[i]);
  }
}

// One warp a page and head: the call's rows of that page quantised into its
// cells, then the bounds of all the rows the page holds. A CTA looks at `chunk`
// source rows and takes the pages whose first new row is among them, so that
// every page has one writer and the pages need not be listed beforehand.
template <typename T, int D, int FMT, bool WIDE>
__global__ __launch_bounds__(kThreads) void k_write(Store c, Table t, Rows r, uint32_t chunk) {
  constexpr int V = 16 / sizeof(T), L = D / V, RP = 32 / L;  // elements a lane, lanes a row, rows a pass
  __shared__ uint32_t s_count, s_seq[kRowsMost], s_pos[kRowsMost], s_new[kRowsMost], s_held[kRowsMost];
  __shared__ uint64_t s_row[kRowsMost];
  if (threadIdx.x == 0) s_count = 0;
  __syncthreads();
  if (threadIdx.x < chunk) {
    const uint64_t i = uint64_t(blockIdx.x) * chunk + threadIdx.x;
    Place p;
    if (place_of(t, r, i, &p)) {
      const uint32_t at = uint32_t(p.pos % kPage);
      if (at == 0 || p.nth == 0) {
        const uint32_t k = atomicAdd(&s_count, 1u);
        s_seq[k] = p.seq;
        s_pos[k] = uint32_t(p.pos);
        s_new[k] = uint32_t(min(uint64_t(kPage - at), min(p.count, r.rows - (i - p.nth)) - p.nth));
        s_held[k] = min(kPage, t.lengths[p.seq] - (uint32_t(p.pos) - at));
        s_row[k] = i;
      }
    }
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (uint32_t item = warp; item < s_count * c.heads; item += kWarps) {
    const uint32_t k = item / c.heads, head = item % c.heads;
    const uint32_t page = t.table[uint64_t(s_seq[k]) * t.pitch + s_pos[k] / kPage];
    if (page >= c.pages) continue;
    const uint32_t first = s_pos[k] % kPage, n = s_new[k];
    uint8_t* cells = cell_of<D>(c, page, head, 0);
    for (uint32_t j0 = 0; j0 < n; j0 += RP) {
      const uint32_t j = j0 + lane / L, b = (lane % L) * V;
      const bool there = j < n;
      const uint32_t row = first + j;
      uint8_t* cell = cells + (row / kCell) * cell_bytes(D);
#pragma unroll
      for (int which = 0; which < 2; which++) {
        float x[V];
        float top = 0.0f;
        if (there)
          load<T, V, WIDE>(static_cast<const T*>(which ? r.values : r.keys) + (s_row[k] + j) * r.pitch + head * D + b, x);
#pragma unroll
        for (int i = 0; i < V; i++) {
          x[i] = there ? tame(x[i]) : 0.0f;
          top = fmaxf(top, fabsf(x[i]));
        }
#pragma unroll
        for (int o = 1; o < L; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float scale = fmaxf(__fdiv_rn(top, FMT == kI8 ? kTopI8 : kTopE4M3), kLeastScale);
        uint32_t w[V / 4] = {};
#pragma unroll
        for (int i = 0; i < V; i++) w[i / 4] |= encode<FMT>(x[i], scale) << (8 * (i % 4));
        if (there) {
          const uint32_t rc = row % kCell;
          uint32_t* dst = reinterpret_cast<uint32_t*>(cell + which * kCell * D + (which ? value_at<D>(rc, b) : key_at<D>(rc, b)));
#pragma unroll
          for (int i = 0; i < V / 4; i++) dst[i] = w[i];
          if (lane % L == 0) reinterpret_cast<float*>(cell + 2 * kCell * D)[which * kCell + rc] = scale;
        }
      }
    }
    __syncwarp();
    // the bounds, from the codes as stored: 16 dimensions a lane
    constexpr int LB = D / 16;
    float lo[16], hi[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      lo[i] = __int_as_float(0x7f800000);
      hi[i] = -lo[i];
    }
    const uint32_t held = s_held[k], b = (lane % LB) * 16;
    for (uint32_t row = lane / LB; row < held; row += 32 / LB) {
      const uint8_t* cell = cells + (row / kCell) * cell_bytes(D);
      const uint4 v = *reinterpret_cast<const uint4*>(cell + key_at<D>(row % kCell, b));
      const float scale = reinterpret_cast<const float*>(cell + 2 * kCell * D)[row % kCell];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const float y = decode<FMT>((w[i / 4] >> (8 * (i % 4))) & 0xffu) * scale;
        lo[i] = fminf(lo[i], y);
        hi[i] = fmaxf(hi[i], y);
      }
    }
    float* bounds = c.bounds + (uint64_t(page) * c.heads + head) * 2 * D;
#pragma unroll
    for (int i = 0; i < 16; i++) {
#pragma unroll
      for (int o = LB; o < 32; o <<= 1) {
        lo[i] = fminf(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], o));
        hi[i] = fmaxf(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], o));
      }
      if (lane < LB) {
        bounds[b + i] = lo[i];
        bounds[D + b + i] = hi[i];
      }
    }
  }
}

// Rows read back: a CTA looks up where `chunk` rows lie, then its threads copy
// 16 bytes of output each; rows that the sequence does not hold are 0.
template <typename T, int D, int FMT, bool WIDE>
__global__ __launch_bounds__(kThreads) void k_read(Store c, Table t, Rows r, uint32_t chunk) {
  constexpr int V = 16 / sizeof(T), L = D / V;
  __shared__ uint64_t s_cell[kRowsMost];  // the cell of the row's first head
  __shared__ uint32_t s_at[kRowsMost];    // its row there; kNone: zeros, kNone - 1: not a row of the call
  const uint64_t row0 = uint64_t(blockIdx.x) * chunk;
  if (threadIdx.x < chunk) {
    Place p;
    const uint64_t i = row0 + threadIdx.x;
    const bool mine = i < r.rows && (r.off ? i >= r.off[0] && i < r.off[t.seqs] : i < t.seqs);
    uint32_t at = mine ? kNone : kNone - 1;
    uint64_t cell = 0;
    if (place_of(t, r, i, &p) && p.pos < int64_t(t.lengths[p.seq])) {
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
  const uint32_t n = chunk * c.heads * L;
  for (uint32_t e = threadIdx.x; e < n; e += kThreads) {
    const uint32_t b = e % L * V, head = e / L % c.heads, j = e / (L * c.heads);
    const uint32_t at = s_at[j];
    if (at == kNone - 1) continue;
    const uint8_t* cell = c.cells + (s_cell[j] + head * 2) * cell_bytes(D);
#pragma unroll
    for (int which = 0; which < 2; which++) {
      T* dst = static_cast<T*>(which ? r.values : r.keys);
      if (!dst) continue;
      dst += (row0 + j) * r.pitch + head * D + b;
      T out[V];
      uint32_t w[V / 4] = {};
      float scale = 0.0f;
      if (at != kNone) {
        const uint32_t* src =
            reinterpret_cast<const uint32_t*>(cell + which * kCell * D + (which ? value_at<D>(at, b) : key_at<D>(at, b)));
#pragma unroll
        for (int i = 0; i < V / 4; i++) w[i] = src[i];
        scale = reinterpret_cast<const float*>(cell + 2 * kCell * D)[which * kCell + at];
      }
#pragma unroll
      for (int i = 0; i < V; i++)
        out[i] = from_f32<T>(at == kNone ? 0.0f : decode<FMT>((w[i / 4] >> (8 * (i % 4))) & 0xffu) * scale);
      if (WIDE) {
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(out);
      } else {
#pragma unroll
        for (int i = 0; i < V; i++) dst[i] = out[i];
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

// The `left` largest of n keys (left < n) of one question, by one warp: a radix
// select, 8 bits a pass from the highest bit in which two keys differ, until a
// bin is taken whole. An entry is taken if its key's known bits lie above
// limit's, or equal them and it is among the first `ties` that do.
struct Cut {
  unsigned long long known, limit;
  uint32_t ties;
};
__device__ __forceinline__ Cut cut_of(const unsigned long long* key, uint32_t n, uint32_t left, uint32_t* bin, uint32_t lane) {
  unsigned long long both = ~0ull, any = 0;
  for (uint32_t b = lane; b < n; b += 32) {
    both &= key[b];
    any |= key[b];
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    both &= __shfl_xor_sync(0xffffffffu, both, o);
    any |= __shfl_xor_sync(0xffffffffu, any, o);
  }
  if (both == any) return Cut{~0ull, any, left};  // all are equal
  int shift = 64 - __clzll(static_cast<long long>(both ^ any)) - 8;  // of the 8 bits that begin with the first that differs
  if (shift < 0) shift = 0;
  Cut c{shift + 8 < 64 ? ~0ull << (shift + 8) : 0ull, 0, left};
  c.limit = any & c.known;
  for (;;) {
#pragma unroll
    for (int i = 0; i < 8; i++) bin[lane * 8 + i] = 0;
    __syncwarp();
    for (uint32_t b = lane; b < n; b += 32)
      if ((key[b] & c.known) == c.limit) atomicAdd(&bin[uint32_t(key[b] >> shift) & 255u], 1u);
    __syncwarp();
    uint32_t own[8], sum = 0;  // lane 0 has the highest bins
#pragma unroll
    for (int i = 0; i < 8; i++) sum += own[i] = bin[255 - (lane * 8 + i)];
    uint32_t upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= uint32_t(o)) upto += y;
    }
    const uint32_t who = __ffs(__ballot_sync(0xffffffffu, upto >= c.ties)) - 1;
    uint32_t above = upto - sum, pick = 0, held = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (!found && above + own[i] >= c.ties) {
        found = true;
        pick = 255 - (lane * 8 + i);
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
    __syncwarp();
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
// memory of the CTA that selects for the question, a warp a question. The newest
// blocks are the sequence's last, so they follow whatever is selected.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void k_blocks(BlockArg a, uint32_t ask, uint32_t chunks, uint32_t most) {
  extern __shared__ unsigned long long s_key[];  // [questions of this CTA][most]
  __shared__ double s_q[kAsk][2][D];
  __shared__ uint32_t s_bin[kWarps][256];
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
  const uint32_t part = lane & 3;
  for (uint32_t b0 = (rank * kWarps + warp) * 8; b0 < scored; b0 += ctas * kWarps * 8) {
    const uint32_t b = b0 + lane / 4;
    const uint32_t page = b < scored ? a.t.table[uint64_t(seq) * a.t.pitch + b] : kNone;
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
  const uint32_t k = rank + ctas * warp;
  if (k >= nq) return;
  const unsigned long long* key = s_key + uint64_t(warp) * most;
  uint32_t* out = a.blocks + ((row0 + k) * a.c.heads + head) * a.count;
  const uint32_t under = (1u << lane) - 1;
  uint32_t at = 0;
  if (scored == 0) {  // all that there are
    for (uint32_t b = lane; b < n; b += 32) out[b] = b;
    at = n;
  } else {
    if (a.count > last) {
      const Cut c = cut_of(key, scored, a.count - last, s_bin[warp], lane);
      uint32_t even = 0;
      for (uint32_t b0 = 0; b0 < scored; b0 += 32) {
        const uint32_t b = b0 + lane;
        const unsigned long long x = b < scored ? key[b] & c.known : 0;
        const bool tie = b < scored && x == c.limit, more = b < scored && x > c.limit;
        const uint32_t ties = __ballot_sync(0xffffffffu, tie);
        const bool take = more || (tie && even + __popc(ties & under) < c.ties);
        const uint32_t took = __ballot_sync(0xffffffffu, take);
        if (take) out[at + __popc(took & under)] = b;
        at += __popc(took);
        even += __popc(ties);
      }
    }
    for (uint32_t b = scored + lane; b < n; b += 32) out[at + b - scored] = b;
    at += n - scored;
  }
  for (uint32_t i = at + lane; i < a.count; i += 32) out[i] = kNone;
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
    if (wide) k_write<T, D, FMT, true><<<unsigned(grid), kThreads, 0, s>>>(c, t, r, chunk);
    else k_write<T, D, FMT, false><<<unsigned(grid), kThreads, 0, s>>>(c, t, r, chunk);
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
