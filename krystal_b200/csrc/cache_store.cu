// cache_store.cu — rows quantised into the bank cache, rows read back, and the
// selection of the blocks whose keys can score highest.
#include <algorithm>

#include "cache.cuh"

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

// The blocks that a question's group of heads looks at: with q+ and q- the sums
// of the heads' positive and negative parts,
//   score_b = sum_d q+_d hi_bd + q-_d lo_bd  >=  sum over heads of any q . k in b.
// Products of two f32 are exact in f64 and the sums differ from the definition's
// by about 1e-15 of their terms, so that the choice is the definition's. One CTA
// a question and key head; the scores stay in shared memory, a radix select finds
// the count-th largest, and what is taken leaves in block order.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_blocks(BlockArg a) {
  extern __shared__ unsigned long long s_key[];
  __shared__ double s_q[2][128];
  __shared__ uint32_t s_bin[256], s_scan[kWarps], s_pick, s_left;
  const uint32_t head = blockIdx.x % a.c.heads, row = blockIdx.x / a.c.heads, d = a.c.dim;
  uint32_t seq = row;
  if (a.a.off) {
    if (row < a.a.off[0] || row >= a.a.off[a.t.seqs]) return;
    seq = owner_of(a.a.off, a.t.seqs, row);
  } else if (row >= a.t.seqs) {
    return;
  }
  const uint32_t n = (length_of(a.t, seq) + kPage - 1) / kPage, group = a.a.heads / a.c.heads;
  for (uint32_t i = threadIdx.x; i < d; i += kThreads) {
    double up = 0.0, down = 0.0;
    for (uint32_t g = 0; g < group; g++) {
      const double q = to_f32(static_cast<const T*>(a.a.q)[row * a.a.pitch + (head * group + g) * uint64_t(d) + i]);
      up += q > 0.0 ? q : 0.0;
      down += q > 0.0 ? 0.0 : q;
    }
    s_q[0][i] = up;
    s_q[1][i] = down;
  }
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < n; b += kThreads) {
    const uint32_t page = a.t.table[uint64_t(seq) * a.t.pitch + b];
    double s = -INFINITY;
    if (b + a.recent >= n) {
      s = INFINITY;
    } else if (page < a.c.pages) {
      const float* lo = a.c.bounds + (uint64_t(page) * a.c.heads + head) * 2 * d;
      s = 0.0;
      for (uint32_t i = 0; i < d; i++)
        s = fma(s_q[0][i], double(lo[d + i]), fma(s_q[1][i], double(lo[i]), s));
    }
    s_key[b] = order_key(s);
  }
  __syncthreads();
  // the radix select: `limit` ends as the count-th largest key, `left` as the
  // number of entries equal to it that are taken
  unsigned long long limit = 0, known = 0;
  uint32_t left = min(a.count, n);
  for (int shift = 56; shift >= 0 && left < n; shift -= 8) {
    s_bin[threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < n; b += kThreads)
      if ((s_key[b] & known) == limit) atomicAdd(&s_bin[uint32_t(s_key[b] >> shift) & 255u], 1u);
    __syncthreads();
    if (threadIdx.x == 0) {
      uint32_t above = 0, bin = 255;
      while (above + s_bin[bin] < left) above += s_bin[bin--];
      s_pick = bin;
      s_left = left - above;
    }
    __syncthreads();
    left = s_left;
    limit |= static_cast<unsigned long long>(s_pick) << shift;
    known |= 255ull << shift;
    __syncthreads();
  }
  uint32_t* out = a.blocks + (uint64_t(row) * a.c.heads + head) * a.count;
  uint32_t at = 0, even = 0;  // taken before, and equal to the limit before
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (uint32_t b0 = 0; b0 < n; b0 += kThreads) {
    const uint32_t b = b0 + threadIdx.x;
    const bool all = a.count >= n;
    const bool tie = b < n && !all && s_key[b] == limit, more = b < n && (all || s_key[b] > limit);
    // ranks by two ballots: ties packed in the high half, the others in the low
    const uint32_t mt = __ballot_sync(0xffffffffu, tie), mm = __ballot_sync(0xffffffffu, more);
    if (lane == 0) s_scan[warp] = (__popc(mt) << 16) | __popc(mm);
    __syncthreads();
    uint32_t before_tie = even, before_more = 0, all_tie = 0, all_more = 0;
    for (uint32_t w = 0; w < kWarps; w++) {
      if (w < warp) before_tie += s_scan[w] >> 16, before_more += s_scan[w] & 0xffffu;
      all_tie += s_scan[w] >> 16;
      all_more += s_scan[w] & 0xffffu;
    }
    const uint32_t under = (1u << lane) - 1;
    before_tie += __popc(mt & under);
    before_more += __popc(mm & under);
    const bool take = more || (tie && before_tie < left);
    // entries taken before this one: those above the limit, and the ties among the first `left`
    const uint32_t rank = at + before_more + (min(before_tie, left) - min(even, left));
    if (take) out[rank] = b;
    at += all_more + (min(even + all_tie, left) - min(even, left));
    even += all_tie;
    __syncthreads();
  }
  for (uint32_t i = min(a.count, n) + threadIdx.x; i < a.count; i += kThreads) out[i] = kNone;
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

cudaError_t launch_blocks(const BlockArg& a, int, cudaStream_t s, uint64_t* launches) {
  if (a.a.questions == 0 || a.t.seqs == 0) return cudaSuccess;
  const size_t smem = size_t((a.t.max_len + kPage - 1) / kPage) * 8;
  const unsigned grid = a.a.questions * a.c.heads;
  ++*launches;
  if (a.a.dtype == kF32) k_blocks<float><<<grid, kThreads, smem, s>>>(a);
  else if (a.a.dtype == kF16) k_blocks<__half><<<grid, kThreads, smem, s>>>(a);
  else k_blocks<__nv_bfloat16><<<grid, kThreads, smem, s>>>(a);
  return cudaGetLastError();
}

cudaError_t prepare_store() {
  cudaError_t e;
  const int most = int(kMaxBlocks) * 8;
  if ((e = cudaFuncSetAttribute(k_blocks<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, most)) ||
      (e = cudaFuncSetAttribute(k_blocks<__half>, cudaFuncAttributeMaxDynamicSharedMemorySize, most)) ||
      (e = cudaFuncSetAttribute(k_blocks<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, most)))
    return e;
  return cudaSuccess;
}

}  // namespace cache
}  // namespace kc
