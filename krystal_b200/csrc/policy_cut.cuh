// policy_cut.cuh — rows with cuts: the draws and the policy loss
// (k_policy_small, k_policy_rows).
//
// What the cuts leave is usually short: a bank's grammar admits few records,
// and top-k and top-p keep few. So a row is gathered into a list in shared
// memory, in bank order, and everything else is done on what it left: rows of
// up to 256 entries always (k_policy_small); longer rows if their open entries,
// or with top-k those at or above a lower bound of the k-th largest, are at
// most kList. One warp finishes a list, one entry a lane and slice of 32
// (ListRow). The lower bound is the k-th largest of the 16-byte vectors'
// maxima: k vectors reach it, so k entries do.
//
// A row whose list would be longer is cut where it was loaded (WideRow): the
// keys of CL CTAs' W warps in shared memory, warp g of the group holding the
// contiguous segment g in chunks of one 16-byte load a lane. Loops over it are
// rolled: keys in registers would unroll every pass over the row's length, and
// fetching those instructions took most of the time. After the cuts each warp
// packs what it kept to the front of its segment, so that the 64-bit weights
// are made for kept entries alone.
#pragma once
#include "policy.cuh"

namespace kc {
namespace pol {

// A list is 8 entries a lane, what one warp holds in registers. Top-k up to
// kListTopK looks for one: the bound admits k entries and those that share
// their vectors, so a k near 256 leaves more than a list (at 200: 217 to 236 of
// 4096 f32 entries, which fit, but 246 to 271 of bf16 ones and over 320 of 1024
// f32 ones) and has counted for nothing. 4096 rows, with the bound and without:
// 4096 f32 at k = 50 89 and 172 us, at 200 101 and 189; 4096 bf16 at 100 89 and
// 157, at 200 171 and 160; 1024 f32 at 100 45 and 67, at 200 83 and 73.
constexpr uint32_t kList = 256;
constexpr uint32_t kListTopK = 208;
// Lists up to this are cut by comparing all pairs. 30000 rows under top-p with
// 32, 64 and 128: of 30 entries 46, 58 and 81 us, of 60 87, 78 and 121, of 120
// 116, 117 and 204.
constexpr int kPairs = 64;
constexpr int kBatch = 8;  // rows a CTA takes up to their lists

struct List {
  uint32_t key[kList], where[kList];  // a key, and its index in the row
  double w[kPairs];
};

// Open entries of a row, their smallest and largest key.
struct Stats {
  uint32_t open, lo, hi;
};

// What turns a row's keys into weights.
struct Scale {
  const Tables& t;
  uint32_t top;    // the largest key
  double m, log_m, inv_t;
  bool power;      // probabilities at a temperature other than 1: x from logarithms
  bool plain_p;    // probabilities at T = 1: the weights are the values

  __device__ explicit Scale(const Tables& tables) : t(tables) {}
  __device__ void begin(const Cut& c, const Stats& s, int kind) {
    plain_p = kind == kKindP && c.inv_t == 1.0;
    power = kind == kKindP && !plain_p;
    inv_t = c.inv_t;
    top = s.open ? s.hi : 0xbf800000u;  // (some number)
    m = double(value_of(top));
    log_m = power ? log_tab(value_of(top), t.c, t.l) : 0.0;
  }
  // The tempered log weight of a key in the support. Every lane of the warp
  // calls this, and weight, together.
  __device__ double x_of(uint32_t key) const {
    const float v = value_of(key);
    return power ? (log_tab(v, t.c, t.l) - log_m) * inv_t : (double(v) - m) * inv_t;
  }
  // x of a key (outside the support: 0), and the weight: 0 for key 0 and for
  // dropped entries.
  __device__ double weight(uint32_t key, double& x) const {
    x = x_of(key ? key : top);
    const bool in = key && x >= kDropped;
    if (!in) x = 0.0;
    const double w = exp64(x, t.e2);
    return in ? w : 0.0;
  }
  __device__ double weight(uint32_t key) const {
    if (plain_p) return key ? double(value_of(key)) : 0.0;
    double x;
    return weight(key, x);
  }
};

// The pivot between two values of a row: halfway in value for scores, halfway
// in exponent and mantissa for probabilities (which span decades); after a
// dozen steps the two alternate, so that no row takes more than about 70 steps
// whatever its values.
__device__ __forceinline__ uint32_t pivot(uint32_t lo, uint32_t hi, int step, int kind) {
  const bool by_value = step < 12 ? kind != kKindP : (step & 1);
  uint32_t p = lo + (hi - lo + 1) / 2;
  if (by_value) p = key_of(0.5f * value_of(lo) + 0.5f * value_of(hi));
  return min(max(p, lo + 1), hi);
}

// A gathered list, by one warp.
template <int S>
struct ListRow : Scale {
  Group<1, 1> g;
  uint32_t k[S];          // keys; 0: not in the support
  int slices;             // in use
  const uint32_t* where;  // the entries' indices in the row

  __device__ ListRow(int lane, const Tables& tables, const List& list, uint32_t n)
      : Scale(tables), g(lane), slices(int((n + 31) / 32)), where(list.where) {
#pragma unroll
    for (int s = 0; s < S; s++) {
      const uint32_t j = uint32_t(s) * 32 + lane;
      k[s] = j < n ? list.key[j] : 0u;
    }
  }
  __device__ uint32_t index(int s) const { return where[s * 32 + g.lane]; }
  // f(slice) for every slice in use; the warp together.
  template <typename F>
  __device__ __forceinline__ void each(F f) {
#pragma unroll
    for (int s = 0; s < S; s++) {
      if (s >= slices) break;
      f(s);
    }
  }
  // f(key) for every entry.
  template <typename F>
  __device__ __forceinline__ void keys(F f) {
    each([&](int s) { f(k[s]); });
  }
  // lo only where the search will need it.
  __device__ Stats stats(uint32_t n, bool need_lo) {
    uint32_t hi = 0u, lo = 0xffffffffu;
    keys([&](uint32_t key) {
      hi = max(hi, key);
      if (key) lo = min(lo, key);
    });
    return Stats{n, need_lo ? __reduce_min_sync(0xffffffffu, lo) : 0u, __reduce_max_sync(0xffffffffu, hi)};
  }
  // Drops the entries below the cut and all but the first `ties` at it.
  __device__ void drop(uint32_t cut, uint32_t ties) {
    uint32_t seen = 0;
    each([&](int s) {
      const uint32_t at = __ballot_sync(0xffffffffu, k[s] == cut);
      const uint32_t rank = seen + __popc(at & ((1u << g.lane) - 1u));
      if (k[s] < cut || (k[s] == cut && rank >= ties)) k[s] = 0u;
      seen += __popc(at);
    });
  }
};

// A row over its group: keys in shared memory.
template <typename T, int W, int CL>
struct WideRow : Scale {
  static constexpr int V = 16 / int(sizeof(T));
  Group<W, CL> g;
  uint4* slab;       // this warp's keys: vector j of chunk c at (c V / 4 + j) 32 + lane
  uint16_t* place;   // the packed entries' places in the segment
  int chunks, base;  // of the warp; the row's index of its first entry
  uint32_t live;     // chunks that hold an entry of the support
  uint32_t kept;     // packed entries of this warp

  __device__ WideRow(typename Group<W, CL>::Shared& sh, const Tables& tables, int lane, int warp, uint4* sm, int n)
      : Scale(tables), g(sh, lane, warp), slab(sm + warp * n * 32 * (V / 4)),
        place(reinterpret_cast<uint16_t*>(sm + W * n * 32 * (V / 4)) + warp * n * 32 * V), chunks(n), live(0), kept(0) {}

  __device__ int at(int c) const { return base + c * 32 * V + g.lane * V; }
  // Until the row is packed, the places' memory holds each vector's largest key.
  __device__ uint32_t* best() const { return reinterpret_cast<uint32_t*>(place); }
  __device__ void get(int c, uint32_t* k) const {
#pragma unroll
    for (int j = 0; j < V / 4; j++) {
      const uint4 q = slab[(c * (V / 4) + j) * 32 + g.lane];
      k[4 * j] = q.x; k[4 * j + 1] = q.y; k[4 * j + 2] = q.z; k[4 * j + 3] = q.w;
    }
  }
  __device__ void put(int c, const uint32_t* k) {
#pragma unroll
    for (int j = 0; j < V / 4; j++)
      slab[(c * (V / 4) + j) * 32 + g.lane] = make_uint4(k[4 * j], k[4 * j + 1], k[4 * j + 2], k[4 * j + 3]);
  }
  // f(chunk, its V keys of this lane) for the chunks that hold any; the warp together.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll 2
    for (int c = 0; c < chunks; c++)
      if (live >> c & 1u) {
        uint32_t k[V];
        get(c, k);
        f(c, k);
      }
  }
  template <typename F>
  __device__ __forceinline__ void keys(F f) const {
    each([&](int, const uint32_t* k) {
#pragma unroll
      for (int e = 0; e < V; e++) f(k[e]);
    });
  }

  // Loads n entries from row, four vectors in flight. A lane's 16-byte loads
  // start on 16-byte boundaries; a vector that reaches past either end of the
  // row is read entry by entry, with NaN, which no support holds, outside.
  __device__ void load(const T* row, int n, int kind) {
    base = g.segment() * 32 * V * chunks - int((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    for (int c0 = 0; c0 < chunks; c0 += 4) {
      uint32_t w[4][4];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int i = at(c0 + u);
        if (i >= 0 && i + V <= n && c0 + u < chunks) {
          const uint4 q = __ldcs(reinterpret_cast<const uint4*>(row + i));
          w[u][0] = q.x; w[u][1] = q.y; w[u][2] = q.z; w[u][3] = q.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) w[u][e] = 0xffffffffu;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int i = at(c0 + u);
        if (c0 + u >= chunks) break;
        if (i + V > 0 && i < n && !(i >= 0 && i + V <= n)) {
          float f[V];
#pragma unroll
          for (int e = 0; e < V; e++) f[e] = i + e >= 0 && i + e < n ? as_f32(row[i + e]) : __uint_as_float(0x7fc00000u);
#pragma unroll
          for (int e = 0; e < V; e += 2) set2<T>(w[u], e, f[e], f[e + 1]);
        }
        uint32_t k[V], most = 0;
#pragma unroll
        for (int e = 0; e < V; e++) most = max(most, k[e] = open_key<T>(entry<T>(w[u], e), kind));
        put(c0 + u, k);
        best()[(c0 + u) * 32 + g.lane] = most;
        if (__any_sync(0xffffffffu, most != 0u)) live |= 1u << (c0 + u);
      }
    }
  }

  __device__ Stats stats() {
    Stats s{0u, 0xffffffffu, 0u};
    keys([&](uint32_t k) {
      s.open += k != 0u;
      if (k) s.lo = min(s.lo, k);
      s.hi = max(s.hi, k);
    });
    g.counts(s.open, s.lo, s.hi);
    return s;
  }

  // A key that at least `want` entries reach, few more: see the head of the file.
  __device__ uint32_t lower_bound(uint32_t want, const Stats& s, int kind) {
    auto reach = [&](uint32_t p) {  // vectors whose largest reaches p
      uint32_t n = 0;
#pragma unroll 4
      for (int c = 0; c < chunks; c++) n += best()[c * 32 + g.lane] >= p;
      return g.total(n);
    };
    if (reach(s.lo) < want) return s.lo;
    uint32_t lo = s.lo, cur = s.hi;  // lo is reached often enough; cur + 1 is not
    for (int step = 0; cur > lo && step < 40; step++) {
      const uint32_t p = pivot(lo, cur, step, kind);
      const uint32_t n = reach(p);
      if (n >= want) {
        lo = p;
        if (n <= want + want / 16 + 4) break;
      } else {
        cur = p - 1;
      }
    }
    return lo;
  }

  // The entries at or above `from` into the list, in bank order, if they fit;
  // how many there are. A barrier has to follow.
  __device__ uint32_t gather(uint32_t from, List* list) {
    uint32_t mine = 0, all;
    keys([&](uint32_t k) { mine += k >= from; });
    uint32_t seen = g.ahead(__reduce_add_sync(0xffffffffu, mine), &all);
    if (all > kList) return all;
    each([&](int c, const uint32_t* k) {
      uint32_t in = 0;
#pragma unroll
      for (int e = 0; e < V; e++) in += k[e] >= from;
      if (!__any_sync(0xffffffffu, in != 0u)) return;
      const uint32_t incl = warp_scan(in, g.lane);
      uint32_t r = seen + incl - in;
#pragma unroll
      for (int e = 0; e < V; e++)
        if (k[e] >= from) {
          list->key[r] = k[e];
          list->where[r] = uint32_t(at(c) + e);
          r++;
        }
      seen += __shfl_sync(0xffffffffu, incl, 31);
    });
    return all;
  }

  // Drops the entries below the cut and all but the first `ties` at it.
  __device__ void drop(uint32_t cut, uint32_t ties) {
    uint32_t mine = 0;
    keys([&](uint32_t k) { mine += k == cut; });
    uint32_t seen = g.ahead(__reduce_add_sync(0xffffffffu, mine));
    uint32_t left = 0;
    each([&](int c, uint32_t* k) {
      uint32_t in = 0;
#pragma unroll
      for (int e = 0; e < V; e++) in += k[e] == cut;
      uint32_t r = seen;
      if (__any_sync(0xffffffffu, in != 0u)) {
        const uint32_t incl = warp_scan(in, g.lane);
        r += incl - in;
        seen += __shfl_sync(0xffffffffu, incl, 31);
      }
      uint32_t any = 0;
#pragma unroll
      for (int e = 0; e < V; e++) {
        if (k[e] < cut || (k[e] == cut && r++ >= ties)) k[e] = 0u;
        any |= k[e];
      }
      put(c, k);
      if (__any_sync(0xffffffffu, any != 0u)) left |= 1u << c;
    });
    live = left;
  }

  // Packs what is left to the front of the warp's segment, in bank order. A
  // chunk's own words are read before any is written, and no later chunk's are.
  __device__ void pack() {
    uint32_t* key = reinterpret_cast<uint32_t*>(slab);
    kept = 0;
    for (int c = 0; c < chunks; c++) {
      if (!(live >> c & 1u)) continue;
      uint32_t k[V], ahead = 0, all = 0;
      get(c, k);
      __syncwarp();
#pragma unroll
      for (int e = 0; e < V; e++) {
        const uint32_t b = __ballot_sync(0xffffffffu, k[e] != 0u);
        ahead += __popc(b & ((1u << g.lane) - 1u));
        all += __popc(b);
      }
      uint32_t r = kept + ahead;
#pragma unroll
      for (int e = 0; e < V; e++)
        if (k[e]) {
          key[r] = k[e];
          place[r] = uint16_t(c * 32 * V + g.lane * V + e);
          r++;
        }
      kept += all;
    }
    __syncwarp();
  }
  // f(key, index) for the packed entries, 32 at a time (key 0 behind the last).
  template <typename F>
  __device__ __forceinline__ void packed(F f) {
    const uint32_t* key = reinterpret_cast<const uint32_t*>(slab);
    for (uint32_t j0 = 0; j0 < kept; j0 += 32) {
      const uint32_t j = j0 + g.lane;
      const bool in = j < kept;
      f(in ? key[j] : 0u, in ? uint32_t(base + int(place[j])) : kNone);
    }
  }
};

// top-p's search by approximate weights: f32 exponentials in units of 2^-20 of
// the largest, summed as integers (a warp's at most 2^31). An entry above half
// a unit has |x| <= 21 ln 2; three f32 roundings of the exponent and ex2's
// 2^-22 put its weight within 3e-6, and for probabilities lg2's 2^-22 of log2 v
// and of log2 m add 3.4e-7 (|log2 m| + 21 T) / T. A mass that clears the goal
// by `err` of the total and half a unit an entry is on its side for certain;
// the first pivot that does not leaves [lo, cur] to the 64-bit search. What it
// usually leaves is one value.
template <typename R>
__device__ __forceinline__ void narrow(R& r, double top_p, uint32_t open, int kind, uint32_t& lo, uint32_t& cur) {
  const float mv = float(r.m), it = float(r.inv_t) * (kind == kKindP ? 1.0f : 1.44269504f);
  const float mu = kind == kKindP ? log2_fast(mv) : mv;
  auto units = [&](uint32_t key) {
    const float v = value_of(key);
    const float u = ((kind == kKindP ? log2_fast(v) : v) - mu) * it;
    return __float2uint_rn(exp2_fast(fminf(u, 0.0f)) * 1048576.0f);
  };
  uint32_t all = 0;
  r.keys([&](uint32_t k) { all += k ? units(k) : 0u; });
  const double total = r.g.sum_u32(all);
  const double goal = top_p * total;
  const double err = (1e-5 + 1e-5 * r.inv_t + 4e-7 * fabs(double(mu)) * (kind == kKindP ? r.inv_t : 0.0)) * total +
                     0.5 * open + 1.0;
  const double above = goal + err, below = goal - err;
  for (int step = 0; cur != lo; step++) {
    const uint32_t p = pivot(lo, cur, step, kind);
    uint32_t mass = 0, mn = 0xffffffffu, mx = 0u;
    r.keys([&](uint32_t k) {
      if (k >= p) { mass += units(k); mn = min(mn, k); }
      else mx = max(mx, k);
    });
    const double a = r.g.masses(mass, mn, mx);
    if (a >= above) lo = mn;
    else if (a < below) cur = mx;
    else return;
  }
}

// The cuts by searching for their values; afterwards r holds exactly what top-k
// and top-p keep (min-p and the dropping are left to the weights' pass).
template <typename R>
__device__ __forceinline__ void cut_search(R& r, const Cut& c, const Stats& s, int kind) {
  if (s.open == 0) return;
  uint32_t left = s.open, lo = s.lo;
  if (c.k && c.k < s.open) {
    // the largest t with count(k >= t) >= c.k; `above`: count(k > t's bracket)
    uint32_t cur = s.hi, above = 0;
    for (int step = 0; cur != lo; step++) {
      const uint32_t p = pivot(lo, cur, step, kind);
      uint32_t n = 0, mn = 0xffffffffu, mx = 0u;
      r.keys([&](uint32_t k) {
        if (k >= p) { n++; mn = min(mn, k); }
        else mx = max(mx, k);
      });
      r.g.counts(n, mn, mx);
      if (n >= c.k) lo = mn;
      else { cur = mx; above = n; }
    }
    r.drop(lo, c.k - above);
    left = c.k;
  }
  if (c.top_p < 1.0) {
    // the largest t with mass(k >= t) >= goal
    uint32_t cur = s.hi;
    narrow(r, c.top_p, left, kind, lo, cur);
    uint32_t ties = 0, mn = 0xffffffffu, mx = 0u;
    r.keys([&](uint32_t k) { ties += k == lo; });
    r.g.counts(ties, mn, mx);
    if (cur == lo && ties == 1) {
      r.drop(lo, 1u);
      return;
    }
    double part = 0.0, over = 0.0;
    r.keys([&](uint32_t k) {
      if (!__any_sync(0xffffffffu, k != 0u)) return;
      const double w = r.weight(k);
      part += w;
      if (k > cur) over += w;
    });
    const double goal = c.top_p * r.g.sum(part);
    double above = r.g.sum(over);
    for (int step = 0; cur != lo; step++) {
      const uint32_t p = pivot(lo, cur, step, kind);
      double mass = 0.0;
      uint32_t n = 0;
      mn = 0xffffffffu, mx = 0u;
      r.keys([&](uint32_t k) {
        const bool in = k >= p && k <= cur;
        if (__any_sync(0xffffffffu, in)) mass += r.weight(in ? k : 0u);
        if (k >= p) mn = min(mn, k);
        else mx = max(mx, k);
      });
      mass = above + r.g.sum(mass);
      r.g.counts(n, mn, mx);
      if (mass >= goal) lo = mn;
      else { cur = mx; above = mass; }
    }
    const double w = r.weight(lo);
    const double need = w > 0.0 ? ceil((goal - above) / w) : 1.0;
    r.drop(lo, need < 1.0 ? 1u : need >= 4294967295.0 ? 0xffffffffu : uint32_t(need));
  }
}

// The cuts of a list of up to 32 S entries, without a search: every lane sums
// up, over the list in shared memory, the entries ahead of its own in
// descending order (ties in bank order): how many, for top-k, and their exact
// weights, for top-p. w: the lanes' weights, left at 0 for what is cut.
template <int S>
__device__ __forceinline__ void cut_pairs(ListRow<S>& r, const Cut& c, const uint32_t* key, double* shared_w, int n,
                                          double* w) {
  const int lane = r.g.lane;
  if (c.k && c.k < uint32_t(n)) {
    uint32_t bar[S], rank[S];
#pragma unroll
    for (int s = 0; s < S; s++) {
      bar[s] = r.k[s];
      rank[s] = 0u;
    }
#pragma unroll 4
    for (int j = 0; j < n; j++) {
      const uint32_t kj = key[j];
#pragma unroll
      for (int s = 0; s < S; s++) {
        bar[s] += j == s * 32 + lane;  // behind itself, an equal entry is not ahead
        rank[s] += kj >= bar[s];
      }
    }
#pragma unroll
    for (int s = 0; s < S; s++)
      if (rank[s] >= c.k) {
        r.k[s] = 0u;
        w[s] = 0.0;
      }
  }
  if (c.top_p < 1.0) {
    uint32_t bar[S];
    double ahead[S], mine = 0.0;
#pragma unroll
    for (int s = 0; s < S; s++) {
      bar[s] = r.k[s];
      ahead[s] = 0.0;
      shared_w[s * 32 + lane] = w[s];
      mine += w[s];
    }
    __syncwarp();
    const double goal = c.top_p * warp_add(mine);
#pragma unroll 4
    for (int j = 0; j < n; j++) {
      const uint32_t kj = key[j];
      const double wj = shared_w[j];
#pragma unroll
      for (int s = 0; s < S; s++) {
        bar[s] += j == s * 32 + lane;
        if (kj >= bar[s]) ahead[s] += wj;
      }
    }
#pragma unroll
    for (int s = 0; s < S; s++)
      if (!(ahead[s] < goal) && r.k[s] != r.top) {
        r.k[s] = 0u;
        w[s] = 0.0;
      }
    // the largest entry stays whatever top_p is: the first of its value
    uint32_t seen = 0u;
#pragma unroll
    for (int s = 0; s < S; s++) {
      const uint32_t at = __ballot_sync(0xffffffffu, r.k[s] == r.top);
      const bool first = !seen && at && lane == __ffs(at) - 1;
      if (r.k[s] == r.top && !first && !(ahead[s] < goal)) {
        r.k[s] = 0u;
        w[s] = 0.0;
      }
      seen |= at;
    }
  }
}

// What a draw found: the entry (kNone: an empty row), its pi, and how many entries were kept.
struct Drawn {
  uint32_t hit, kept;
  double pi;
};
__device__ __forceinline__ void report(const DrawArg& a, uint32_t row, const Drawn& d) {
  if (a.index) a.index[row] = d.hit;
  if (a.logp) a.logp[row] = d.hit == kNone ? -INFINITY : float(log64(d.pi));
  if (a.kept) a.kept[row] = d.kept;
}

// The draw of a list after its cuts, every lane with the answer; pi go into a
// row that was cleared. A lane and slice holds one entry, so the entry that a
// uniform hits is the first one whose prefix passes it.
template <int S>
__device__ __forceinline__ Drawn draw_list(ListRow<S>& r, const Cut& c, const DrawArg& a, const RowAt& at, bool fits,
                                           double u, double* w) {
  const int lane = r.g.lane;
  const double floor_w = c.min_p * (r.plain_p ? r.m : 1.0);
  double incl[S], z = 0.0;
  uint32_t kept[S];
#pragma unroll
  for (int s = 0; s < S; s++) {
    incl[s] = 0.0;
    kept[s] = 0u;
    if (s >= r.slices) continue;
    if (w[s] < floor_w) w[s] = 0.0;
    kept[s] = __ballot_sync(0xffffffffu, w[s] > 0.0);
    const double sc = warp_scan(w[s], lane);
    incl[s] = z + sc;
    z += __shfl_sync(0xffffffffu, sc, 31);
  }
  Drawn d{kNone, 0u, 0.0};
#pragma unroll
  for (int s = 0; s < S; s++) d.kept += __popc(kept[s]);
  if (d.kept == 0) return d;
  const double inv = 1.0 / z;
  // u z < cum by the sign of u z - cum, whose one rounding keeps it: u on an
  // entry's edge falls where the reals put it. No u: the first largest entry,
  // whose weight is the largest there is.
  int at_s = -1, at_lane = 0;
#pragma unroll
  for (int s = 0; s < S; s++) {
    const bool past = a.uniforms ? fma(u, z, -incl[s]) < 0.0 : r.k[s] == r.top;
    const uint32_t who = kept[s] & __ballot_sync(0xffffffffu, past);
    if (at_s < 0 && who) {
      at_s = s;
      at_lane = __ffs(who) - 1;
    }
  }
  if (at_s < 0) {  // u of 1, or a last bit short of it: the last kept entry
#pragma unroll
    for (int s = 0; s < S; s++)
      if (kept[s]) {
        at_s = s;
        at_lane = 31 - __clz(kept[s]);
      }
  }
  double we = 0.0;
#pragma unroll
  for (int s = 0; s < S; s++)
    if (s == at_s) we = __shfl_sync(0xffffffffu, w[s], at_lane);
  d.hit = r.where[at_s * 32 + at_lane];
  d.pi = we * inv;
  if (a.p && fits) {
    float* out = a.p + at.out;
#pragma unroll
    for (int s = 0; s < S; s++)
      if (kept[s] >> lane & 1u) out[r.index(s)] = float(w[s] * inv);
  }
  return d;
}

// The draw of a row that stayed spread over its group, after its cuts: written
// to the outputs; pi go into a row that was cleared.
template <typename T, int W, int CL>
__device__ __forceinline__ void finish_wide(WideRow<T, W, CL>& r, const Cut& c, const DrawArg& a, uint32_t row,
                                            const RowAt& at, bool fits) {
  const int lane = r.g.lane;
  const double floor_w = c.min_p * (r.plain_p ? r.m : 1.0);
  auto weight = [&](uint32_t key) {
    const double w = r.weight(key);
    return w < floor_w ? 0.0 : w;
  };
  r.pack();
  double mine = 0.0;
  uint32_t kept = 0, last = 0u, hit = 0xffffffffu;
  r.packed([&](uint32_t key, uint32_t i) {
    const double w = weight(key);
    mine += w;
    if (w > 0.0) {
      kept++;
      last = i + 1u;
      if (!a.uniforms && key == r.top) hit = min(hit, i);
    }
  });
  double before, through;
  const double z = r.g.prefix(mine, before, through);
  double drawn = 0.0;
  if (a.uniforms) {
    // cum > u z by the sign of u z - cum, whose one rounding keeps it. The warp
    // whose weights the target falls among walks them, 32 at a time.
    const double u = fmin(fmax(a.uniforms[row], 0.0), 1.0);
    if (fma(u, z, -through) < 0.0 && !(fma(u, z, -before) < 0.0)) {
      double cum = before;
      r.packed([&](uint32_t key, uint32_t i) {
        const double w = weight(key), sc = warp_scan(w, lane);
        const uint32_t who = __ballot_sync(0xffffffffu, w > 0.0 && fma(u, z, -(cum + sc)) < 0.0);
        if (who && hit == 0xffffffffu) hit = __shfl_sync(0xffffffffu, i, __ffs(who) - 1);
        cum += __shfl_sync(0xffffffffu, sc, 31);
      });
      if (hit == 0xffffffffu) hit = __reduce_max_sync(0xffffffffu, last) - 1u;  // a last bit short: its last entry
    }
  }
  r.g.counts(kept, hit, last);
  if (r.g.segment() == 0 && lane == 0) {
    if (a.kept) a.kept[row] = kept;
    if (kept == 0) report(a, row, Drawn{kNone, 0u, 0.0});
  }
  if (kept == 0) return;
  if (hit == 0xffffffffu) hit = last - 1u;  // u of 1
  const double inv = 1.0 / z;
  float* out = a.p && fits ? a.p + at.out : nullptr;
  const int64_t mine_at = int64_t(hit) - r.base;  // whether this warp holds the entry
  if (!out && !(mine_at >= 0 && mine_at < int64_t(r.chunks) * 32 * WideRow<T, W, CL>::V)) return;
  r.packed([&](uint32_t key, uint32_t i) {
    if (!out && !__any_sync(0xffffffffu, i == hit)) return;
    const double w = weight(key);
    if (out && w > 0.0) out[i] = float(w * inv);
    if (i == hit) drawn = w;
  });
  if (drawn > 0.0) report(a, row, Drawn{hit, kept, drawn * inv});
}

// The loss of what the cuts left, and its gradient:
//   loss = -A log pi(a) - beta H(pi), H = log Z - sum w x / Z,
//   dloss/dv_j = (A (pi_j - [j = a]) + beta pi_j (log pi_j + H)) / T
// for what is kept, 0 elsewhere (the row was cleared), times the row's weight.
// The group's sums: of w, of w x, the action's x, whether it is kept.
struct Slope {
  double adv, beta, g0, inv_z, base;
  bool learns;
  uint32_t act;
  __device__ float of(double w, double x, uint32_t i) const {
    const double pi = w * inv_z;
    return float(g0 * fma(adv, pi - (i == act ? 1.0 : 0.0), beta * pi * (x + base)));
  }
};
__device__ __forceinline__ Slope loss_row(const LossArg& a, const Cut& c, uint32_t row, double z, double sx, double xa,
                                          bool any, bool live, bool lead) {
  const uint32_t act = a.actions[row];
  const bool asked = act != kNone;
  const double log_z = any ? log64(z) : 0.0, inv_z = any ? 1.0 / z : 0.0;
  const double h = any ? log_z - sx * inv_z : 0.0, logp = xa - log_z;
  const bool learns = asked && live && !c.greedy;  // one answer has no gradient
  const double adv = double(a.advantage[row]), beta = double(a.beta);
  if (lead) {
    if (a.loss) a.loss[row] = learns ? float(-adv * logp - beta * h) : 0.0f;
    if (a.logp) a.logp[row] = !asked ? 0.0f : live ? float(logp) : -INFINITY;
    if (a.entropy) a.entropy[row] = float(h);
  }
  return Slope{adv, beta, (a.row_weight ? double(a.row_weight[row]) : 1.0) * c.inv_t, inv_z, h - log_z, learns, act};
}

template <typename T, int S>
__device__ __forceinline__ void loss_list(ListRow<S>& r, const Cut& c, const LossArg& a, uint32_t row, const RowAt& at,
                                          bool fits, const double* w) {
  const uint32_t act = a.actions[row];
  double z = 0.0, sx = 0.0, xa = 0.0, x[S];
  bool live = false;
  uint32_t kept = 0;
  r.each([&](int s) {
    x[s] = r.x_of(r.k[s] ? r.k[s] : r.top);
    const bool in = w[s] > 0.0 && w[s] >= c.min_p;
    if (!in) r.k[s] = 0u;
    else {
      z += w[s];
      sx = fma(w[s], x[s], sx);
      if (r.index(s) == act) { live = true; xa = x[s]; }
    }
    kept += __popc(__ballot_sync(0xffffffffu, in));
  });
  live = __any_sync(0xffffffffu, live);
  const Slope sl = loss_row(a, c, row, warp_add(z), warp_add(sx), warp_add(xa), kept != 0, live, r.g.lane == 0);
  if (!a.grad || !fits || !sl.learns) return;
  T* out = static_cast<T*>(a.grad) + at.out;
  r.each([&](int s) {
    if (r.k[s]) out[r.index(s)] = from_f32<T>(sl.of(w[s], x[s], r.index(s)));
  });
}

template <typename T, int W, int CL>
__device__ __forceinline__ void finish_wide(WideRow<T, W, CL>& r, const Cut& c, const LossArg& a, uint32_t row,
                                            const RowAt& at, bool fits) {
  const uint32_t act = a.actions[row];
  double z = 0.0, sx = 0.0, xa = 0.0;
  uint32_t kept = 0, live = 0xffffffffu, none = 0u;
  r.pack();
  r.packed([&](uint32_t key, uint32_t i) {
    double x;
    const double w = r.weight(key, x);
    if (w > 0.0 && w >= c.min_p) {
      z += w;
      sx = fma(w, x, sx);
      kept++;
      if (i == act) { live = 0u; xa = x; }
    }
  });
  z = r.g.sum(z);
  sx = r.g.sum(sx);
  xa = r.g.sum(xa);
  r.g.counts(kept, live, none);
  const Slope sl = loss_row(a, c, row, z, sx, xa, kept != 0, live == 0u, r.g.segment() == 0 && r.g.lane == 0);
  if (!a.grad || !fits || !sl.learns) return;
  T* out = static_cast<T*>(a.grad) + at.out;
  r.packed([&](uint32_t key, uint32_t i) {
    double x;
    const double w = r.weight(key, x);
    if (w > 0.0 && w >= c.min_p) out[i] = from_f32<T>(sl.of(w, x, i));
  });
}

// Whether a row keeps the stated bound and the group holds it, misaligned as it is.
template <typename T>
__device__ __forceinline__ bool row_fits(const RowsArg& r, const RowAt& at, uint32_t cap) {
  const uint32_t shift = uint32_t((reinterpret_cast<uintptr_t>(static_cast<const T*>(r.values) + at.in) & 15) / sizeof(T));
  return at.n <= r.row_len && at.n + shift <= cap;
}

// Clears the output that is laid out like the rows.
template <typename T> __device__ __forceinline__ void clear_out(const DrawArg& a, const RowAt& at, int n, int tid, int threads) {
  if (a.p) clear_row(a.p + at.out, n, tid, threads);
}
template <typename T> __device__ __forceinline__ void clear_out(const LossArg& a, const RowAt& at, int n, int tid, int threads) {
  if (a.grad) clear_row(static_cast<T*>(a.grad) + at.out, n, tid, threads);
}
// Everything after the gathering, by one warp on a list of n <= 32 S entries:
// a draw to be reported, or a loss that has been written.
template <typename T, int S>
__device__ __forceinline__ Drawn finish_list(ListRow<S>& r, const Cut& c, const DrawArg& a, uint32_t, const RowAt& at,
                                             bool fits, double u, double* w) {
  return draw_list<S>(r, c, a, at, fits, u, w);
}
template <typename T, int S>
__device__ __forceinline__ Drawn finish_list(ListRow<S>& r, const Cut& c, const LossArg& a, uint32_t row,
                                             const RowAt& at, bool fits, double, double* w) {
  loss_list<T, S>(r, c, a, row, at, fits, w);
  return Drawn{kNone, 0u, 0.0};
}
template <typename T, int S, typename Arg>
__device__ __forceinline__ Drawn list_as(List& list, uint32_t n, const Tables& tables, int lane, const Cut& c,
                                         const Arg& a, uint32_t row, const RowAt& at, bool fits, double u) {
  ListRow<S> r(lane, tables, list, n);
  const bool cuts = (c.k && c.k < n) || c.top_p < 1.0;
  constexpr bool pairs = S <= kPairs / 32;
  const Stats s = r.stats(n, cuts && !pairs);
  r.begin(c, s, a.r.kind);
  if (!pairs && cuts) cut_search(r, c, s, a.r.kind);
  double w[S];
#pragma unroll
  for (int e = 0; e < S; e++) {
    w[e] = 0.0;
    if (e < r.slices) w[e] = r.weight(r.k[e]);
  }
  if constexpr (pairs) {
    if (cuts) cut_pairs<S>(r, c, list.key, list.w, int(n), w);
  }
  return finish_list<T, S>(r, c, a, row, at, fits, u, w);
}
template <typename T, typename Arg>
__device__ __forceinline__ Drawn list_row(List& list, uint32_t n, const Tables& tables, int lane, const Cut& c,
                                          const Arg& a, uint32_t row, const RowAt& at, bool fits, double u) {
  if (n <= uint32_t(kPairs)) return list_as<T, kPairs / 32>(list, n, tables, lane, c, a, row, at, fits, u);
  return list_as<T, kList / 32>(list, n, tables, lane, c, a, row, at, fits, u);
}

// What a warp keeps of its rows' draws until it writes them: lane i has the
// draw of row first + i, so that the logarithms of 32 rows are one evaluation.
template <typename Arg> struct Answers {
  __device__ double uniform(const Arg&, uint32_t) { return 0.0; }
  __device__ void take(const Drawn&, const Arg&, uint32_t, int) {}
  __device__ void done(const Arg&, uint32_t, int) {}
};
template <> struct Answers<DrawArg> {
  Drawn mine{kNone, 0u, 0.0};
  int held = 0;
  __device__ double uniform(const DrawArg& a, uint32_t row) {
    return a.uniforms ? fmin(fmax(a.uniforms[row], 0.0), 1.0) : 0.0;
  }
  __device__ __forceinline__ void take(const Drawn& d, const DrawArg& a, uint32_t row, int lane) {
    if (lane == held) mine = d;
    if (++held == 32) done(a, row, lane);
  }
  // Writes what is held, the last of it row's.
  __device__ void done(const DrawArg& a, uint32_t row, int lane) {
    if (lane < held) report(a, row + 1 - held + lane, mine);
    held = 0;
  }
};

// Rows of up to 256 entries: a warp a row, always by its list. A warp takes a
// run of rows one after another: its tables are made once, the frame is
// searched for once, and the next row's entries and uniform are fetched while
// it works.
//
// Bound by instruction issue: 34818 drawn rows of 8 to 240 probabilities, a
// quarter open, take 93 us at an IPC of 2.5, about 1500 warp instructions a row
// (64-bit exponentials and logarithms, all pairs of the list), and 2 % of the
// memory's bandwidth; the loss of 4096 rows takes 17 us, the latency of single
// rows: 1024 CTAs on the 888 that fit, each with its own tables.
// CTAs an SM (80 registers: f32 draws spill 292 bytes a thread, the others 164
// to 244). More warps hide more of a row's latency, more registers spill
// less: 34818 drawn rows took 95, 97, 105 and 96 us with 5 to 8, the loss of
// 4096 rows between 19 and 20.
constexpr int kSmallCtas = 6;
template <typename T, typename Arg>
__global__ void __launch_bounds__(128, kSmallCtas) k_policy_small(const __grid_constant__ Arg a) {
  constexpr int V = 16 / int(sizeof(T)), kVecs = int(kList) / 32 / V;
  __shared__ List lists[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t warps = gridDim.x * 4, each = (a.r.rows + warps - 1) / warps;
  const uint32_t first = (blockIdx.x * 4 + warp) * each, end = min(a.r.rows, first + each);
  if (first >= a.r.rows) return;
  Walk walk;
  if (!walk.start(a.r, a.out_pitch, first, lane)) return;
  const Tables tables(lane, a.r.kind == kKindP);
  Answers<Arg> answers;
  List& list = lists[warp];
  // A lane's vectors of the row; a vector that reaches past either end of the
  // row is read entry by entry, with NaN, which no row's support holds, outside.
  uint32_t q[kVecs][4];
  double u;
  auto fits = [&](const RowAt& at) { return at.n <= a.r.row_len && at.n + V - 1 <= kList; };
  auto fetch = [&](const RowAt& at, uint32_t row) {
    const int n = fits(at) ? int(at.n) : 0;
    const T* in = static_cast<const T*>(a.r.values) + at.in;
    const int i0 = lane * V - int((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
#pragma unroll
    for (int v = 0; v < kVecs; v++) {
      const int i = i0 + v * 32 * V;
      if (i >= 0 && i + V <= n) {
        const uint4 x = __ldcs(reinterpret_cast<const uint4*>(in + i));
        q[v][0] = x.x; q[v][1] = x.y; q[v][2] = x.z; q[v][3] = x.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) q[v][e] = 0xffffffffu;
        if (i + V > 0 && i < n) {
          float f[V];
#pragma unroll
          for (int e = 0; e < V; e++) f[e] = i + e >= 0 && i + e < n ? as_f32(in[i + e]) : __uint_as_float(0x7fc00000u);
#pragma unroll
          for (int e = 0; e < V; e += 2) set2<T>(q[v], e, f[e], f[e + 1]);
        }
      }
    }
    u = answers.uniform(a, row);
  };
  fetch(walk.at, first);
  for (uint32_t row = first; row < end; row++) {
    const RowAt at = walk.at;
    const bool ok = fits(at);
    const T* in = static_cast<const T*>(a.r.values) + at.in;
    const int i0 = lane * V - int((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
    // the open entries into the list, in bank order
    uint32_t count = 0;
#pragma unroll
    for (int v = 0; v < kVecs; v++) {
      uint32_t k[V], ahead = 0, all = 0;
#pragma unroll
      for (int e = 0; e < V; e++) {
        k[e] = open_key<T>(entry<T>(q[v], e), a.r.kind);
        const uint32_t b = __ballot_sync(0xffffffffu, k[e] != 0u);
        ahead += __popc(b & ((1u << lane) - 1u));
        all += __popc(b);
      }
      uint32_t r = count + ahead;
#pragma unroll
      for (int e = 0; e < V; e++)
        if (k[e]) {
          list.key[r] = k[e];
          list.where[r] = uint32_t(i0 + v * 32 * V + e);
          r++;
        }
      count += all;
    }
    // (grad and p may lie over the values: this row's have been read)
    if (ok) clear_out<T>(a, at, int(at.n), lane, 32);
    const double u_row = u;
    const bool more = row + 1 < end && walk.step(a.r, row + 1);
    if (more) fetch(walk.at, row + 1);
    __syncwarp();
    answers.take(list_row<T>(list, count, tables, lane, cut_of(a.c, row), a, row, at, ok, u_row), a, row, lane);
    if (!more) {
      answers.done(a, row, lane);
      return;
    }
    __syncwarp();  // the list is written again for the next row
  }
}

// Longer rows: CL CTAs of W warps a row, `chunks` vectors a lane. A CTA on its
// own (CL = 1) takes `batch` rows, one after another up to their lists, which
// its warps then finish side by side: one warp at the end of one row would
// leave the SM idle.
// 4096 drawn rows of 4096 under top-k 200, top-p and min-p take 127 us: issue
// (IPC 2.75; statistics, the lower bound's counts, one warp a list) and
// barriers. 32 bf16 rows of 131071 with limits of their own take 34 to 42 us:
// latency, a dozen cluster-wide reductions one after another, on 128 of the SMs.
// The registers of two CTAs of 16 warps an SM (64) spill 108 to 176 bytes a
// thread, those of the largest rows' too, whose shared memory leaves one.
template <typename T, int W, int CL, typename Arg>
__global__ void __launch_bounds__(W * 32, 32 / W) k_policy_rows(const __grid_constant__ Arg a, uint32_t batch,
                                                               uint32_t chunks) {
  constexpr int V = 16 / int(sizeof(T)), kLists = CL > 1 ? 1 : W < kBatch ? W : kBatch;
  extern __shared__ uint4 keys[];
  __shared__ typename Group<W, CL>::Shared sh;
  __shared__ List lists[kLists];
  __shared__ struct { RowAt at; uint32_t row, count; } todo[kLists];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t cap = uint32_t(32 * V * W * CL) * chunks;
  const Tables tables(lane, a.r.kind == kKindP);
  uint32_t made = 0;
  for (uint32_t b = 0; b < batch; b++) {
    const uint32_t row = blockIdx.x / CL * batch + b;
    RowAt at;
    if (row >= a.r.rows || !locate(a.r, a.out_pitch, row, lane, &at)) break;
    WideRow<T, W, CL> r(sh, tables, lane, warp, keys, int(chunks));
    const bool fits = row_fits<T>(a.r, at, cap);
    const int n = fits ? int(at.n) : 0;
    r.load(static_cast<const T*>(a.r.values) + at.in, n, a.r.kind);
    const Cut c = cut_of(a.c, row);
    Stats s = r.stats();
    uint32_t from = s.lo, count = s.open;
    List* to = &lists[made];
    if constexpr (CL > 1) to = cooperative_groups::this_cluster().map_shared_rank(to, 0);
    if (s.open > kList && c.k && c.k <= kListTopK) {
      from = r.lower_bound(c.k, s, a.r.kind);
      count = r.gather(from, to);
    } else if (s.open <= kList) {
      r.gather(from, to);
    }
    // (grad and p may lie over the values: this row's have been read)
    if (fits) clear_out<T>(a, at, n, r.g.rank * W * 32 + int(threadIdx.x), W * 32 * CL);
    if (count <= kList) {
      if (threadIdx.x == 0) {
        todo[made].at = at;
        todo[made].row = row;
        todo[made].count = count;
      }
      made++;
    } else {
      if (from != s.lo) {  // top-k's search starts from the smallest entry at or above the bound
        uint32_t mn = 0xffffffffu, none = 0, mx = 0;
        r.keys([&](uint32_t k) {
          if (k >= from) mn = min(mn, k);
        });
        r.g.counts(none, mn, mx);
        s.lo = mn;
        s.open = count;
      }
      r.begin(c, s, a.r.kind);
      cut_search(r, c, s, a.r.kind);
      // orders the clearing before the entries that others write
      if constexpr (CL > 1) cooperative_groups::this_cluster().sync();
      else __syncthreads();
      finish_wide(r, c, a, row, at, fits);
    }
    if (b + 1 < batch) __syncthreads();  // the group's slots and keys start again with the next row
  }
  if constexpr (CL > 1) cooperative_groups::this_cluster().sync();
  else __syncthreads();
  if (warp >= int(made) || (CL > 1 && cooperative_groups::this_cluster().block_rank() != 0)) return;
  const RowAt at = todo[warp].at;
  const uint32_t row = todo[warp].row;
  const bool fits = row_fits<T>(a.r, at, cap);
  Answers<Arg> answers;
  answers.take(list_row<T>(lists[warp], todo[warp].count, tables, lane, cut_of(a.c, row), a, row, at, fits,
                           answers.uniform(a, row)), a, row, lane);
  answers.done(a, row, lane);
}

}  // namespace pol
}  // namespace kc
