// policy_cut.cuh — rows with cuts: the draws (k_draw, k_draw_small) and the
// policy loss (k_policy_loss, k_policy_loss_small).
//
// A row is loaded into registers, E entries a thread: a warp up to 256 entries,
// a CTA to 32768, a cluster of 8 CTAs beyond. Warp g of the row's group owns
// the contiguous segment [32 E g, 32 E (g + 1)), in chunks of one 16-byte load
// a lane, so that bank order is (warp, chunk, lane, entry).
//
// What the cuts leave is usually short: a bank's grammar admits few records,
// and top-k and top-p keep few. So a row is first gathered: its open entries,
// or with top-k those at or above a lower bound of the k-th largest, go to a
// list in shared memory in bank order, and if it holds at most kList entries
// one warp does everything else on it, with one entry a lane and slice
// of 32 (ListRow). The lower bound is the k-th largest of the chunks' maxima:
// k chunks reach it, so k entries do. Rows whose list would be longer stay
// spread over their group.
#pragma once
#include "policy.cuh"

namespace kc {
namespace pol {

constexpr uint32_t kList = 256;
constexpr uint32_t kListTopK = 208;  // top-k up to this looks for a list

constexpr int kPairs = 64;  // lists up to this are cut by comparing all pairs
struct List {
  uint32_t key[kList], where[kList];  // a key, and its index in the row
  double w[kPairs];
};

// Open entries of a row, their smallest and largest key.
struct Stats {
  uint32_t open, lo, hi;
};

// A row's entries (V of them in a vector; V = 1: a gathered list), and its cut.
template <int E, int V, int W, int CL>
struct Row {
  static constexpr int kChunks = E / V;
  static constexpr uint32_t kCap = uint32_t(32) * E * W * CL;
  static constexpr bool kCached = E <= 32;  // the registers hold a weight an entry beside the keys
  static_assert(E % V == 0 && kChunks <= 32, "a thread holds whole vectors");
  static constexpr float kUnit = 1048576.0f;
  static_assert(32 * E <= 2048, "a warp's units fit 32 bits");

  Group<W, CL> g;
  const Tables& t;
  uint32_t k[E];   // keys; 0: not in the support
  uint32_t live;   // chunks of this warp that hold an entry of the support
  int slices;      // of a list: 32 entries each
  uint32_t top;    // the largest key
  double m, log_m, inv_t;
  bool power;      // probabilities at a temperature other than 1: x from logarithms
  bool plain_p;    // probabilities at T = 1: the weights are the values
  int i0;          // index of this lane's first entry of chunk 0
  const uint32_t* where;  // a list's indices

  __device__ Row(typename Group<W, CL>::Shared& sh, const Tables& tables, int lane, int warp)
      : g(sh, lane, warp), t(tables) {}
  __device__ Row(int lane, const Tables& tables) : g(lane), t(tables) {}  // one warp

  __device__ int at(int c) const { return i0 + c * 32 * V; }
  __device__ uint32_t index(int e) const {
    if constexpr (V == 1) return where[e * 32 + g.lane];
    else return uint32_t(at(e / V) + e % V);
  }

  // f(entry) for every entry of the chunks that hold any; the warp together.
  template <typename F>
  __device__ __forceinline__ void each(F f) {
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      if constexpr (V == 1) {
        if (c >= slices) break;
      }
      if (V == 1 || (live >> c & 1u)) {
#pragma unroll
        for (int e = 0; e < V; e++) f(c * V + e);
      }
    }
  }
  __device__ void find_live() {
    if constexpr (V == 1) return;
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
  template <typename T>
  __device__ void load(const T* row, uint32_t n, int kind) {
    static_assert(V == 16 / int(sizeof(T)), "a vector is 16 bytes");
    const int shift = int((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    i0 = g.segment() * 32 * E + g.lane * V - shift;
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      const int i = at(c);
      if (i >= 0 && i + V <= int(n)) {
        const uint4 q = __ldcs(reinterpret_cast<const uint4*>(row + i));
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int e = 0; e < V; e++) k[c * V + e] = open_key<T>(entry<T>(w, e), kind);
      } else {
#pragma unroll
        for (int e = 0; e < V; e++)
          k[c * V + e] = i + e >= 0 && i + e < int(n) ? open_key<T>(as_f32(row[i + e]), kind) : 0u;
      }
    }
    find_live();
  }
  // Takes up a list of n entries.
  __device__ void take(const List& list, uint32_t n) {
    where = list.where;
    slices = int((n + 31) / 32);
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      const uint32_t j = uint32_t(c) * 32 + g.lane;
      k[c] = j < n ? list.key[j] : 0u;
    }
  }
  // The stats of a list of n entries; lo only where the search will need it.
  __device__ Stats list_stats(uint32_t n, bool need_lo) {
    Stats s{n, 0u, 0u};
    uint32_t lo = 0xffffffffu;
    each([&](int e) {
      s.hi = max(s.hi, k[e]);
      if (k[e]) lo = min(lo, k[e]);
    });
    s.hi = __reduce_max_sync(0xffffffffu, s.hi);
    s.lo = need_lo ? __reduce_min_sync(0xffffffffu, lo) : 0u;
    return s;
  }
  __device__ bool in_use(int c) const { return V == 1 ? c < slices : (live >> c & 1u); }

  __device__ Stats stats() {
    Stats s{0u, 0xffffffffu, 0u};
    each([&](int e) {
      s.open += k[e] != 0u;
      if (k[e]) s.lo = min(s.lo, k[e]);
      s.hi = max(s.hi, k[e]);
    });
    g.counts(s.open, s.lo, s.hi);
    return s;
  }

  // A key that at least `want` entries reach, few more: see the head of the file.
  __device__ uint32_t lower_bound(uint32_t want, const Stats& s, int kind) {
    uint32_t best[kChunks], n = 0;
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      best[c] = 0u;
#pragma unroll
      for (int e = 0; e < V; e++) best[c] = max(best[c], k[c * V + e]);
      n += best[c] != 0u;
    }
    if (g.total(n) < want) return s.lo;
    uint32_t lo = s.lo, cur = s.hi;  // count(best >= lo) >= want; cur + 1 does not reach it
    for (int step = 0; cur > lo && step < 40; step++) {
      const uint32_t p = pivot(lo, cur, step, kind);
      n = 0;
#pragma unroll
      for (int c = 0; c < kChunks; c++) n += best[c] >= p;
      n = g.total(n);
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
    each([&](int e) { mine += k[e] >= from; });
    uint32_t seen = g.ahead(__reduce_add_sync(0xffffffffu, mine), &all);
    if (all > kList) return all;
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      if (!in_use(c)) continue;
      uint32_t in = 0;
#pragma unroll
      for (int e = 0; e < V; e++) in += k[c * V + e] >= from;
      const uint32_t incl = warp_scan(in, g.lane);
      uint32_t r = seen + incl - in;
#pragma unroll
      for (int e = 0; e < V; e++)
        if (k[c * V + e] >= from) {
          list->key[r] = k[c * V + e];
          list->where[r] = index(c * V + e);
          r++;
        }
      seen += __shfl_sync(0xffffffffu, incl, 31);
    }
    return all;
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

  // Drops the entries below the cut c and all but the first `ties` of the
  // `all` at it.
  __device__ void apply(uint32_t cut, uint32_t ties, uint32_t all) {
    if (ties >= all) {
      each([&](int e) { if (k[e] < cut) k[e] = 0u; });
    } else {
      uint32_t mine = 0;
      each([&](int e) { mine += k[e] == cut; });
      uint32_t seen = g.ahead(__reduce_add_sync(0xffffffffu, mine));
#pragma unroll
      for (int c = 0; c < kChunks; c++) {
        if (!in_use(c)) continue;
        uint32_t in = 0;
#pragma unroll
        for (int e = 0; e < V; e++) in += k[c * V + e] == cut;
        const uint32_t incl = warp_scan(in, g.lane);
        uint32_t r = seen + incl - in;
#pragma unroll
        for (int e = 0; e < V; e++) {
          const uint32_t key = k[c * V + e];
          if (key == cut) {
            if (r >= ties) k[c * V + e] = 0u;
            r++;
          } else if (key < cut) {
            k[c * V + e] = 0u;
          }
        }
        seen += __shfl_sync(0xffffffffu, incl, 31);
      }
    }
    find_live();
  }

  // top-p's search by approximate weights: f32 exponentials in units of 2^-20
  // of the largest, summed as integers (a warp's at most 2^31). An entry above half a unit has |x| <=
  // 21 ln 2; three f32 roundings of the exponent and ex2's 2^-22 put its weight
  // within 3e-6, and for probabilities lg2's 2^-22 of log2 v and of log2 m add
  // 3.4e-7 (|log2 m| + 21 T) / T. A mass that clears the goal by `err` of the
  // total and half a unit an entry is on its side for certain; the first pivot
  // that does not leaves [lo, cur] to the 64-bit search. What it usually
  // leaves is one value.
  __device__ void narrow(double top_p, uint32_t open, int kind, uint32_t& lo, uint32_t& cur) {
    uint32_t q[kCached ? E : 1], all = 0;
    const float mv = float(m), it = float(inv_t) * (kind == kKindP ? 1.0f : 1.44269504f);
    const float mu = kind == kKindP ? log2_fast(mv) : mv;
    auto units = [&](uint32_t key) {
      const float v = value_of(key);
      const float u = ((kind == kKindP ? log2_fast(v) : v) - mu) * it;
      return __float2uint_rn(exp2_fast(fminf(u, 0.0f)) * kUnit);
    };
    each([&](int e) {
      const uint32_t x = k[e] ? units(k[e]) : 0u;
      if constexpr (kCached) q[e] = x;
      all += x;
    });
    const double total = g.sum_u32(all);
    const double goal = top_p * total;
    const double err = (1e-5 + 1e-5 * inv_t + 4e-7 * fabs(double(mu)) * (kind == kKindP ? inv_t : 0.0)) * total +
                       0.5 * open + 1.0;
    const double above = goal + err, below = goal - err;
    for (int step = 0; cur != lo; step++) {
      const uint32_t p = pivot(lo, cur, step, kind);
      uint32_t mass = 0, mn = 0xffffffffu, mx = 0u;
      each([&](int e) {
        if (k[e] >= p) {
          if constexpr (kCached) mass += q[e];
          else mass += units(k[e]);
          mn = min(mn, k[e]);
        } else {
          mx = max(mx, k[e]);
        }
      });
      const double a = g.masses(mass, mn, mx);
      if (a >= above) lo = mn;
      else if (a < below) cur = mx;
      else return;
    }
  }

  // What the weights need of the row: s.hi is its largest key.
  __device__ void begin(const Cut& c, const Stats& s, int kind) {
    plain_p = kind == kKindP && c.inv_t == 1.0;
    power = kind == kKindP && !plain_p;
    inv_t = c.inv_t;
    top = s.open ? s.hi : 0xbf800000u;  // (some number)
    m = double(value_of(top));
    log_m = power ? log_tab(value_of(top), t.c, t.l) : 0.0;
  }

  // The cuts; afterwards k[e] != 0 exactly for what top-k and top-p keep (min-p
  // and the dropping are left to the weights' pass).
  __device__ void cut(const Cut& c, const Stats& s, int kind) {
    if (s.open == 0) return;
    uint32_t left = s.open, lo = s.lo;
    const uint32_t top = s.hi;
    if (c.k && c.k < s.open) {
      // the largest t with count(k >= t) >= c.k; `above`: count(k > t's bracket)
      uint32_t cur = top, above = 0, at_lo = s.open;
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
      narrow(c.top_p, left, kind, lo, cur);
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
  }
};

template <int S> using ListRow = Row<S, 1, 1, 1>;

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
    if (!r.in_use(s)) continue;
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
      if (kept[s] >> lane & 1u) out[r.where[s * 32 + lane]] = float(w[s] * inv);
  }
  return d;
}

// The draw of a row that stayed spread over its group, after its cuts.
template <typename R, int V>
__device__ __forceinline__ void finish(R& r, const Cut& c, const DrawArg& a, uint32_t row, const RowAt& at, int n,
                                       bool fits) {
  constexpr int E = sizeof(r.k) / 4;
  const int lane = r.g.lane;
  // the weights, their prefix sums chunk by chunk in bank order
  const double floor_w = c.min_p * (r.plain_p ? r.m : 1.0);
  double incl[R::kChunks], w[R::kCached ? E : 1], run = 0.0;
  uint32_t kept = 0, last = 0u;
#pragma unroll
  for (int ch = 0; ch < R::kChunks; ch++) {
    incl[ch] = run;
    if (!r.in_use(ch)) continue;
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
      const bool past = r.in_use(ch) && fma(u, z, -(before + incl[ch])) < 0.0;
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
    r.each([&](int e) {
      if (r.k[e] == r.top) hit = min(hit, r.index(e));
    });
  }
  r.g.counts(kept, hit, last);
  if (kept && hit == 0xffffffffu) hit = last - 1u;
  const double inv = kept ? 1.0 / z : 0.0;
  // the owner of the entry writes the row's answer
  const bool lead = r.g.segment() == 0 && lane == 0;
  if (kept == 0) {
    if (lead) {
      if (a.index) a.index[row] = kNone;
      if (a.logp) a.logp[row] = -INFINITY;
      if (a.kept) a.kept[row] = 0u;
    }
  } else {
    double drawn = 0.0;
    r.each([&](int e) {
      const bool mine = r.k[e] && r.index(e) == hit;
      if (__any_sync(0xffffffffu, mine)) {
        const double we = weight(e);
        if (mine) drawn = we;
      }
    });
    if (drawn > 0.0) {
      if (a.index) a.index[row] = hit;
      if (a.logp) a.logp[row] = float(log64(drawn * inv));
    }
    if (lead && a.kept) a.kept[row] = kept;
  }
  if (!a.p || !fits) return;
  float* out = a.p + at.out;
#pragma unroll
  for (int ch = 0; ch < R::kChunks; ch++) {
    const int i = r.at(ch);
    alignas(16) float v[V];
#pragma unroll
    for (int e = 0; e < V; e++) {
      v[e] = 0.0f;
      if (r.in_use(ch)) v[e] = float(weight(ch * V + e) * inv);
    }
    if (i >= 0 && i + V <= n && (reinterpret_cast<uintptr_t>(out + i) & 15) == 0) {
#pragma unroll
      for (int e = 0; e < V; e += 4) *reinterpret_cast<float4*>(out + i + e) = *reinterpret_cast<float4*>(v + e);
    } else {
#pragma unroll
      for (int e = 0; e < V; e++)
        if (i + e >= 0 && i + e < n) out[i + e] = v[e];
    }
  }
}

// The loss of a row after its cuts, and its gradient:
//   loss = -A log pi(a) - beta H(pi), H = log Z - sum w x / Z,
//   dloss/dv_j = (A (pi_j - [j = a]) + beta pi_j (log pi_j + H)) / T
// for what is kept, 0 elsewhere, times the row's weight.
// given: a list's weights, 0 for what is cut.
template <typename T, typename R, int V>
__device__ __forceinline__ void finish(R& r, const Cut& c, const LossArg& a, uint32_t row, const RowAt& at, int n,
                                       bool fits, const double* given = nullptr) {
  constexpr int E = sizeof(r.k) / 4;
  const int lane = r.g.lane;
  const uint32_t act = a.actions[row];
  const bool asked = act != kNone;
  double part = 0.0, px = 0.0, xa = 0.0;
  uint32_t kept = 0, live = 0xffffffffu, dummy = 0u;
  double ws[R::kCached ? E : 1];
  r.each([&](int e) {
    uint32_t& key = r.k[e];
    double x, w;
    if constexpr (V == 1) {
      x = r.x_of(key ? key : r.top);
      w = given[e];
    } else {
      w = r.weight(key, x);
    }
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
  const double log_z = kept ? log64(z) : 0.0, inv_z = kept ? 1.0 / z : 0.0;
  const double h = kept ? log_z - sx * inv_z : 0.0;
  const double logp = xa - log_z;
  const bool learns = asked && live == 0u && !c.greedy;  // one answer has no gradient
  const double adv = double(a.advantage[row]), beta = double(a.beta);
  if (r.g.segment() == 0 && lane == 0) {
    if (a.loss) a.loss[row] = learns ? float(-adv * logp - beta * h) : 0.0f;
    if (a.logp) a.logp[row] = !asked ? 0.0f : live == 0u ? float(logp) : -INFINITY;
    if (a.entropy) a.entropy[row] = float(h);
  }
  if (!a.grad || !fits) return;
  T* out = static_cast<T*>(a.grad) + at.out;
  const double g0 = (a.row_weight ? double(a.row_weight[row]) : 1.0) * c.inv_t, base = h - log_z;
  auto slope = [&](int e) {
    const uint32_t key = r.k[e];
    double x, pi;
    if constexpr (R::kCached) {
      x = r.x_of(key ? key : r.top);
      pi = ws[e] * inv_z;
    } else {
      pi = r.weight(key, x) * inv_z;
    }
    const double one = key && r.index(e) == act ? 1.0 : 0.0;
    return key ? float(g0 * fma(adv, pi - one, beta * pi * (x + base))) : 0.0f;
  };
  if constexpr (V == 1) {
    if (learns)
      r.each([&](int e) {
        const float d = slope(e);
        if (r.k[e]) out[r.index(e)] = from_f32<T>(d);
      });
  } else {
    RowWriter<T> writer(out, n, lane, r.i0);
#pragma unroll
    for (int ch = 0; ch < R::kChunks; ch++) {
      float f[V];
      uint32_t v[4];
#pragma unroll
      for (int e = 0; e < V; e++) {
        f[e] = 0.0f;
        if (learns && r.in_use(ch)) f[e] = slope(ch * V + e);
      }
#pragma unroll
      for (int e = 0; e < V; e += 2) set2<T>(v, e, f[e], f[e + 1]);
      writer.put(v, r.at(ch));
    }
    writer.finish();
  }
}

// Whether a row keeps the stated bound and the group holds it, misaligned as it is.
template <typename T>
__device__ __forceinline__ bool row_fits(const RowsArg& r, const RowAt& at, uint32_t cap) {
  const uint32_t shift = uint32_t((reinterpret_cast<uintptr_t>(static_cast<const T*>(r.values) + at.in) & 15) / sizeof(T));
  return at.n <= r.row_len && at.n + shift <= cap;
}

// The output laid out like the rows, and which of the two finishes it takes.
template <typename T> __device__ __forceinline__ void clear_out(const DrawArg& a, const RowAt& at, int n, int tid, int threads) {
  if (a.p) clear_row(a.p + at.out, n, tid, threads);
}
template <typename T> __device__ __forceinline__ void clear_out(const LossArg& a, const RowAt& at, int n, int tid, int threads) {
  if (a.grad) clear_row(static_cast<T*>(a.grad) + at.out, n, tid, threads);
}
template <typename T, int V, typename R>
__device__ __forceinline__ void finish_as(R& r, const Cut& c, const DrawArg& a, uint32_t row, const RowAt& at, int n, bool fits) {
  finish<R, V>(r, c, a, row, at, n, fits);
}
template <typename T, int V, typename R>
__device__ __forceinline__ void finish_as(R& r, const Cut& c, const LossArg& a, uint32_t row, const RowAt& at, int n, bool fits) {
  finish<T, R, V>(r, c, a, row, at, n, fits);
}

// The finish of a list whose weights are known: a draw to be reported, or a
// loss that has been written.
template <typename T, int S>
__device__ __forceinline__ Drawn finish_list(ListRow<S>& r, const Cut& c, const DrawArg& a, uint32_t, const RowAt& at,
                                             bool fits, double u, double* w) {
  return draw_list<S>(r, c, a, at, fits, u, w);
}
template <typename T, int S>
__device__ __forceinline__ Drawn finish_list(ListRow<S>& r, const Cut& c, const LossArg& a, uint32_t row,
                                             const RowAt& at, bool fits, double, double* w) {
  finish<T, ListRow<S>, 1>(r, c, a, row, at, int(at.n), fits, w);
  return Drawn{kNone, 0u, 0.0};
}

// Everything after the gathering, by one warp on a list of n <= 32 S entries.
template <typename T, int S, typename Arg>
__device__ __forceinline__ Drawn list_as(List& list, uint32_t n, const Tables& tables, int lane, const Cut& c,
                                         const Arg& a, uint32_t row, const RowAt& at, bool fits, double u) {
  ListRow<S> r(lane, tables);
  r.take(list, n);
  const bool cuts = (c.k && c.k < n) || c.top_p < 1.0;
  constexpr bool pairs = S <= kPairs / 32;
  const Stats s = r.list_stats(n, cuts && !pairs);
  r.begin(c, s, a.r.kind);
  if (!pairs && cuts) r.cut(c, s, a.r.kind);
  double w[S];
#pragma unroll
  for (int e = 0; e < S; e++) {
    w[e] = 0.0;
    if (r.in_use(e)) w[e] = r.weight(r.k[e]);
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
// CTAs an SM. More warps hide more of a row's latency, more registers spill
// less: 34818 drawn rows took 95, 109 and 102 us with 6, 7 and 8, the loss of
// 4096 rows 20.6, 18.1 and 19.6.
template <typename Arg> constexpr int kSmallCtas = 6;
template <> constexpr int kSmallCtas<LossArg> = 7;
template <typename T, typename Arg>
__global__ void __launch_bounds__(128, kSmallCtas<Arg>) k_policy_small(const __grid_constant__ Arg a) {
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

// Longer rows: CL CTAs of W warps a row. A CTA on its own (CL = 1) takes
// `batch` rows, one after another up to their lists, which its warps then
// finish side by side: one warp at the end of one row would leave the SM idle.
// FIT CTAs share an SM: three of eight warps where lists are what rows come to
// (top-k), two where a row stays in its registers (top-p alone).
constexpr int kBatch = 8;
template <typename T, int E, int W, int CL, int FIT, typename Arg>
__global__ void __launch_bounds__(W * 32, FIT) k_policy_rows(const __grid_constant__ Arg a,
                                                                                       uint32_t batch) {
  constexpr int V = 16 / int(sizeof(T)), kLists = CL > 1 ? 1 : W < kBatch ? W : kBatch;
  using R = Row<E, V, W, CL>;
  __shared__ typename Group<W, CL>::Shared sh;
  __shared__ List lists[kLists];
  __shared__ struct { RowAt at; uint32_t row, count; } todo[kLists];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Tables tables(lane, a.r.kind == kKindP);
  uint32_t made = 0;
  for (uint32_t b = 0; b < batch; b++) {
    const uint32_t row = blockIdx.x / CL * batch + b;
    RowAt at;
    if (row >= a.r.rows || !locate(a.r, a.out_pitch, row, lane, &at)) break;
    R r(sh, tables, lane, warp);
    const bool fits = row_fits<T>(a.r, at, R::kCap);
    const uint32_t n = fits ? uint32_t(at.n) : 0u;
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
    if (count <= kList) {
      // (grad and p may lie over the values: this row's have been read)
      if (fits) clear_out<T>(a, at, int(n), r.g.rank * W * 32 + int(threadIdx.x), W * 32 * CL);
      if (threadIdx.x == 0) {
        todo[made].at = at;
        todo[made].row = row;
        todo[made].count = count;
      }
      made++;
    } else {
      if (from != s.lo) {  // top-k's search starts from the smallest entry at or above the bound
        uint32_t mn = 0xffffffffu, none = 0, mx = 0;
        r.each([&](int e) {
          if (r.k[e] >= from) mn = min(mn, r.k[e]);
        });
        r.g.counts(none, mn, mx);
        s.lo = mn;
        s.open = count;
      }
      r.begin(c, s, a.r.kind);
      r.cut(c, s, a.r.kind);
      finish_as<T, V>(r, c, a, row, at, int(n), fits);
    }
    if (W > 1 && b + 1 < batch) __syncthreads();  // the group's slots start again with the next row
  }
  if constexpr (CL > 1) cooperative_groups::this_cluster().sync();
  else __syncthreads();
  if (warp >= int(made) || (CL > 1 && cooperative_groups::this_cluster().block_rank() != 0)) return;
  const RowAt at = todo[warp].at;
  const uint32_t row = todo[warp].row;
  const bool fits = row_fits<T>(a.r, at, R::kCap);
  Answers<Arg> answers;
  answers.take(list_row<T>(lists[warp], todo[warp].count, tables, lane, cut_of(a.c, row), a, row, at, fits,
                           answers.uniform(a, row)), a, row, lane);
  answers.done(a, row, lane);
}

}  // namespace pol
}  // namespace kc
