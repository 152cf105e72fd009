// az_sample.hip -- draws an action a row from truncated policy logits (include/az_layers.h).
// Part of libaz_mcts.so (gfx950 only).
//
// Every truncation keeps a prefix of the row's descending order, so a row's legal actions are cut at one logit, or
// at one index among the actions that share it; no row is sorted.  The cut is found by histograms of counts
// (top_k) or weights (top_p): first over logit / temperature in linear bins, whose bins a row of logits fills
// evenly, then over the order-preserving integer of the logit within the bin that holds the cut, until that bin is a
// single logit.  Weights are summed as 64-bit integers: the order of the LDS atomics does not matter.
//
// Up to 1024 actions a wave takes a row, which it holds in LDS.  Beyond, a workgroup holds the row in registers (up to
// 32768 actions; wider rows are read from L2 again), takes the first histogram over it -- for top_k over the threads'
// largest logits alone -- and moves the actions of the bins up to the cut's, in index order, into a list in LDS; one wave
// ends the draw on a short list, all of them on a long one.  Of up to 256 candidates every one is compared with every
// other: that gives each its place in the descending order and the weight ahead of it at once.  A row whose list would
// not fit (ties, a flat distribution) is left to a second kernel that works over the row in memory.
//
// 4096 x 32768 float32, top_k 100 and top_p 0.9: 164 us, of which reading the 537 MB takes 126-139 in this form (104 at a
// large copy's rate: two rows a compute unit are in flight, as many as the registers hold); 4096 x 362 with a mask and
// top_p: 15 us, the latency of a wave's steps; 64 x 18: 5 us.  Bound by the weights' exponentials in 64 bits instead:
// top_p alone over 4096 x 32768, for normal logits of deviation 2.5 0.48 ms at 0.8 (all rows end in the list), 0.88 at 0.9, 1.6
// at 0.95, 1.9 for equal logits; no cut 0.29.  2048 x 65536, whose rows are read again for each pass, 296 us (as above).
#include <hip/hip_runtime.h>

#include <cfloat>

#include "az_host.h"
#include "az_types.h"

namespace {

typedef unsigned long long u64;

constexpr double LEAST = 0x1p-40;   // weights below this share of the largest are never drawn
constexpr int LIST = 4096;          // actions of the list
constexpr int BINS = 2048;          // of the workgroup's histogram

__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l + 0.0f);   // (-0 and +0 are one logit)
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float((key >> 31) ? key ^ 0x80000000u : ~key);
}

// exp(x) for x <= 0, to about one unit in the last place down to 2^-1000 (then 0): 2^n times the Taylor polynomial
// of degree 13 on |r| <= ln 2 / 2, whose remainder is below 2^-57.
__device__ __forceinline__ double exp_neg(double x) {
  const double n = rint(x * 1.4426950408889634);
  double r = fma(n, -0x1.62e42fefa38p-1, x);       // ln 2 in two parts, the first with zeros at its end
  r = fma(n, -0x1.ef35793c7673p-45, r);
  double p = 1.0 / 6227020800.0;
  p = fma(p, r, 1.0 / 479001600.0);
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return x < -690.0 ? 0.0 : ldexp(p, (int)fmax(n, -1000.0));
}

// A row's weights: exp((l - top) / temperature), also in units of 1 / unit, rounded.
struct Weights {
  float top;
  double inv_t, unit;
  __device__ __forceinline__ double operator()(float l) const { return exp_neg(((double)l - (double)top) * inv_t); }
  __device__ __forceinline__ u64 whole(double w) const {   // (w * unit <= 2^51)
    return (u64)__double_as_longlong(fma(w, unit, 0x1p52)) - 0x4330000000000000ull;
  }
  __device__ __forceinline__ u64 mass(float l) const { return whole((*this)(l)); }
  // linear bins over 32 temperatures below the top; the last one takes what is beyond
  __device__ __forceinline__ float scale(int bins) const { return (float)fmin(inv_t * (bins / 32), 1e30); }
};

// (halves, whose difference is finite for any two logits)
__device__ __forceinline__ float place_of(float top, float l, float scale) {
  return fmaf(l, -0.5f, 0.5f * top) * (2.0f * scale);
}

__device__ __forceinline__ int bin_of(float top, float l, float scale, int bins) {
  return (int)fminf(place_of(top, l, scale), (float)(bins - 1));
}

// ---------------------------------------------------------------------------
// Rows: `fetch(c, l)` gives this lane's V logits of chunk c (64 V consecutive actions of its wave's run), -inf where there
// is no legal action, `index(c, v)` their actions; chunks, lanes, elements in this order are in index order.

// in memory, spread over NT threads
template <typename T, int NT>
struct MemoryRow {
  static constexpr int V = 16 / sizeof(T), THREADS = NT;
  const T* logits;
  const uint8_t* invalid;
  int actions, chunks, start;   // start: this lane's first action
  bool infinite;                // +inf logits are present: they become 0, all others -inf

  __device__ __forceinline__ void init(const T* l, const uint8_t* inv, int n, int chunks_) {
    logits = l, invalid = inv, actions = n, infinite = false, chunks = chunks_;
    start = (threadIdx.x >> 6) * chunks * 64 * V + (threadIdx.x & 63) * V;
  }
  __device__ __forceinline__ int index(int c, int v) const { return start + c * 64 * V + v; }
  __device__ __forceinline__ void fetch(int c, float* l) const {
    const int i = start + c * 64 * V;
    if (i + V <= actions) {
      const AzVec<T, V> r = az_loadu<T, V>(logits + i);
      for (int v = 0; v < V; ++v) l[v] = (float)r.v[v];
      if (invalid) {
        const AzVec<uint8_t, V> m = az_loadu<uint8_t, V>(invalid + i);
        for (int v = 0; v < V; ++v)
          if (m.v[v]) l[v] = -INFINITY;
      }
    } else {
      for (int v = 0; v < V; ++v)
        l[v] = i + v < actions && !(invalid && invalid[i + v]) ? (float)logits[i + v] : -INFINITY;
    }
    for (int v = 0; v < V; ++v) {
      if (l[v] != l[v]) l[v] = -INFINITY;
      if (infinite) l[v] = l[v] == INFINITY ? 0.0f : -INFINITY;
    }
  }
};

// in LDS, spread over NT threads
template <int NT>
struct ListRow {
  static constexpr int V = 1, THREADS = NT;
  const float* l;
  const int* at;    // null: the place itself
  int n, chunks;
  __device__ __forceinline__ int place(int c) const {
    return ((NT > 64 ? (threadIdx.x >> 6) * chunks : 0) + c) * 64 + (threadIdx.x & 63);
  }
  __device__ __forceinline__ int index(int c, int) const {
    const int j = place(c);
    return at ? (j < n ? at[j] : 0) : j;
  }
  __device__ __forceinline__ void fetch(int c, float* x) const {
    const int j = place(c);
    *x = j < n ? l[j] : -INFINITY;
  }
};

// f(logit, action) for each legal action of this thread
template <typename Row, typename F>
__device__ __forceinline__ void each(const Row& row, F&& f) {
  for (int c = 0; c < row.chunks; ++c) {
    float l[Row::V];
    row.fetch(c, l);
    for (int v = 0; v < Row::V; ++v)
      if (l[v] > -INFINITY) f(l[v], row.index(c, v));
  }
}

// ---------------------------------------------------------------------------
template <int NT, int NB>
struct Shared {
  u64 bins[NB];
  u64 waves[NT / 64];
  u64 found_before;
  uint32_t lo, hi;
  int found, index;
};

// Orders LDS accesses of a row's threads; a single wave needs no barrier (and has none: the workgroup's other waves
// may have ended).
template <int NT>
__device__ __forceinline__ void sync() {
  if constexpr (NT == 64) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}

__device__ __forceinline__ u64 shfl_up64(u64 x, int d) {
  const uint32_t lo = __shfl_up((uint32_t)x, d), hi = __shfl_up((uint32_t)(x >> 32), d);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 shfl_xor64(u64 x, int d) {
  const uint32_t lo = __shfl_xor((uint32_t)x, d), hi = __shfl_xor((uint32_t)(x >> 32), d);
  return (u64)hi << 32 | lo;
}

__device__ __forceinline__ u64 wave_sum(u64 x) {
  for (int off = 32; off > 0; off >>= 1) x += shfl_xor64(x, off);
  return x;
}

__device__ __forceinline__ u64 wave_scan(u64 x) {   // inclusive
  const int lane = threadIdx.x & 63;
  for (int off = 1; off < 64; off <<= 1) {
    const u64 y = shfl_up64(x, off);
    if (lane >= off) x += y;
  }
  return x;
}

// Sum over the threads' x, and of the waves before this one.
template <int NT, typename S>
__device__ __forceinline__ u64 group_sum(u64 x, S& s, u64* ahead) {
  x = wave_sum(x);
  *ahead = 0;
  if constexpr (NT == 64) return x;
  sync<NT>();
  if ((threadIdx.x & 63) == 0) s.waves[threadIdx.x >> 6] = x;
  sync<NT>();
  u64 total = 0;
  for (int w = 0; w < NT / 64; ++w) {
    if (w == (int)(threadIdx.x >> 6)) *ahead = total;
    total += s.waves[w];
  }
  return total;
}

// Where the prefix ends: logits with a key above `key` are in, of those equal to it the first `ties`.
struct Cut {
  uint32_t key;
  u64 ties;       // all of them: ~0
};

// A number in [0, 1) as m / 2^shift, for exact shares of integer sums.
struct Share {
  u64 m;
  int shift;
  __device__ __forceinline__ explicit Share(double x) {   // (subnormal numbers count as 0)
    const u64 bits = (u64)__double_as_longlong(x);
    const int e = (int)(bits >> 52);
    m = e ? (bits & 0xfffffffffffffull) | 1ull << 52 : 0;
    shift = 1075 - e;
  }
  // n times it, rounded down or up
  __device__ __forceinline__ u64 of(u64 n, bool up) const {
    u64 hi = __umul64hi(n, m), lo = n * m;
    if (shift >= 128) return up && (hi | lo) ? 1 : 0;
    if (shift >= 64) {
      const u64 cut = shift == 64 ? 0 : hi & ((1ull << (shift - 64)) - 1);
      return (hi >> (shift - 64)) + (up && (cut | lo) ? 1 : 0);
    }
    return (hi << (64 - shift) | lo >> shift) + (up && (lo & ((1ull << shift) - 1)) ? 1 : 0);
  }
};

// Scans the bins: the first whose inclusive sum, with `before`, reaches the goal is left in s.found (NB: none),
// the sum ahead of it in s.found_before.  With a `share` below 1 the goal is that share of the bins' total but `less` (of
// the first one at least).
template <int NT, int NB>
__device__ __forceinline__ u64 find(Shared<NT, NB>& s, u64 before, u64 goal, double share = 1.0, u64 less = 0) {
  constexpr int PER = NB / NT;
  const int t = threadIdx.x & (NT - 1);
  u64 mine = 0, ahead, h[PER];
  for (int i = 0; i < PER; ++i) mine += h[i] = s.bins[t * PER + i];
  const u64 scan = wave_scan(mine);
  const u64 total = group_sum<NT>(mine, s, &ahead);
  if (t == 0) s.found = NB;
  sync<NT>();
  if (share < 1.0) {
    goal = Share(share).of(total - less, true);
    if (goal == 0) goal = 1;
  }
  u64 cum = before + ahead + scan - mine;
  for (int i = 0; i < PER; ++i) {   // one bin crosses at most
    const u64 next = cum + h[i];
    if (cum < goal && next >= goal) s.found = t * PER + i, s.found_before = cum;
    cum = next;
  }
  sync<NT>();
  return goal;
}

template <int NT, int NB>
__device__ __forceinline__ void clear(Shared<NT, NB>& s) {
  sync<NT>();
  for (int i = threadIdx.x & (NT - 1); i < NB; i += NT) s.bins[i] = 0;
  sync<NT>();
}

template <bool MASS, int NT, int NB>
__device__ __forceinline__ void count(Shared<NT, NB>& s, int bin, const Weights& w, float l) {
  if constexpr (MASS)
    atomicAdd(&s.bins[bin], w.mass(l));
  else
    atomicAdd(reinterpret_cast<uint32_t*>(&s.bins[bin]), 1u);
}

// Where a top_k cut falls into the last bin, whose actions are never drawn: the weight of those behind its first `kept`, which
// are out of the weight that top_p is a share of.  Their weights are at most 33 units (2^51 e^-31.875), so the numbers
// of actions of each weight tell it; from 38 temperatures on they are none (2^51 e^-38 < 1 / 2).  `over(f)` calls f for
// each legal logit.
template <int NT, int NB, typename Over>
__device__ __forceinline__ u64 beyond(Shared<NT, NB>& s, const Weights& w, u64 kept, Over&& over) {
  const float scale = w.scale(NB);
  clear(s);
  over([&](float l) {
    const float at = place_of(w.top, l, scale);
    if (at >= NB - 1 && at < 38.0f * (NB / 32)) {
      const u64 m = w.mass(l);
      if (m > 0) atomicAdd(reinterpret_cast<uint32_t*>(&s.bins[m < 63 ? m : 63]), 1u);
    }
  });
  sync<NT>();
  u64 less = 0;
  for (int m = 63; m >= 0; --m) {
    const u64 n = s.bins[m], in = n < kept ? n : kept;
    kept -= in;
    less += (n - in) * m;
  }
  return less;
}

// The shortest prefix of the descending order, among logits with a key >= `least`, whose counts (MASS: weights) sum up
// to the goal; false if there is none (no cut).
template <bool MASS, int NB, typename Row>
__device__ __forceinline__ bool select(const Row& row, Shared<Row::THREADS, NB>& s, const Weights& w, u64 goal, double share,
                       uint32_t least, u64 less, Cut* cut) {
  constexpr int NT = Row::THREADS;
  const float scale = w.scale(NB);
  clear(s);
  each(row, [&](float l, int) {
    if (key_of(l) >= least) count<MASS>(s, bin_of(w.top, l, scale, NB), w, l);
  });
  sync<NT>();
  goal = find(s, 0, goal, share, less);
  const int bin = s.found;
  u64 before = s.found_before;
  // (a count that ends in the last bin cuts only weights that are never drawn)
  if (bin == NB || (!MASS && bin == NB - 1)) return false;
  if ((threadIdx.x & (NT - 1)) == 0) s.lo = 0xffffffffu, s.hi = 0;
  sync<NT>();
  uint32_t lo = 0xffffffffu, hi = 0;
  each(row, [&](float l, int) {
    const uint32_t k = key_of(l);
    if (k >= least && bin_of(w.top, l, scale, NB) == bin) lo = min(lo, k), hi = max(hi, k);
  });
  if (lo <= hi) atomicMin(&s.lo, lo), atomicMax(&s.hi, hi);
  sync<NT>();
  lo = s.lo, hi = s.hi;
  while (lo < hi) {
    const int bits = 32 - __clz(hi - lo), shift = max(0, bits - (31 - __clz(NB)));
    clear(s);
    each(row, [&](float l, int) {
      const uint32_t k = key_of(l);
      if (k >= lo && k <= hi) count<MASS>(s, (hi - k) >> shift, w, l);
    });
    sync<NT>();
    find(s, before, goal);
    // (the sums over these keys are those of the bin that crossed, so one of its bins crosses)
    if (s.found >= NB) break;
    const uint32_t b = s.found;
    before = s.found_before;
    hi -= b << shift;
    const uint32_t width = (1u << shift) - 1;
    lo = hi - lo > width ? hi - width : lo;
    sync<NT>();
  }
  cut->key = lo;
  // the fewest ties that reach the goal
  const u64 one = MASS ? w.mass(logit_of(lo)) : 1;
  cut->ties = one > 1 ? (goal - before + one - 1) / one : goal - before;
  return true;
}

// The action at which the running sum of `value`, in index order, first exceeds `target` (less than the total).
template <int NB, typename Row, typename F>
__device__ __forceinline__ int at_sum(const Row& row, Shared<Row::THREADS, NB>& s, u64 target, F&& value) {
  constexpr int NT = Row::THREADS, V = Row::V;
  u64 ahead = 0;
  bool here = true;
  if constexpr (NT > 64) {
    u64 mine = 0;
    each(row, [&](float l, int i) { mine += value(l, i); });
    const u64 in_wave = wave_sum(mine);
    group_sum<NT>(mine, s, &ahead);
    here = target >= ahead && target < ahead + in_wave;
  }
  if (here) {   // this wave has it: chunk by chunk
    u64 run = ahead;
    for (int c = 0; c < row.chunks; ++c) {
      float l[V];
      u64 x[V], sum = 0;
      row.fetch(c, l);
      for (int v = 0; v < V; ++v) sum += x[v] = l[v] > -INFINITY ? value(l[v], row.index(c, v)) : 0;
      const u64 scan = wave_scan(sum);
      const u64 total = (u64)__shfl((uint32_t)(scan >> 32), 63) << 32 | (u64)(uint32_t)__shfl((uint32_t)scan, 63);
      if (target < run + total) {
        const u64 mask = __ballot(target < run + scan);
        if ((int)(threadIdx.x & 63) == __ffsll(mask) - 1) {
          u64 cum = run + scan - sum;
          int found = -1;
          for (int v = 0; v < V; ++v) {
            cum += x[v];
            if (found < 0 && target < cum) found = row.index(c, v);
          }
          s.index = found;
        }
        break;
      }
      run += total;
    }
  }
  sync<NT>();
  return s.index;
}

struct Options {
  int top_k;          // 0: all
  double top_p;       // 1: all
  double min_p;       // at least LEAST
  float uniform;
  u64 goal;           // the weight that top_p asks for where it is known (0: the row has it)
};

struct Result {
  int action;
  double mass;        // of the kept actions, as a share of the largest weight
};

__device__ __forceinline__ u64 target_of(float u, u64 total) {
  u64 target = u > 0.0f ? total : 0;   // (not a number: 0)
  if (u > 0.0f && u < 1.0f) target = Share((double)u).of(total, false);
  return target >= total ? total - 1 : target;
}

// The whole draw over a row.
template <int NB, typename Row>
__device__ __forceinline__ Result draw(const Row& row, Shared<Row::THREADS, NB>& s, const Weights& w, const Options& o) {
  constexpr int NT = Row::THREADS;
  Cut cut = {0, ~0ull};
  u64 less = 0;
  auto ties_of = [&](uint32_t key) {
    u64 ties = 0, ahead;
    each(row, [&](float l, int) { ties += key_of(l) == key; });
    return group_sum<NT>(ties, s, &ahead);
  };
  if (o.top_k > 0) {
    Cut c;
    if (select<false>(row, s, w, (u64)o.top_k, 1.0, 0, 0, &c))
      cut = c;
    else if (s.found == NB - 1 && o.top_p < 1.0 && !o.goal)
      less = beyond(s, w, (u64)o.top_k - s.found_before, [&](auto&& f) { each(row, [&](float l, int) { f(l); }); });
  }
  if (o.top_p < 1.0) {
    // the weight of the ties at the top_k cut that are out
    if (cut.key && !o.goal) less = (ties_of(cut.key) - cut.ties) * w.mass(logit_of(cut.key));
    Cut c;
    if (select<true>(row, s, w, o.goal, o.goal ? 1.0 : o.top_p, cut.key, less, &c)) {
      if (c.key > cut.key)
        cut = c;
      else if (c.key == cut.key && c.ties < cut.ties)
        cut.ties = c.ties;
    }
  }
  int last_tie = 0x7fffffff;
  if (cut.ties != ~0ull && cut.ties < ties_of(cut.key)) {
    const uint32_t key = cut.key;
    last_tie = at_sum(row, s, cut.ties - 1, [&](float l, int) { return (u64)(key_of(l) == key); });
  }
  auto kept = [&](float l, int i) -> u64 {
    const uint32_t k = key_of(l);
    if (k < cut.key || (k == cut.key && i > last_tie)) return 0;
    const double x = w(l);
    return x >= o.min_p ? w.whole(x) : 0;
  };
  u64 mine = 0, ahead;
  each(row, [&](float l, int i) { mine += kept(l, i); });
  const u64 total = group_sum<NT>(mine, s, &ahead);
  return {at_sum(row, s, target_of(o.uniform, total), kept), (double)total / w.unit};
}

// The whole draw over at most FEW actions in LDS (their indices `at`, or their places), by one wave: E a lane.
constexpr int FEW = 256;

struct FewScratch {
  u64 order[FEW];    // key, then the place from behind: greater is earlier in the descending order
  u64 mass[FEW];
};

template <int E>
__device__ __forceinline__ Result draw_ranked(const float* l, const int* at, int n, FewScratch& s, const Weights& w,
                                              const Options& o) {
  const int lane = threadIdx.x & 63;
  uint32_t rank[E];
  u64 order[E], m[E], ahead[E];
  double x[E];
  bool in[E];
  for (int e = 0; e < E; ++e) {
    const int i = e * 64 + lane;
    const float v = i < n ? l[i] : -INFINITY;
    in[e] = v > -INFINITY;
    order[e] = (u64)key_of(v) << 32 | (uint32_t)~i;
    x[e] = in[e] ? w(v) : 0.0;
    m[e] = w.whole(x[e]);
    rank[e] = 0, ahead[e] = 0;
    s.mass[i] = m[e], s.order[i] = order[e];
  }
  sync<64>();
#pragma unroll 4
  for (int j = 0; j < n; ++j) {
    const u64 other = s.order[j], mass = s.mass[j];
    for (int e = 0; e < E; ++e) {
      const bool first = other > order[e];
      rank[e] += first;
      ahead[e] += first ? mass : 0;
    }
  }
  u64 sum = 0;
  for (int e = 0; e < E; ++e) {
    in[e] = in[e] && (o.top_k <= 0 || rank[e] < (uint32_t)o.top_k);
    sum += in[e] ? m[e] : 0;
  }
  u64 goal = o.goal;
  if (o.top_p < 1.0 && !goal) {
    goal = Share(o.top_p).of(wave_sum(sum), true);
    if (goal == 0) goal = 1;
  }
  u64 scan[E], total = 0;
  for (int e = 0; e < E; ++e) {
    in[e] = in[e] && (o.top_p >= 1.0 || ahead[e] < goal) && x[e] >= o.min_p;
    scan[e] = total + wave_scan(in[e] ? m[e] : 0);
    total = (u64)__shfl((uint32_t)(scan[e] >> 32), 63) << 32 | (u64)(uint32_t)__shfl((uint32_t)scan[e], 63);
  }
  const u64 target = target_of(o.uniform, total);
  int found = 0;
  for (int e = E - 1; e >= 0; --e) {
    const u64 over = __ballot(target < scan[e]);
    if (over) found = e * 64 + __ffsll(over) - 1;
  }
  return {at ? at[found] : found, (double)total / w.unit};
}

__device__ __forceinline__ Result draw_few(const float* l, const int* at, int n, FewScratch& s, const Weights& w,
                                           const Options& o) {
  if (n <= 64) return draw_ranked<1>(l, at, n, s, w, o);
  if (n <= 128) return draw_ranked<2>(l, at, n, s, w, o);
  if (n <= 192) return draw_ranked<3>(l, at, n, s, w, o);
  return draw_ranked<4>(l, at, n, s, w, o);
}

// ---------------------------------------------------------------------------
__device__ __forceinline__ Options options_of(const az_sample_desc& d, int b, double* temperature) {
  Options o;
  *temperature = d.temperature_rows ? (double)d.temperature_rows[b] : d.temperature;
  o.top_k = d.top_k_rows ? d.top_k_rows[b] : d.top_k;
  o.top_p = d.top_p_rows ? (double)d.top_p_rows[b] : d.top_p;
  o.min_p = d.min_p_rows ? (double)d.min_p_rows[b] : d.min_p;
  o.uniform = d.uniform[b];
  o.goal = 0;
  if (!(*temperature > 1e-300)) *temperature = 1.0, o.top_k = 1;
  if (o.top_k <= 0 || o.top_k >= d.actions) o.top_k = 0;
  o.top_p = o.top_p < 1.0 ? (o.top_p > 0.0 ? o.top_p : 0.0) : 1.0;
  o.min_p = o.min_p > LEAST ? fmin(o.min_p, 1.0) : LEAST;
  return o;
}

template <typename T>
__device__ __forceinline__ void write(const az_sample_desc& d, int b, const Weights& w, const Result& r, int32_t* action,
                                      float* log_prob) {
  action[b] = r.action;
  if (!log_prob) return;
  float l = (float)((const T*)d.logits)[(int64_t)b * d.actions + r.action];
  if (l == INFINITY) l = 0.0f;   // (then the top is 0 too)
  log_prob[b] = (float)(((double)l - (double)w.top) * w.inv_t - log(r.mass));
}

__device__ __forceinline__ void write_none(int b, int32_t* action, float* log_prob) {
  action[b] = 0;
  if (log_prob) log_prob[b] = -INFINITY;
}

// A logit that is at most that of every action in the bins up to `bound`, whatever the roundings of bin_of: taking the
// actions from it on may take some of the next bin along, in which the draw over them finds the same cut.
__device__ __forceinline__ float least_of(float top, float scale, int bound) {
  const float reach = (float)(bound + 1) / scale * (1.0f + 0x1p-18f);
  return fmaxf(top - reach - (fabsf(top) + reach) * 0x1p-20f, -FLT_MAX);   // (finite: above what stands for no action)
}

__device__ __forceinline__ float wave_max(float x) {
  for (int off = 32; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor(x, off));
  return x;
}

// Up to MOST actions: a wave a row, WAVES rows a workgroup.
template <typename T, int MOST, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_sample_wave(az_sample_desc d, int32_t* action, float* log_prob,
                                                            double unit) {
  constexpr int V = 16 / sizeof(T), NB = 256;
  // (the histogram and the candidates' scratch are not used at the same time; 16 rows fit a compute unit's LDS)
  union Scratch {
    Shared<64, NB> s;
    FewScratch few;
    __device__ Scratch() {}
  };
  __shared__ Scratch scratch[WAVES];
  __shared__ float list[WAVES][MOST];
  __shared__ float few[WAVES][FEW];
  __shared__ int few_at[WAVES][FEW];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, b = blockIdx.x * WAVES + wave;
  if (b >= d.rows) return;
  double temperature;
  Options o = options_of(d, b, &temperature);
  MemoryRow<T, 64> memory;
  memory.init((const T*)d.logits + (int64_t)b * d.actions, d.invalid ? d.invalid + (int64_t)b * d.actions : nullptr,
              d.actions, (d.actions + 64 * V - 1) / (64 * V));
  memory.start = lane * V;
  float top = -INFINITY;
  for (int c = 0; c < memory.chunks; ++c) {
    float l[V];
    memory.fetch(c, l);
    for (int v = 0; v < V; ++v) {
      top = fmaxf(top, l[v]);
      if (memory.index(c, v) < d.actions) list[wave][memory.index(c, v)] = l[v];
    }
  }
  top = wave_max(top);
  if (top == -INFINITY) {
    if (lane == 0) write_none(b, action, log_prob);
    return;
  }
  sync<64>();
  if (top == INFINITY) {
    for (int i = lane; i < d.actions; i += 64) list[wave][i] = list[wave][i] == INFINITY ? 0.0f : -INFINITY;
    top = 0.0f;
    sync<64>();
  }
  const Weights w = {top, 1.0 / temperature, unit};
  const float* l = list[wave];
  Result r;
  if (d.actions <= FEW) {
    r = draw_few(l, nullptr, d.actions, scratch[wave].few, w, o);
  } else {
    const ListRow<64> row = {l, nullptr, d.actions, (d.actions + 63) / 64};
    Shared<64, NB>& s = scratch[wave].s;
    // the bin that holds the first cut, and the actions up to it (k_sample_group has the same, over more threads)
    const float scale = w.scale(NB);
    int bound = NB;
    u64 less = 0;
    if (o.top_k > 0) {
      clear(s);
      each(row, [&](float x, int) { count<false>(s, bin_of(top, x, scale, NB), w, x); });
      sync<64>();
      find(s, 0, (u64)o.top_k);
      bound = s.found;
      if (bound == NB - 1 && o.top_p < 1.0)
        less = beyond(s, w, (u64)o.top_k - s.found_before, [&](auto&& f) { each(row, [&](float x, int) { f(x); }); });
      if (bound >= NB - 1) bound = NB, o.top_k = 0;   // nothing that could be drawn is cut
    }
    if (bound == NB && o.top_p < 1.0) {
      clear(s);
      each(row, [&](float x, int) { count<true>(s, bin_of(top, x, scale, NB), w, x); });
      sync<64>();
      o.goal = find(s, 0, 0, o.top_p, less);
      bound = s.found;
    }
    int n = FEW + 1;
    if (bound < NB) {
      const float least = least_of(top, scale, bound);
      n = 0;
      for (int c = 0; c < row.chunks; ++c) {
        float x;
        row.fetch(c, &x);
        const u64 has = __ballot(x >= least);
        const int to = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(has >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)has, 0));
        if (x >= least && to < FEW) few[wave][to] = x, few_at[wave][to] = c * 64 + lane;
        n += __popcll(has);
      }
      sync<64>();
    }
    r = n <= FEW ? draw_few(few[wave], few_at[wave], n, scratch[wave].few, w, o) : draw<NB>(row, s, w, o);
  }
  if (lane == 0) write<T>(d, b, w, r, action, log_prob);
}

// The same value, of which the compiler does not know it: what a pass over the row computes from it is not kept in
// registers for the next pass.
__device__ __forceinline__ float anew(float x) {
  asm volatile("" : "+v"(x));
  return x;
}

// A row in the registers of a workgroup (CHUNKS > 0) or in memory.
template <typename T, int NT, int CHUNKS>
struct FrontRow {
  static constexpr int V = 16 / sizeof(T);
  float reg[CHUNKS > 0 ? CHUNKS : 1][V];
  // f(c, logits) for each chunk
  template <typename F>
  __device__ __forceinline__ void chunks(const MemoryRow<T, NT>& m, F&& f) const {
    if constexpr (CHUNKS > 0) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        f(c, reg[c]);
        __builtin_amdgcn_sched_barrier(0);   // (chunks worked side by side would need the registers of all of them)
      }
    } else {
      for (int c = 0; c < m.chunks; ++c) {
        float l[V];
        m.fetch(c, l);
        f(c, l);
      }
    }
  }
};

// DIRECT: rows that no top_k or top_p truncates.  Otherwise the truncated ones; what does not fit this kernel (a row
// without a cut, a list that is too long) is left with action -1 for k_sample_rest.
template <typename T, int NT, int CHUNKS, bool DIRECT>
__global__ __launch_bounds__(NT, 4) void k_sample_group(az_sample_desc d, int32_t* action, float* log_prob, double unit) {
  constexpr int V = 16 / sizeof(T), NW = NT / 64;
  __shared__ Shared<NT, DIRECT ? NT : BINS> s;
  __shared__ Shared<64, 64> s1;   // (DIRECT)
  __shared__ float list[DIRECT ? 1 : LIST];
  __shared__ int list_at[DIRECT ? 1 : LIST];
  __shared__ FewScratch scratch;
  __shared__ float tops[NW];
  __shared__ int counts[NW];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double temperature;
  Options o = options_of(d, b, &temperature);
  MemoryRow<T, NT> memory;
  memory.init((const T*)d.logits + (int64_t)b * d.actions, d.invalid ? d.invalid + (int64_t)b * d.actions : nullptr,
              d.actions, CHUNKS > 0 ? CHUNKS : (d.actions + NT * V - 1) / (NT * V));
  FrontRow<T, NT, CHUNKS> front;
  if constexpr (CHUNKS > 0) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) memory.fetch(c, front.reg[c]);
  }
  float top = -INFINITY;
  front.chunks(memory, [&](int, const float* l) {
#pragma unroll
    for (int v = 0; v < V; ++v) top = fmaxf(top, l[v]);
  });
  float own = top;   // the thread's largest
  top = wave_max(top);
  if (lane == 0) tops[wave] = top;
  __syncthreads();
  for (int i = 0; i < NW; ++i) top = fmaxf(top, tops[i]);
  top = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(top)));
  if (top == -INFINITY) {
    if (threadIdx.x == 0) write_none(b, action, log_prob);
    return;
  }
  if (top == INFINITY) {
    memory.infinite = true, top = 0.0f;
    own = own == INFINITY ? 0.0f : -INFINITY;
    if constexpr (CHUNKS > 0) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int v = 0; v < V; ++v) front.reg[c][v] = front.reg[c][v] == INFINITY ? 0.0f : -INFINITY;
    }
  }
  const Weights w = {top, 1.0 / temperature, unit};
  if constexpr (DIRECT) {
    // sums over the row, then the one wave that has the action looks for it
    u64 mine = 0, ahead;
    auto kept = [&](float l, int) -> u64 {
      const double x = w(l);
      return x >= o.min_p ? w.whole(x) : 0;
    };
    front.chunks(memory, [&](int, const float* l) {
#pragma unroll
      for (int v = 0; v < V; ++v) mine += kept(l[v], 0);   // (0 for no action)
    });
    const u64 in_wave = wave_sum(mine), total = group_sum<NT>(mine, s, &ahead);
    const u64 target = target_of(o.uniform, total);
    if (target >= ahead && target < ahead + in_wave) {
      MemoryRow<T, 64> run;   // the wave's part of the row
      run.init(memory.logits, memory.invalid, d.actions, memory.chunks);
      run.start = memory.start, run.infinite = memory.infinite;
      const int i = at_sum(run, s1, target - ahead, kept);
      if (lane == 0) write<T>(d, b, w, Result{i, (double)total / w.unit}, action, log_prob);
    }
  } else {
    const float scale = w.scale(BINS);
    // the bin that holds the first cut
    int bound = BINS;
    u64 less = 0;
    if (o.top_k > 0 && o.top_k <= NT) {
      // top_k threads whose largest logits are at or above some logit hold top_k actions there: the histogram of
      // the threads' largest ones gives a bin that is low enough
      clear(s);
      if (own > -INFINITY) count<false>(s, bin_of(top, own, scale, BINS), w, own);
      __syncthreads();
      find(s, 0, (u64)o.top_k);
      bound = s.found;
      if (bound == BINS - 1) bound = BINS;
    }
    if (bound == BINS && o.top_k > 0) {
      clear(s);
      const float none = anew(-INFINITY), scale_ = anew(scale);
      front.chunks(memory, [&](int, const float* l) {
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (l[v] > none) count<false>(s, bin_of(top, l[v], scale_, BINS), w, l[v]);
      });
      __syncthreads();
      find(s, 0, (u64)o.top_k);
      bound = s.found;
      if (bound == BINS - 1 && o.top_p < 1.0)
        less = beyond(s, w, (u64)o.top_k - s.found_before, [&](auto&& f) {
          const float none_ = anew(-INFINITY);
          front.chunks(memory, [&](int, const float* l) {
#pragma unroll
            for (int v = 0; v < V; ++v)
              if (l[v] > none_) f(l[v]);
          });
        });
      if (bound >= BINS - 1) bound = BINS, o.top_k = 0;   // nothing that could be drawn is cut
    }
    if (bound == BINS && o.top_p < 1.0) {
      clear(s);
      const float none = anew(-INFINITY), scale_ = anew(scale);
      front.chunks(memory, [&](int, const float* l) {
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (l[v] > none) count<true>(s, bin_of(top, l[v], scale_, BINS), w, l[v]);
      });
      __syncthreads();
      o.goal = find(s, 0, 0, o.top_p, less);
      bound = s.found;
    }
    // the actions up to that bin, in index order, into the list
    const float least = anew(least_of(top, scale, bound));
    int mine = 0;
    front.chunks(memory, [&](int, const float* l) {
#pragma unroll
      for (int v = 0; v < V; ++v) mine += __popcll(__ballot(l[v] >= least));
    });
    if (lane == 0) counts[wave] = mine;
    __syncthreads();
    int n = 0, at = 0;
    for (int i = 0; i < NW; ++i) {
      if (i == wave) at = n;
      n += counts[i];
    }
    if (bound == BINS || n > LIST) {
      if (threadIdx.x == 0) action[b] = -1;
      return;
    }
    front.chunks(memory, [&](int c, const float* l) {
      u64 has[V], any = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) any |= has[v] = __ballot(l[v] >= least);
      if (any == 0) return;
      int to = at;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        to += __builtin_amdgcn_mbcnt_hi((uint32_t)(has[v] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)has[v], 0));
        at += __popcll(has[v]);
      }
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (l[v] >= least) {
          list[to] = l[v];
          list_at[to++] = memory.index(c, v);
        }
    });
    __syncthreads();
    if (n > FEW) {
      const ListRow<NT> row = {list, list_at, n, (n + NT - 1) / NT};
      const Result r = draw<BINS>(row, s, w, o);
      if (threadIdx.x == 0) write<T>(d, b, w, r, action, log_prob);
      return;
    }
    if (wave > 0) return;
    const Result r = draw_few(list, list_at, n, scratch, w, o);
    if (lane == 0) write<T>(d, b, w, r, action, log_prob);
  }
}

// The rows that k_sample_group left, over the row in memory: a workgroup looks through `per` rows, up to 64.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void k_sample_rest(az_sample_desc d, int32_t* action, float* log_prob, double unit,
                                                    int per) {
  constexpr int V = 16 / sizeof(T), NW = NT / 64;
  __shared__ Shared<NT, BINS> s;
  __shared__ float tops[NW];
  const int64_t first = (int64_t)blockIdx.x * per;
  // (every wave reads the flags of its own accord; a row's is overwritten behind a barrier that all of them passed)
  const int64_t mine = first + (threadIdx.x & 63);
  u64 left = __ballot((int)(threadIdx.x & 63) < per && mine < d.rows && action[mine] == -1);
  __syncthreads();
  for (; left; left &= left - 1) {
    const int b = (int)first + __ffsll(left) - 1;
    double temperature;
    const Options o = options_of(d, b, &temperature);
    MemoryRow<T, NT> memory;
    memory.init((const T*)d.logits + (int64_t)b * d.actions, d.invalid ? d.invalid + (int64_t)b * d.actions : nullptr,
                d.actions, (d.actions + NT * V - 1) / (NT * V));
    float top = -INFINITY;
    each(memory, [&](float l, int) { top = fmaxf(top, l); });
    top = wave_max(top);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int i = 0; i < NW; ++i) top = fmaxf(top, tops[i]);
    if (top == INFINITY) memory.infinite = true, top = 0.0f;
    const Weights w = {top, 1.0 / temperature, unit};
    const Result r = draw<BINS>(memory, s, w, o);
    if (threadIdx.x == 0) write<T>(d, b, w, r, action, log_prob);
    __syncthreads();
  }
}

template <typename T, int CHUNKS>
void launch_group(const az_sample_desc& d, int32_t* action, float* log_prob, double unit, hipStream_t stream) {
  const bool direct = !d.temperature_rows && !d.top_k_rows && !d.top_p_rows && d.temperature > 1e-300 &&
                      (d.top_k <= 0 || d.top_k >= d.actions) && !(d.top_p < 1.0);
  if (direct) {
    k_sample_group<T, 512, CHUNKS, true><<<dim3(d.rows), dim3(512), 0, stream>>>(d, action, log_prob, unit);
  } else {
    // (the rows left are often all or none: a workgroup a row up to 1024, so that all of them share the work; 4096 x
    // 32768 with top_p 0.9 alone 842 us against 988 with eight rows a workgroup at every size)
    const int per = d.rows >= 8192 ? 8 : d.rows >= 1024 ? d.rows / 1024 : 1;
    k_sample_group<T, 512, CHUNKS, false><<<dim3(d.rows), dim3(512), 0, stream>>>(d, action, log_prob, unit);
    k_sample_rest<T, 512><<<dim3((unsigned)az_ceil(d.rows, per)), dim3(512), 0, stream>>>(d, action, log_prob, unit, per);
  }
}

}  // namespace

extern "C" int az_sample_actions(const az_sample_desc* d, int32_t* action, float* log_prob, void* stream_) {
  if (!d) return az_fail(AZ_ERR_INVALID, "sample: null descriptor");
  if (d->dtype < AZ_TYPE_F32 || d->dtype > AZ_TYPE_F16) return az_fail(AZ_ERR_INVALID, "sample: unknown type %d", d->dtype);
  if (d->rows < 0 || d->actions < 1) return az_fail(AZ_ERR_INVALID, "sample: rows=%d actions=%d", d->rows, d->actions);
  if (d->actions > AZ_SAMPLE_MAX_ACTIONS)
    return az_fail(AZ_ERR_UNSUPPORTED, "sample: up to %d actions", AZ_SAMPLE_MAX_ACTIONS);
  if (d->rows == 0) return AZ_OK;
  if (!az_grid_fits(d->rows, d->actions <= 1024 ? 64 : 512))
    return az_fail(AZ_ERR_UNSUPPORTED, "sample: %d rows are too many for one launch", d->rows);
  if (!d->logits || !d->uniform || !action) return az_fail(AZ_ERR_INVALID, "sample: null logits, uniform or action");
  hipStream_t stream = (hipStream_t)stream_;
  // weights of up to one unit each sum up below 2^62, and each is exact in float64
  int bits = 62 - (32 - __builtin_clz((unsigned)d->actions));
  if (bits > 51) bits = 51;
  const double unit = (double)(1ull << bits);
  return az_dispatch_type(d->dtype, [&]<typename T>() -> int {
    constexpr int V = 16 / sizeof(T);
    const int n = d->actions;
    const dim3 rows(d->rows);
    // In microseconds, no cut / top_p 0.9 / top_k 100 too.  A wave a row against a workgroup: 4096 x 300 13 / 16 / 20 against 58 / 83 /
    // 119, 4096 x 1000 27 / 48 / 23 against 69 / 142 / 124, 64 x 1000 15 / 18 / 13 against 10 / 20 / 16.  The row in registers against read
    // again for each pass: 4096 x 32768 246 / 864 / 163 against 279 / 971 / 311, 4096 x 20000 238 / 444 / 167 against 185 / 442 / 232.
    if (n <= 256)
      k_sample_wave<T, 256, 1><<<rows, dim3(64), 0, stream>>>(*d, action, log_prob, unit);
    else if (n <= 512)
      k_sample_wave<T, 512, 1><<<rows, dim3(64), 0, stream>>>(*d, action, log_prob, unit);
    else if (n <= 1024)
      k_sample_wave<T, 1024, 1><<<rows, dim3(64), 0, stream>>>(*d, action, log_prob, unit);
    else if (n <= 512 * 16)
      launch_group<T, 16 / V>(*d, action, log_prob, unit, stream);
    else if (n <= 512 * 32)
      launch_group<T, 32 / V>(*d, action, log_prob, unit, stream);
    else if (n <= 512 * 64)
      launch_group<T, 64 / V>(*d, action, log_prob, unit, stream);
    else
      launch_group<T, 0>(*d, action, log_prob, unit, stream);
    AZ_LAUNCH_CHECK();
    return AZ_OK;
  });
}
