// az_sample.hip -- draws an action a row from truncated policy logits (include/az_layers.h).
// Part of libaz_mcts.so (gfx950 only).
//
// Every truncation keeps a prefix of the row's descending order, so a row's legal actions are cut at one logit, or
// at one index among the actions that share it; no row is sorted.  The cut is found by histograms of counts
// (top_k) or weights (top_p): first over logit / temperature in linear bins, whose bins a row of logits fills
// evenly, then over the order-preserving integer of the logit within the bin that holds the cut, until that bin is a
// single logit.  Weights are summed as 64-bit integers: the order of the LDS atomics does not matter.
// A row is held in the registers of one workgroup (one wave for small action sets); only rows beyond that are read
// again from L2.  float64 exponentials are taken where a weight is needed: of every action for top_p
// alone or without truncation, of the kept actions otherwise.
#include <hip/hip_runtime.h>

#include "az_host.h"
#include "az_types.h"

namespace {

typedef unsigned long long u64;

constexpr double LEAST = 0x1p-40;   // weights below this share of the largest are never drawn

__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l + 0.0f);   // (-0 and +0 are one logit)
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

// A row spread over NT threads: a wave owns a run of chunks, a chunk is 64 x V consecutive actions, V a lane.
template <typename T, int NT, int CHUNKS, bool REGS>
struct Row {
  static constexpr int V = 16 / sizeof(T), NW = NT / 64;
  const T* logits;
  const uint8_t* invalid;
  int actions, chunks, wave, lane, start;   // start: this lane's first action
  float reg[REGS ? CHUNKS : 1][V];
  float infinite;   // 0, or +inf where such logits are present: they become 0, all others -inf

  __device__ void init(const T* l, const uint8_t* inv, int n) {
    logits = l, invalid = inv, actions = n, infinite = 0.0f;
    chunks = REGS ? CHUNKS : (n + NT * V - 1) / (NT * V);
    wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    start = wave * chunks * 64 * V + lane * V;
    if constexpr (REGS)
      for (int c = 0; c < CHUNKS; ++c) fetch(c, reg[c]);
  }
  // the chunk's logits of this lane, -inf where there is no legal action
  __device__ void fetch(int c, float* l) const {
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
      if (infinite > 0.0f) l[v] = l[v] == infinite ? 0.0f : -INFINITY;
    }
  }
  __device__ void only_infinite() {
    infinite = INFINITY;
    if constexpr (REGS)
      for (int c = 0; c < CHUNKS; ++c)
        for (int v = 0; v < V; ++v) reg[c][v] = reg[c][v] == INFINITY ? 0.0f : -INFINITY;
  }
  // f(logit, action) for each legal action of this lane, in index order
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    if constexpr (REGS) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (reg[c][v] > -INFINITY) f(reg[c][v], start + c * 64 * V + v);
    } else {
      for (int c = 0; c < chunks; ++c) {
        float l[V];
        fetch(c, l);
        for (int v = 0; v < V; ++v)
          if (l[v] > -INFINITY) f(l[v], start + c * 64 * V + v);
      }
    }
  }
};

template <int NT, int NB>
struct Shared {
  u64 bins[NB];
  u64 waves[NT / 64];
  u64 before, found_before;
  uint32_t lo, hi;
  int found, index;
  float top[NT / 64];
};

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
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.waves[threadIdx.x >> 6] = x;
  __syncthreads();
  u64 total = 0;
  *ahead = 0;
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
  __device__ explicit Share(double x) {
    int e;
    m = (u64)ldexp(frexp(x, &e), 53);
    shift = x > 0.0 ? 53 - e : 53;
  }
  // n times it, rounded down or up
  __device__ u64 of(u64 n, bool up) const {
    u64 hi = __umul64hi(n, m), lo = n * m;
    if (shift >= 128) return up && (hi | lo) ? 1 : 0;
    if (shift >= 64) {
      const u64 cut = shift == 64 ? 0 : hi & ((1ull << (shift - 64)) - 1);
      return (hi >> (shift - 64)) + (up && (cut | lo) ? 1 : 0);
    }
    return (hi << (64 - shift) | lo >> shift) + (up && (lo & ((1ull << shift) - 1)) ? 1 : 0);
  }
};

template <typename T, int NT, int CHUNKS, bool REGS, int NB>
struct Draw {
  Row<T, NT, CHUNKS, REGS> row;
  Shared<NT, NB>& s;
  float top;
  double inv_t, unit;

  __device__ double weight(float l) const { return exp(((double)l - (double)top) * inv_t); }
  __device__ u64 mass(float l) const { return (u64)(weight(l) * unit + 0.5); }

  // Scans the bins: the first whose inclusive sum, with `before`, reaches the goal is left in s.found (NB: none),
  // the sum ahead of it in s.found_before.  With `share` the goal is that share of the bins' total but `less`.
  __device__ u64 find(u64 before, u64 goal, const Share* share, u64 less) {
    constexpr int PER = NB / NT;
    u64 mine = 0, ahead, h[PER];
    for (int i = 0; i < PER; ++i) mine += h[i] = s.bins[threadIdx.x * PER + i];
    const u64 scan = wave_scan(mine);
    const u64 total = group_sum<NT>(mine, s, &ahead);
    if (threadIdx.x == 0) s.found = NB;
    __syncthreads();
    if (share) {
      goal = share->of(total - less, true);
      if (goal == 0) goal = 1;   // the first one at least
    }
    u64 cum = before + ahead + scan - mine;
    for (int i = 0; i < PER; ++i) {   // exactly one bin crosses
      const u64 next = cum + h[i];
      if (cum < goal && next >= goal) s.found = threadIdx.x * PER + i, s.found_before = cum;
      cum = next;
    }
    __syncthreads();
    return goal;
  }

  // The shortest prefix of the descending order, among logits with a key >= `least`, whose counts (MASS: weights) sum up
  // to the goal; false if there is none (no cut).
  template <bool MASS>
  __device__ bool select(u64 goal, const Share* share, uint32_t least, u64 less, Cut* cut) {
    // linear bins over (top - l) / temperature: 32 of it, the last bin takes what is beyond
    const float scale = (float)fmin(inv_t * (NB / 32), 1e30);
    auto bin_of = [&](float l) { return (int)fminf((top - l) * scale, (float)(NB - 1)); };
    auto add = [&](int bin, float l) {
      if constexpr (MASS)
        atomicAdd(&s.bins[bin], mass(l));
      else
        atomicAdd(reinterpret_cast<uint32_t*>(&s.bins[bin]), 1u);
    };
    auto clear = [&] {
      __syncthreads();
      for (int i = threadIdx.x; i < NB; i += NT) s.bins[i] = 0;
      __syncthreads();
    };
    clear();
    row.each([&](float l, int) {
      if (key_of(l) >= least) add(bin_of(l), l);
    });
    __syncthreads();
    goal = find(0, goal, share, less);
    const int bin = s.found;
    u64 before = s.found_before;
    // (a count that ends in the last bin cuts only weights that are never drawn)
    if (bin == NB || (!MASS && bin == NB - 1)) return false;
    if (threadIdx.x == 0) s.lo = 0xffffffffu, s.hi = 0;
    __syncthreads();
    uint32_t lo = 0xffffffffu, hi = 0;
    row.each([&](float l, int) {
      const uint32_t k = key_of(l);
      if (k >= least && bin_of(l) == bin) lo = min(lo, k), hi = max(hi, k);
    });
    for (int off = 32; off > 0; off >>= 1)
      lo = min(lo, (uint32_t)__shfl_xor(lo, off)), hi = max(hi, (uint32_t)__shfl_xor(hi, off));
    if ((threadIdx.x & 63) == 0 && lo <= hi) atomicMin(&s.lo, lo), atomicMax(&s.hi, hi);
    __syncthreads();
    lo = s.lo, hi = s.hi;
    while (lo < hi) {
      const int bits = 32 - __clz(hi - lo), shift = max(0, bits - (31 - __clz(NB)));
      clear();
      row.each([&](float l, int) {
        const uint32_t k = key_of(l);
        if (k >= lo && k <= hi) add((hi - k) >> shift, l);
      });
      __syncthreads();
      find(before, goal, nullptr, 0);
      // (the sums over these keys are those of the bin that crossed, so one of its bins crosses)
      if (s.found >= NB) break;
      const uint32_t b = s.found;
      before = s.found_before;
      hi -= b << shift;
      const uint32_t width = (1u << shift) - 1;
      lo = hi - lo > width ? hi - width : lo;
      __syncthreads();
    }
    cut->key = lo;
    // the fewest ties that reach the goal
    const u64 w = MASS ? mass(logit_of(lo)) : 1;
    cut->ties = (goal - before + w - 1) / max(w, (u64)1);
    return true;
  }

  __device__ static float logit_of(uint32_t key) {
    return __uint_as_float((key >> 31) ? key ^ 0x80000000u : ~key);
  }

  // The action at which the running sum of `value`, in index order, first exceeds `target` (less than the total).
  template <typename F>
  __device__ int at_sum(u64 target, F&& value) {
    u64 mine = 0, ahead;
    row.each([&](float l, int i) { mine += value(l, i); });
    const u64 in_wave = wave_sum(mine);
    group_sum<NT>(mine, s, &ahead);
    if (target >= ahead && target < ahead + in_wave) {
      // this wave has it: chunk by chunk
      u64 run = ahead;
      int found = -1;
      auto chunk = [&](int c, const float* l) {
        if (found >= 0) return;
        u64 v[Row<T, NT, CHUNKS, REGS>::V], sum = 0;
        for (int j = 0; j < row.V; ++j)
          sum += v[j] = l[j] > -INFINITY ? value(l[j], row.start + c * 64 * row.V + j) : 0;
        const u64 scan = wave_scan(sum);
        const u64 total = (u64)__shfl((uint32_t)(scan >> 32), 63) << 32 | (u64)(uint32_t)__shfl((uint32_t)scan, 63);
        if (target < run + total) {
          const u64 mask = __ballot(target < run + scan);
          const int first = __ffsll((unsigned long long)mask) - 1;
          found = 0;
          if (row.lane == first) {
            u64 cum = run + scan - sum;
            for (int j = 0; j < row.V; ++j) {
              cum += v[j];
              if (target < cum) {
                s.index = row.start + c * 64 * row.V + j;
                break;
              }
            }
          }
        }
        run += total;
      };
      if constexpr (REGS) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) chunk(c, row.reg[c]);
      } else {
        for (int c = 0; c < row.chunks && found < 0; ++c) {
          float l[Row<T, NT, CHUNKS, REGS>::V];
          row.fetch(c, l);
          chunk(c, l);
        }
      }
    }
    __syncthreads();
    return s.index;
  }
};

template <typename T, int NT, int CHUNKS, bool REGS>
__global__ __launch_bounds__(NT) void k_sample(az_sample_desc d, int32_t* action, float* log_prob, double unit) {
  constexpr int NB = NT == 64 ? 256 : NT == 256 ? 1024 : 2048;
  __shared__ Shared<NT, NB> s;
  const int b = blockIdx.x;
  Draw<T, NT, CHUNKS, REGS, NB> w{{}, s};
  w.row.init((const T*)d.logits + (int64_t)b * d.actions, d.invalid ? d.invalid + (int64_t)b * d.actions : nullptr,
             d.actions);
  double temperature = d.temperature_rows ? (double)d.temperature_rows[b] : d.temperature;
  int top_k = d.top_k_rows ? d.top_k_rows[b] : d.top_k;
  double top_p = d.top_p_rows ? (double)d.top_p_rows[b] : d.top_p;
  double min_p = d.min_p_rows ? (double)d.min_p_rows[b] : d.min_p;
  if (!(temperature > 0)) temperature = 1.0, top_k = 1;
  if (top_k <= 0 || top_k >= d.actions) top_k = d.actions;
  const bool nucleus = top_p < 1.0;
  if (!(top_p > 0.0)) top_p = 0.0;
  min_p = min_p > LEAST ? fmin(min_p, 1.0) : LEAST;

  float top = -INFINITY;
  w.row.each([&](float l, int) { top = fmaxf(top, l); });
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  if (w.row.lane == 0) s.top[w.row.wave] = top;
  if (threadIdx.x == 0) s.index = 0;
  __syncthreads();
  for (int i = 0; i < NT / 64; ++i) top = fmaxf(top, s.top[i]);
  if (top == -INFINITY) {   // no legal action
    if (threadIdx.x == 0) {
      action[b] = 0;
      if (log_prob) log_prob[b] = -INFINITY;
    }
    return;
  }
  if (top == INFINITY) w.row.only_infinite(), top = 0.0f;
  w.top = top, w.inv_t = 1.0 / temperature, w.unit = unit;

  Cut cut = {0, ~0ull};
  if (top_k < d.actions) {
    Cut c;
    if (w.template select<false>(top_k, nullptr, 0, 0, &c)) cut = c;
  }
  if (nucleus) {
    u64 less = 0;   // the weight of the ties at the top_k cut that are out
    if (cut.key) {
      const uint32_t key = cut.key;
      u64 ties = 0, ahead;
      w.row.each([&](float l, int) { ties += key_of(l) == key; });
      ties = group_sum<NT>(ties, s, &ahead);
      less = (ties - cut.ties) * w.mass(w.logit_of(key));
    }
    Cut c;
    const Share share(top_p);
    if (w.template select<true>(0, &share, cut.key, less, &c)) {
      if (c.key > cut.key)
        cut = c;
      else if (c.key == cut.key && c.ties < cut.ties)
        cut.ties = c.ties;
    }
  }
  int last_tie = 0x7fffffff;
  if (cut.ties != ~0ull) {
    const uint32_t key = cut.key;
    u64 ties = 0, ahead;
    w.row.each([&](float l, int) { ties += key_of(l) == key; });
    ties = group_sum<NT>(ties, s, &ahead);
    if (cut.ties < ties) last_tie = w.at_sum(cut.ties - 1, [&](float l, int) { return (u64)(key_of(l) == key); });
  }
  auto kept = [&](float l, int i) -> u64 {
    const uint32_t k = key_of(l);
    if (k < cut.key || (k == cut.key && i > last_tie)) return 0;
    const double x = w.weight(l);
    return x >= min_p ? (u64)(x * unit + 0.5) : 0;
  };
  u64 mine = 0, ahead;
  w.row.each([&](float l, int i) { mine += kept(l, i); });
  const u64 total = group_sum<NT>(mine, s, &ahead);
  const float u = d.uniform[b];
  u64 target = u > 0.0f ? total : 0;   // (not a number: 0)
  if (u > 0.0f && u < 1.0f) target = Share((double)u).of(total, false);
  if (target >= total) target = total - 1;
  const int i = w.at_sum(target, kept);
  if (threadIdx.x == 0) {
    action[b] = i;
    if (log_prob) {
      float l = (float)((const T*)d.logits)[(int64_t)b * d.actions + i];
      if (l == INFINITY) l = 0.0f;   // (then top is 0 too)
      log_prob[b] = (float)(((double)l - (double)top) * w.inv_t - log((double)total / unit));
    }
  }
}

template <typename T, int NT, int CHUNKS, bool REGS>
void launch(const az_sample_desc& d, int32_t* action, float* log_prob, hipStream_t stream) {
  // weights of up to one unit each sum up below 2^62, and each is exact in float64
  int bits = 62 - (32 - __builtin_clz((unsigned)d.actions));
  if (bits > 52) bits = 52;
  k_sample<T, NT, CHUNKS, REGS>
      <<<dim3(d.rows), dim3(NT), 0, stream>>>(d, action, log_prob, (double)(1ull << bits));
}

}  // namespace

extern "C" int az_sample_actions(const az_sample_desc* d, int32_t* action, float* log_prob, void* stream_) {
  if (!d) return az_fail(AZ_ERR_INVALID, "sample: null descriptor");
  if (d->dtype < AZ_TYPE_F32 || d->dtype > AZ_TYPE_F16) return az_fail(AZ_ERR_INVALID, "sample: unknown type %d", d->dtype);
  if (d->rows < 0 || d->actions < 1) return az_fail(AZ_ERR_INVALID, "sample: rows=%d actions=%d", d->rows, d->actions);
  if (d->actions > AZ_SAMPLE_MAX_ACTIONS)
    return az_fail(AZ_ERR_UNSUPPORTED, "sample: up to %d actions", AZ_SAMPLE_MAX_ACTIONS);
  if (d->rows == 0) return AZ_OK;
  if (!d->logits || !d->uniform || !action) return az_fail(AZ_ERR_INVALID, "sample: null logits, uniform or action");
  hipStream_t stream = (hipStream_t)stream_;
  return az_dispatch_type(d->dtype, [&]<typename T>() -> int {
    constexpr int V = 16 / sizeof(T);
    const int n = d->actions;
    if (n <= 64 * V)
      launch<T, 64, 1, true>(*d, action, log_prob, stream);
    else if (n <= 64 * 2 * V)
      launch<T, 64, 2, true>(*d, action, log_prob, stream);
    else if (n <= 256 * V * (8 / V))
      launch<T, 256, 8 / V, true>(*d, action, log_prob, stream);
    else if (n <= 1024 * 8)
      launch<T, 1024, 8 / V, true>(*d, action, log_prob, stream);
    else if (n <= 1024 * 16)
      launch<T, 1024, 16 / V, true>(*d, action, log_prob, stream);
    else if (n <= 1024 * 32)
      launch<T, 1024, 32 / V, true>(*d, action, log_prob, stream);
    else
      launch<T, 1024, 1, false>(*d, action, log_prob, stream);
    AZ_LAUNCH_CHECK();
    return AZ_OK;
  });
}
