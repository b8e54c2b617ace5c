// Drawing one token per row of logits from a given random number, for gfx950.
//
//   w_v = exp((z_v - max z) / T);  order: falling logit, equal ones by rising index
//   kept: the first k; of those, the ones whose predecessors weigh less than p times all
//   of them; of those, w >= min_p.  token = the first in vocabulary order whose running sum
//   of kept weights exceeds u times their total; logprob = log(w / total).  T = 0 draws
//   the first maximum.
//
// Every filter keeps a prefix of the order, so a row's kept set is "logits above a
// threshold, and the first m that equal it".  The threshold is found by counting, not by
// sorting: a histogram over bins of log weight (64 octaves below the maximum), then, inside
// the bin that the border falls into, over ranges of the logit's bits until at most
// kCandidates logits are left, which are sorted in LDS.  A token depends on a border of the
// running sum, and the tail's weights are far below fp32's rounding of the sum: weights are
// fp64, sums over bins exact integers of 2^-scale (order-free), the running sum fp64 in a
// fixed order.
//
// One work-group per row.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "timing.h"
#include "../../include/thundersync_hip.h"

namespace ts {
namespace sample {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kGroup = 8;                      // consecutive logits per thread and step
constexpr int kBins = 2048;
constexpr float kBinsPerOctave = 32.f;         // kBins / 64 octaves
constexpr int kCandidates = 4096;              // logits sorted in LDS
constexpr int kMaxVocab = 1 << 21;
constexpr int kTile = kThreads * kGroup;       // logits per step of the work-group
constexpr int kMaxTiles = kMaxVocab / kTile + 1;

struct Options {       // a value for every row, or one per row
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  double temperature_all, top_p_all, min_p_all;
  int64_t top_k_all;
};

struct Args {
  const void* logits;
  int64_t ld;
  int vocab;
  const void* uniform;  // fp32 or fp64
  int uniform_wide;
  Options o;
  double fixed;         // 2^scale: weights as integers
  int64_t* tokens;
  float* logprobs;
};

__device__ __forceinline__ float inf() { return __builtin_huge_valf(); }

// A row in groups of kGroup consecutive logits that start on a 16-byte border: group g holds
// the indices [kGroup g - lead, ...) that lie in the row.
template <typename T> struct Row {
  const T* z;
  int vocab, lead, groups;
  __device__ __forceinline__ Row(const void* base, int64_t ld, int64_t row, int vocab_)
      : z((const T*)base + row * ld), vocab(vocab_) {
    lead = (int)(((uintptr_t)z & 15) / sizeof(T));
    groups = (vocab + lead + kGroup - 1) / kGroup;
  }
  __device__ __forceinline__ int first(int g) const { return g * kGroup - lead; }
  // logits of group g, -inf outside the row
  __device__ __forceinline__ void load(int g, float (&x)[kGroup]) const {
    const int i0 = first(g);
    if (i0 >= 0 && i0 + kGroup <= vocab) {
      load8(z + i0, x);
    } else {
#pragma unroll
      for (int j = 0; j < kGroup; ++j) x[j] = i0 + j >= 0 && i0 + j < vocab ? to_f(z[i0 + j]) : -inf();
    }
    // -0 and 0 are one logit
#pragma unroll
    for (int j = 0; j < kGroup; ++j) x[j] += 0.f;
  }
};

// order-preserving bits of a logit
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// What a row's weights are made of.
struct Weights {
  float top;      // the row's maximum
  double inv_t;   // 1 / T
  float octaves;  // log2(e) / T
  double fixed;
  __device__ __forceinline__ double of(float x) const {
    if (x == top) return 1.;
    return x == -inf() || top == inf() ? 0. : exp(((double)x - (double)top) * inv_t);
  }
  __device__ __forceinline__ uint64_t fixed_of(float x) const { return (uint64_t)(of(x) * fixed + 0.5); }
  // falls with the logit, equal for equal logits
  __device__ __forceinline__ int bin(float x) const {
    if (x == top) return 0;
    const float b = (top - x) * octaves * kBinsPerOctave;
    return b < (float)(kBins - 1) ? (int)b : kBins - 1;
  }
};

// A border in the order: logits above `key` are kept, and the first `ties` (in index order)
// of those that equal it.
struct Border {
  uint32_t key;
  int ties;
};

struct Shared {
  uint32_t count[kBins];
  uint64_t mass[kBins];
  uint64_t cand[kCandidates];
  uint64_t wave_u[kWaves];
  double wave_d[kWaves];
  uint32_t wave_c[kWaves];
  double tile_sum[kMaxTiles];
  uint32_t tile_ties[kMaxTiles];
  int bin, n_cand;
  uint32_t lo, hi;
  uint64_t before_mass;
  uint32_t before_count;
  Border border;
  int token;
  double weight, target;
};

template <typename F> __device__ __forceinline__ void each(int n, F&& f) {
  for (int i = threadIdx.x; i < n; i += kThreads) f(i);
}

// sums in a fixed order: lanes by halving distances, waves in order; every thread gets it
__device__ __forceinline__ double block_sum(double x, Shared& s) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.wave_d[threadIdx.x >> 6] = x;
  __syncthreads();
  double t = s.wave_d[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) t += s.wave_d[w];
  return t;
}
__device__ __forceinline__ uint32_t block_count(uint32_t x, Shared& s) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.wave_c[threadIdx.x >> 6] = x;
  __syncthreads();
  uint32_t t = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) t += s.wave_c[w];
  return t;
}
// exclusive prefix sum over the threads
template <typename V> __device__ __forceinline__ V block_prefix(V x, V* per_wave, V& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  V incl = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V y = __shfl_up(incl, o, 64);
    if (lane >= o) incl += y;
  }
  __syncthreads();
  if (lane == 63) per_wave[wave] = incl;
  __syncthreads();
  V before = (V)0;
  total = (V)0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave) before = total;
    total += per_wave[w];
  }
  // the lanes before this one, as the previous lane's inclusive sum
  const V prev = __shfl_up(incl, 1, 64);
  return lane ? before + prev : before;
}

// Where the running count (BY_MASS false: the first `want` elements) or the running mass
// (the first elements whose predecessors weigh less than `want`) ends, among the logits
// above `limit` and its first ties.
template <typename T, bool BY_MASS>
__device__ void find_border(const Row<T>& row, const Weights& w, uint64_t want, const Border* limit, Shared& s) {
  const uint32_t limit_key = limit ? limit->key : 0;
  const uint32_t limit_ties = limit ? (uint32_t)limit->ties : 0;
  const bool limited = limit != nullptr;
  // the histogram over a range of the order; `range` false: bins of log weight, else of keys in [lo, hi]
  uint32_t lo = 0, hi = 0;
  int shift = 0, bin0 = -1;  // bin0: the log-weight bin that key ranges refine
  bool range = false;
  uint64_t before_mass = 0;
  uint32_t before_count = 0;
  // the part of a logit that counts: 1 above the limit; the limit's own ties are added once
  auto counts = [&](uint32_t k) { return !limited || k > limit_key; };
  auto bin_of = [&](float x, uint32_t k) -> int {
    if (!range) return w.bin(x);
    return k >= lo && k <= hi && w.bin(x) == bin0 ? (int)((hi - k) >> shift) : -1;
  };
  while (true) {
    each(kBins, [&](int b) {
      s.count[b] = 0;
      s.mass[b] = 0;
    });
    __syncthreads();
    for (int g = threadIdx.x; g < row.groups; g += kThreads) {
      float x[kGroup];
      row.load(g, x);
#pragma unroll
      for (int j = 0; j < kGroup; ++j) {
        if (x[j] == -inf()) continue;
        const uint32_t k = key_of(x[j]);
        if (!counts(k)) continue;
        const int b = bin_of(x[j], k);
        if (b < 0) continue;
        atomicAdd(&s.count[b], 1u);
        if (BY_MASS) atomicAdd((unsigned long long*)&s.mass[b], (unsigned long long)w.fixed_of(x[j]));
      }
    }
    if (limited && threadIdx.x == 0) {
      const float x = of_key(limit_key);
      const int b = bin_of(x, limit_key);
      if (b >= 0) {
        atomicAdd(&s.count[b], limit_ties);
        if (BY_MASS) atomicAdd((unsigned long long*)&s.mass[b], (unsigned long long)(limit_ties * w.fixed_of(x)));
      }
    }
    __syncthreads();
    // the first bin in which the wanted amount is reached: two bins a thread
    const int t = threadIdx.x;
    const uint32_t c0 = s.count[2 * t], c1 = s.count[2 * t + 1];
    const uint64_t m0 = s.mass[2 * t], m1 = s.mass[2 * t + 1];
    uint32_t total_c;
    uint64_t total_m;
    const uint32_t pc = block_prefix<uint32_t>(c0 + c1, s.wave_c, total_c) + before_count;
    const uint64_t pm = block_prefix<uint64_t>(m0 + m1, s.wave_u, total_m) + before_mass;
    if (t == 0) {
      s.bin = -1;
      s.lo = 0xffffffffu;
      s.hi = 0;
      s.n_cand = 0;
    }
    __syncthreads();
    // reached in a bin: its end is at or past the wanted amount, its start is not
    auto reached = [&](uint64_t at, uint64_t end, uint32_t n) { return n > 0 && at < want && end >= want; };
    const uint64_t at0 = BY_MASS ? pm : pc, at1 = BY_MASS ? pm + m0 : pc + c0, at2 = BY_MASS ? pm + m0 + m1 : pc + c0 + c1;
    if (reached(at0, at1, c0)) {
      s.bin = 2 * t;
      s.before_mass = pm;
      s.before_count = pc;
    } else if (reached(at1, at2, c1)) {
      s.bin = 2 * t + 1;
      s.before_mass = pm + m0;
      s.before_count = pc + c0;
    }
    __syncthreads();
    if (s.bin < 0) {
      // fewer elements (or less mass) than wanted: everything up to the limit
      if (t == 0) s.border = limited ? *limit : Border{key_of(-inf()), 0};
      __syncthreads();
      return;
    }
    const int b = s.bin;
    const uint32_t n = s.count[b];
    before_mass = s.before_mass;
    before_count = s.before_count;
    if (n <= (uint32_t)kCandidates) {
      // gather the bin's logits, sort them, walk them
      for (int g = threadIdx.x; g < row.groups; g += kThreads) {
        float x[kGroup];
        row.load(g, x);
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
          if (x[j] == -inf()) continue;
          const uint32_t k = key_of(x[j]);
          if (!counts(k) || bin_of(x[j], k) != b) continue;
          s.cand[atomicAdd(&s.n_cand, 1)] = ((uint64_t)k << 32) | (0xffffffffu - (uint32_t)(row.first(g) + j));
        }
      }
      __syncthreads();
      if (limited && bin_of(of_key(limit_key), limit_key) == b) {
        // the limit's ties, the last of the bin: one index is as good as another
        const int at = s.n_cand;
        each((int)limit_ties, [&](int i) { s.cand[at + i] = ((uint64_t)limit_key << 32) | (0xffffffffu - (uint32_t)i); });
        __syncthreads();
        if (t == 0) s.n_cand = at + (int)limit_ties;
        __syncthreads();
      }
      const int have = s.n_cand;
      int size = 64;
      while (size < have) size *= 2;
      each(size - have, [&](int i) { s.cand[have + i] = 0; });
      __syncthreads();
      for (int len = 2; len <= size; len *= 2)
        for (int step = len / 2; step >= 1; step /= 2) {
          each(size / 2, [&](int i) {
            const int p = 2 * step * (i / step) + i % step, q = p + step;
            const uint64_t a = s.cand[p], c = s.cand[q];
            const bool falling = (p & len) == 0;
            if (falling ? a < c : a > c) {
              s.cand[p] = c;
              s.cand[q] = a;
            }
          });
          __syncthreads();
        }
      // the position of the border's element: four candidates a thread, by prefix sums
      constexpr int PER = kCandidates / kThreads;
      uint64_t mine = 0, sum = 0;
      uint64_t part[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int at = PER * t + i;
        part[i] = at < have ? (BY_MASS ? w.fixed_of(of_key((uint32_t)(s.cand[at] >> 32))) : 1) : 0;
        sum += part[i];
      }
      uint64_t total;
      mine = block_prefix<uint64_t>(sum, s.wave_u, total) + (BY_MASS ? before_mass : before_count);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int at = PER * t + i;
        if (at < have && mine < want && mine + part[i] >= want) s.bin = at;  // one element
        mine += part[i];
      }
      __syncthreads();
      // its key and how many of that key's elements come up to it
      const int last = s.bin;
      const uint32_t key = (uint32_t)(s.cand[last] >> 32);
      uint32_t ties = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int at = PER * t + i;
        ties += at <= last && (uint32_t)(s.cand[at] >> 32) == key;
      }
      ties = block_count(ties, s);
      if (t == 0) s.border = Border{key, (int)ties};
      __syncthreads();
      return;
    }
    // too many: the range of keys in the bin
    uint32_t kmin = 0xffffffffu, kmax = 0;
    for (int g = threadIdx.x; g < row.groups; g += kThreads) {
      float x[kGroup];
      row.load(g, x);
#pragma unroll
      for (int j = 0; j < kGroup; ++j) {
        if (x[j] == -inf()) continue;
        const uint32_t k = key_of(x[j]);
        if (!counts(k) || bin_of(x[j], k) != b) continue;
        kmin = min(kmin, k);
        kmax = max(kmax, k);
      }
    }
    if (limited && t == 0 && limit_ties && bin_of(of_key(limit_key), limit_key) == b) {
      kmin = min(kmin, limit_key);
      kmax = max(kmax, limit_key);
    }
    atomicMin(&s.lo, kmin);
    atomicMax(&s.hi, kmax);
    __syncthreads();
    if (!range) bin0 = b;
    lo = s.lo;
    hi = s.hi;
    range = true;
    __syncthreads();
    if (lo == hi) {
      // one logit many times over
      if (t == 0) {
        const uint64_t each_w = w.fixed_of(of_key(lo));
        const uint64_t left = want - (BY_MASS ? before_mass : before_count);
        const uint64_t ties = BY_MASS ? (left + each_w - 1) / each_w : left;
        s.border = Border{lo, (int)ties};
      }
      __syncthreads();
      return;
    }
    shift = 0;
    while (((hi - lo) >> shift) >= (uint32_t)kBins) ++shift;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(Args a) {
  __shared__ Shared s;
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x;
  const Row<T> row(a.logits, a.ld, r, a.vocab);
  const double temp = a.o.temperature ? (double)a.o.temperature[r] : a.o.temperature_all;
  const int64_t top_k = a.o.top_k ? (int64_t)a.o.top_k[r] : a.o.top_k_all;
  const double top_p = a.o.top_p ? (double)a.o.top_p[r] : a.o.top_p_all;
  const double min_p = fmin(a.o.min_p ? (double)a.o.min_p[r] : a.o.min_p_all, 1.);
  const double u = a.uniform_wide ? ((const double*)a.uniform)[r] : (double)((const float*)a.uniform)[r];
  const bool greedy = !(temp > 0.);

  // the maximum and its first index; a NaN shows in its own flag
  float top = -inf();
  int at = 0x7fffffff;
  bool nan = false;
  for (int g = t; g < row.groups; g += kThreads) {
    float x[kGroup];
    row.load(g, x);
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      nan |= x[j] != x[j];
      if (x[j] > top) {
        top = x[j];
        at = row.first(g) + j;
      }
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const float xo = __shfl_xor(top, o, 64);
    const int ao = __shfl_xor(at, o, 64);
    if (xo > top || (xo == top && ao < at)) {
      top = xo;
      at = ao;
    }
  }
  if ((t & 63) == 0) {
    s.wave_d[t >> 6] = (double)top;
    s.wave_c[t >> 6] = (uint32_t)at;
  }
  const bool any_nan = __syncthreads_or(nan);
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float xo = (float)s.wave_d[w];
    const int ao = (int)s.wave_c[w];
    if (xo > top || (xo == top && ao < at)) {
      top = xo;
      at = ao;
    }
  }
  __syncthreads();
  if (any_nan || top == -inf()) {  // nothing to draw
    if (t == 0) {
      a.tokens[r] = -1;
      a.logprobs[r] = __builtin_nanf("");
    }
    return;
  }
  if (greedy || top_k == 1) {
    if (t == 0) {
      a.tokens[r] = at;
      a.logprobs[r] = 0.f;
    }
    return;
  }
  Weights w;
  w.top = top;
  w.inv_t = 1. / temp;
  w.octaves = (float)(1.4426950408889634 / temp);
  w.fixed = a.fixed;

  Border border{key_of(-inf()), 0};
  const bool by_k = top_k > 0 && top_k < a.vocab, by_p = top_p < 1.;
  if (by_k) {
    find_border<T, false>(row, w, (uint64_t)top_k, nullptr, s);
    border = s.border;
  }
  if (by_p) {
    // the mass of what top_k keeps, then the border of p times it
    uint64_t mass = 0;
    for (int g = t; g < row.groups; g += kThreads) {
      float x[kGroup];
      row.load(g, x);
#pragma unroll
      for (int j = 0; j < kGroup; ++j)
        if (x[j] != -inf() && key_of(x[j]) > border.key) mass += w.fixed_of(x[j]);
    }
    uint64_t total;
    block_prefix<uint64_t>(mass, s.wave_u, total);
    if (border.ties) total += border.ties * w.fixed_of(of_key(border.key));
    // the smallest whole mass that is p times the total or more; at least the first element
    const double goal = ceil(top_p * (double)total);
    const uint64_t want = goal > 1. ? (uint64_t)goal : 1;
    const Border limit = border;
    find_border<T, true>(row, w, want, by_k ? &limit : nullptr, s);
    border = s.border;
  }
  // a partial tie only matters where not all of the logits that equal the border's are kept;
  // counting them in index order covers both
  const float border_x = of_key(border.key);
  auto above = [&](float x) { return x != -inf() && key_of(x) > border.key; };
  const double tie_weight = border.ties ? w.of(border_x) : 0.;
  const bool tie_kept = border.ties && (tie_weight >= min_p);
  auto weight = [&](float x) {
    const double y = w.of(x);  // 1 for the maximum, which min_p never drops
    return y >= min_p ? y : 0.;
  };
  // kept mass and ties per tile of kTile logits
  const int tiles = (row.groups + kThreads - 1) / kThreads;
  for (int i = 0; i < tiles; ++i) {
    const int g = i * kThreads + t;
    double m = 0.;
    uint32_t ties = 0;
    if (g < row.groups) {
      float x[kGroup];
      row.load(g, x);
#pragma unroll
      for (int j = 0; j < kGroup; ++j) {
        if (above(x[j])) m += weight(x[j]);
        else if (tie_kept && x[j] == border_x) ++ties;
      }
    }
    m = block_sum(m, s);
    if (tie_kept) ties = block_count(ties, s);
    if (t == 0) {
      s.tile_sum[i] = m;
      s.tile_ties[i] = ties;
    }
  }
  __syncthreads();
  // the tile that the draw falls into
  if (t == 0) {
    double total = 0.;
    uint32_t left = tie_kept ? (uint32_t)border.ties : 0;
    for (int i = 0; i < tiles; ++i) {
      const uint32_t n = min(left, s.tile_ties[i]);
      s.tile_ties[i] = n;
      left -= n;
      s.tile_sum[i] += n * tie_weight;
      total += s.tile_sum[i];
    }
    const double target = u * total;
    double before = 0.;
    int pick = -1, last = 0;
    for (int i = 0; i < tiles && pick < 0; ++i) {
      if (s.tile_sum[i] > 0.) last = i;
      if (before + s.tile_sum[i] > target) pick = i;
      else before += s.tile_sum[i];
    }
    if (pick < 0) {  // u of 1 or more, or NaN: the last one
      pick = last;
      before = -__builtin_huge_val();
    }
    s.bin = pick;
    s.target = target - before;  // infinite: the last kept logit of the tile
    s.weight = total;
    s.token = -1;
    s.n_cand = -1;
  }
  __syncthreads();
  {
    const int g = s.bin * kThreads + t;
    float x[kGroup];
    double y[kGroup];
    double sum = 0.;
    uint32_t ties = 0;
    if (g < row.groups) row.load(g, x);
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      if (g >= row.groups) x[j] = -inf();
      y[j] = above(x[j]) ? weight(x[j]) : 0.;
      ties += tie_kept && x[j] == border_x;
    }
    uint32_t all_ties, tie = block_prefix<uint32_t>(ties, s.wave_c, all_ties);
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      if (tie_kept && x[j] == border_x) {
        if (tie < s.tile_ties[s.bin]) y[j] = tie_weight;
        ++tie;
      }
      sum += y[j];
    }
    double total;
    double run = block_prefix<double>(sum, s.wave_d, total);
    const double target = s.target;
    int hit = -1, last = -1;
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      run += y[j];
      if (y[j] > 0.) {
        last = j;
        if (hit < 0 && run > target) hit = j;
      }
    }
    // the first hit of the work-group, or (by rounding) the tile's last kept logit
    const int i0 = row.first(g);
    if (t == 0) s.token = 0x7fffffff;
    __syncthreads();
    if (hit >= 0) atomicMin(&s.token, i0 + hit);
    if (last >= 0) atomicMax(&s.n_cand, i0 + last);
    __syncthreads();
    if (t == 0) {
      const int token = s.token != 0x7fffffff ? s.token : s.n_cand;
      a.tokens[r] = token;
      a.logprobs[r] = (float)log(w.of(to_f(row.z[token]) + 0.f) / s.weight);
    }
  }
}

}  // namespace sample
}  // namespace ts

extern "C" {

int ts_sample(const void* logits, int64_t ld_logits, int64_t rows, int64_t vocab, const void* uniform,
              int uniform_dtype, const float* temperature, double temperature_all, const int32_t* top_k,
              int64_t top_k_all, const float* top_p, double top_p_all, const float* min_p, double min_p_all,
              int64_t* tokens, float* logprobs, int dtype, void* stream) {
  using namespace ts::sample;
  TS_CHECK_ARG(dtype == TS_F32 || dtype == TS_F16 || dtype == TS_BF16, "ts_sample: dtype %d", dtype);
  TS_CHECK_ARG(uniform_dtype == TS_F32 || uniform_dtype == TS_F64, "ts_sample: uniform dtype %d", uniform_dtype);
  TS_CHECK_ARG(rows >= 0 && rows < (1ll << 31) && vocab >= 1 && vocab <= kMaxVocab && ld_logits >= 0,
               "ts_sample: bad shape rows=%lld vocab=%lld (1 .. %d)", (long long)rows, (long long)vocab, kMaxVocab);
  TS_CHECK_ARG((temperature || temperature_all >= 0) && (top_k || top_k_all >= 0) && (top_p || top_p_all >= 0) &&
                   (min_p || min_p_all >= 0),
               "ts_sample: an option is negative or NaN");
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(logits && uniform && tokens && logprobs, "ts_sample: null pointer");
  Args a;
  a.logits = logits;
  a.ld = ld_logits;
  a.vocab = (int)vocab;
  a.uniform = uniform;
  a.uniform_wide = uniform_dtype == TS_F64;
  a.o = Options{temperature, top_k, top_p, min_p, temperature_all, top_p_all, min_p_all, top_k_all};
  int bits = 0;
  while ((1ll << bits) < vocab) ++bits;
  a.fixed = (double)(1ull << (62 - bits));  // vocab weights of at most 1 stay below 2^62
  a.tokens = tokens;
  a.logprobs = logprobs;
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("sampling.sample_kernel", s);
    const dim3 grid((unsigned)rows), block(kThreads);
    if (dtype == TS_F32) hipLaunchKernelGGL(sample_kernel<float>, grid, block, 0, s, a);
    else if (dtype == TS_F16) hipLaunchKernelGGL(sample_kernel<ts::f16>, grid, block, 0, s, a);
    else hipLaunchKernelGGL(sample_kernel<ts::bf16>, grid, block, 0, s, a);
  }
  return ts::check_launch("ts_sample");
}

}  // extern "C"
