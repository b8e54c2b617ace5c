// Drawing one token per row of logits from a given random number, for gfx950.
//
//   w_v = exp((z_v - max z) / T);  order: falling logit, equal ones by rising index
//   kept: the first k; of those, the ones whose predecessors weigh less than p times all
//   of them; of those, w >= min_p.  token = the first in vocabulary order whose running sum
//   of kept weights exceeds u times their total; logprob = log(w / total).  T = 0 draws
//   the first maximum.
//
// Every filter keeps a prefix of the order, so a row's kept set is "logits above a border
// element, and those that equal it up to its index".  The border is found by counting, not
// by sorting the row.  A row is cut into slices of kSlice logits, and up to five launches of
// work-groups over (rows x slices) work on it:
//   maxima   each slice's maximum, minimum, NaN; without filters also its sum of weights
//   bins     a histogram (count and mass) of the row over kBins bins of logit below its maximum
//   search   the bins that the borders fall into
//   gather   their logits as candidates; per slice the sum of the weights above them
//   draw     one work-group a row: sorts the candidates in LDS, finds the border, picks the
//            slice that u falls into and reads that slice again for the token
// A row with more than kCandidates logits in its border bins (equal logits, or very many in a
// narrow range) is resolved by its draw work-group alone, which narrows the range bin by bin.
//
// A token depends on a border of the running sum, and the tail's weights are far below fp32's
// rounding of the sum: weights are fp64, sums over bins exact integers of 2^-scale (order-free),
// the running sum fp64 in a fixed order.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "timing.h"
#include "../../include/thundersync_hip.h"

namespace ts {
namespace sample {

constexpr int kMaxThreads = 256;                // maxima
constexpr int kThreads = 512;                  // bins and gather: few work-groups a row, each pays the histogram
constexpr int kDrawThreads = 512;              // draw
constexpr int kGroup = 8;                      // consecutive logits per thread and step
constexpr int kBins = 2048;
constexpr float kBinsPerOctave = 32.f;         // kBins / 64 octaves
constexpr int kCandidates = 4096;              // logits sorted in LDS
constexpr int kMaxVocab = 1 << 21;
constexpr int kSliceGroups = 1024, kSlice = kSliceGroups * kGroup;  // logits per slice
constexpr int kMaxSlices = kMaxVocab / kSlice + 1;

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
  // logits of group g, -inf outside the row; -0 and 0 are one logit
  __device__ __forceinline__ void load(int g, float (&x)[kGroup]) const {
    load_raw(g, x);
#pragma unroll
    for (int j = 0; j < kGroup; ++j) x[j] += 0.f;
  }
  // the same without the zeros' care: for sums and maxima
  __device__ __forceinline__ void load_raw(int g, float (&x)[kGroup]) const {
    const int i0 = first(g);
    if (i0 >= 0 && i0 + kGroup <= vocab) {
      load8(z + i0, x);
    } else {
#pragma unroll
      for (int j = 0; j < kGroup; ++j) x[j] = i0 + j >= 0 && i0 + j < vocab ? to_f(z[i0 + j]) : -inf();
    }
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

// 2^(j / kTable) for j in [0, kTable), worked out by the compiler: the exponential's series
// of j ln 2 / kTable, whose terms fall below 2^-60 by the 20th, summed from the smallest
constexpr int kTable = 256;
struct Table {
  double at[kTable];
  constexpr Table() : at{} {
    for (int j = 0; j < kTable; ++j) {
      const double x = 0.693147180559945309417 * j / kTable;
      double s = 1.;
      for (int k = 20; k >= 1; --k) s = 1. + s * x / k;
      at[j] = s;
    }
  }
};
__constant__ const Table kPowers = Table();
__device__ __forceinline__ void fill_table(double* table) {
  for (int j = threadIdx.x; j < kTable; j += blockDim.x) table[j] = kPowers.at[j];
  __syncthreads();
}

// What a row's weights are made of.  exp((x - top) / T) = 2^(k / 256) 2^(r / 256) with k whole
// and |r| <= 1/2: the first from the table and an exponent, the second by its Taylor series to
// the fourth power (the next term is below 2^-54).  k is rounded by adding 1.5 2^52, whose low
// word then holds it, and the exponent is added to the high word: conversions, rounding and
// ldexp of fp64 run at a quarter of the rate of these.
struct Weights {
  const double* table;
  double top;     // the maximum that weights are relative to
  double units;   // kTable log2(e) / T
  double fixed;
  float top_f;
  float bins;     // bins per unit of logit
  // 2^(max(y, -1000 kTable) / kTable), for y of 0 or less; NaN counts as the least
  __device__ __forceinline__ double power(double y) const {
    constexpr double kRound = 6755399441055744., kL = 0.693147180559945309417 / kTable;
    y = fmax(y, -1000. * kTable);
    const double k = y + kRound;
    const double t = y - (k - kRound);
    const double e = fma(fma(fma(fma(t, kL * kL * kL * kL / 24, kL * kL * kL / 6), t, kL * kL / 2), t, kL), t, 1.);
    const int n = __double2loint(k);
    const double p = table[n & (kTable - 1)] * e;
    return __hiloint2double(__double2hiint(p) + ((n & -kTable) << 12), __double2loint(p));
  }
  // a logit's weight, 0 where it is more than 1000 octaves below the maximum (or -inf, or below an infinite one)
  __device__ __forceinline__ double of(float x) const {
    const double y = ((double)x - top) * units, p = power(fmin(y, 0.));
    return y < -1000. * kTable ? 0. : p;
  }
  // the same with 2^-1000 for 0, which adds nothing to a sum that holds the maximum's 1 and no whole number
  __device__ __forceinline__ double of_any(float x) const { return power(fmin(((double)x - top) * units, 0.)); }
  // and where the maximum is finite
  __device__ __forceinline__ double of_finite(float x) const { return power(((double)x - top) * units); }
  // a weight as a whole number of 1 / fixed (at most 2^50), by an addition whose rounding leaves it in the low bits
  __device__ __forceinline__ uint64_t whole(double weight) const {
    const double y = fma(weight, fixed, 4503599627370496.);
    return ((uint64_t)(__double2hiint(y) & 0xfffff) << 32) | (uint32_t)__double2loint(y);
  }
  __device__ __forceinline__ uint64_t fixed_of(float x) const { return whole(of_any(x)); }
  // falls with the logit, equal for equal logits
  __device__ __forceinline__ int bin(float x) const {
    const int b = (int)fminf((top_f - x) * bins, (float)(kBins - 1));
    return x == top_f ? 0 : b;
  }
};
// `low`: the row's lowest finite logit, so that the bins cover no more than there is
__device__ __forceinline__ Weights weights_of(const double* table, float top, float low, double temp, double fixed) {
  Weights w;
  w.table = table;
  // an infinite maximum: above every finite logit, and at its equals (whose difference is clamped to 0)
  w.top = top < inf() ? (double)top : 1e300;
  w.top_f = top;
  // a T so small or so large that nothing, or everything, is the maximum's equal keeps finite products,
  // and one so large still has every finite logit 1000 octaves below an infinite one's 1e300
  w.units = fmin(fmax(kTable * (1.4426950408889634074 / temp), 1e-290), 1e300);
  w.fixed = fixed;
  const float octave = (float)(0.693147180559945309 * temp);  // in units of logit
  w.bins = fminf(fmaxf(kBinsPerOctave / octave, (float)kBins / (top - low)), 1e30f);
  return w;
}

// A border in the order: logits above `key` are kept, and the first `ties` (in index order)
// of those that equal it.
struct Border {
  uint32_t key;
  int ties;
};

// What a work-group of N threads that draws a row's token holds.
template <int N> struct Scratch {
  union {
    uint64_t cand[kCandidates];
    struct {  // find_border's, before it gathers candidates
      uint64_t mass[kBins];
      uint32_t count[kBins];
    };
  };
  double slice_sum[kMaxSlices];
  uint64_t slice_add[kMaxSlices];  // candidates' kept mass, or (slow rows) ties
  double table[kTable];
  uint64_t wave_u[N / 64];
  double wave_d[N / 64];
  uint32_t wave_c[N / 64];
  int bin, n_cand, token;
  double total, target, scale;
  uint32_t lo, hi, before_count;
  uint64_t before_mass;
  Border border;
};

template <int N, typename F> __device__ __forceinline__ void each(int n, F&& f) {
  for (int i = threadIdx.x; i < n; i += N) f(i);
}

// sums in a fixed order: lanes by halving distances, waves in order; every thread gets it
template <int N, typename V> __device__ __forceinline__ V block_sum(V x, V* per_wave) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) per_wave[threadIdx.x >> 6] = x;
  __syncthreads();
  V t = per_wave[0];
#pragma unroll
  for (int w = 1; w < N / 64; ++w) t += per_wave[w];
  return t;
}
// exclusive prefix sum over the threads
template <int N, typename V> __device__ __forceinline__ V block_prefix(V x, V* per_wave, V& total) {
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
  for (int w = 0; w < N / 64; ++w) {
    if (w == wave) before = total;
    total += per_wave[w];
  }
  // the lanes before this one, as the previous lane's inclusive sum
  const V prev = __shfl_up(incl, 1, 64);
  return lane ? before + prev : before;
}

// s.cand[0 .. have) (all different) into falling order.  Few: each one's place is the number of
// larger ones, counted by a thread that reads them all (480 in 256 threads: one step of 2 x 480
// comparisons against 45 steps of the sorting network, each with its barrier).  Many: the
// network, over a power of two padded with zeros.
constexpr int kCounted = 1024;
template <int N> __device__ __forceinline__ void sort_candidates(Scratch<N>& s, int have) {
  if (have <= kCounted) {
    constexpr int PER = kCounted / N;
    uint64_t mine[PER];
    int place[PER] = {};
#pragma unroll
    for (int i = 0; i < PER; ++i) mine[i] = (int)threadIdx.x + N * i < have ? s.cand[threadIdx.x + N * i] : 0;
    if (threadIdx.x == 0 && (have & 1)) s.cand[have] = 0;  // read in pairs; counts for nothing
    __syncthreads();
    auto count = [&](auto used) {
#pragma unroll 8
      for (int j = 0; j < have; j += 2) {
        const uint64_t a = s.cand[j], c = s.cand[j + 1];
#pragma unroll
        for (int i = 0; i < decltype(used)::value; ++i) place[i] += (a > mine[i]) + (c > mine[i]);
      }
    };
    if (have <= N) count(std::integral_constant<int, 1>{});
    else count(std::integral_constant<int, PER>{});
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if ((int)threadIdx.x + N * i < have) s.cand[place[i]] = mine[i];
    __syncthreads();
    return;
  }
  int size = 64;
  while (size < have) size *= 2;
  each<N>(size - have, [&](int i) { s.cand[have + i] = 0; });
  __syncthreads();
  for (int len = 2; len <= size; len *= 2)
    for (int step = len / 2; step >= 1; step /= 2) {
      each<N>(size / 2, [&](int i) {
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
}

// Where the running count (BY_MASS false: the first `want` elements) or the running mass
// (the first elements whose predecessors weigh less than `want`) ends, among the logits
// above `limit` and its first ties.
template <typename T, int N, bool BY_MASS>
__device__ __forceinline__ void find_border(const Row<T>& row, const Weights& w, uint64_t want, const Border* limit, Scratch<N>& s) {
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
    each<N>(kBins, [&](int b) {
      s.count[b] = 0;
      s.mass[b] = 0;
    });
    __syncthreads();
    for (int g = threadIdx.x; g < row.groups; g += N) {
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
    // the first bin in which the wanted amount is reached: consecutive bins a thread
    constexpr int BINS = kBins / N;
    const int t = threadIdx.x;
    uint32_t c = 0, total_c;
    uint64_t m = 0, total_m;
    for (int i = 0; i < BINS; ++i) {
      c += s.count[BINS * t + i];
      m += s.mass[BINS * t + i];
    }
    c = block_prefix<N, uint32_t>(c, s.wave_c, total_c) + before_count;
    m = block_prefix<N, uint64_t>(m, s.wave_u, total_m) + before_mass;
    if (t == 0) {
      s.bin = -1;
      s.lo = 0xffffffffu;
      s.hi = 0;
      s.n_cand = 0;
    }
    __syncthreads();
    for (int i = 0; i < BINS; ++i) {
      const uint32_t cb = s.count[BINS * t + i];
      const uint64_t mb = s.mass[BINS * t + i];
      // reached in this bin: its end is at or past the wanted amount, its start is not
      const uint64_t at = BY_MASS ? m : c, end = BY_MASS ? m + mb : c + cb;
      if (cb > 0 && at < want && end >= want) {
        s.bin = BINS * t + i;
        s.before_mass = m;
        s.before_count = c;
      }
      c += cb;
      m += mb;
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
    __syncthreads();  // the candidates take the histogram's place
    if (n <= (uint32_t)kCandidates) {
      // gather the bin's logits, sort them, walk them
      for (int g = threadIdx.x; g < row.groups; g += N) {
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
        each<N>((int)limit_ties, [&](int i) { s.cand[at + i] = ((uint64_t)limit_key << 32) | (0xffffffffu - (uint32_t)i); });
        __syncthreads();
        if (t == 0) s.n_cand = at + (int)limit_ties;
        __syncthreads();
      }
      const int have = s.n_cand;
      sort_candidates<N>(s, have);
      // the position of the border's element: consecutive candidates a thread, by prefix sums
      const int per = (have + N - 1) / N, first = min(have, per * t), end = min(have, first + per);
      auto part = [&](int i) { return BY_MASS ? w.fixed_of(of_key((uint32_t)(s.cand[i] >> 32))) : (uint64_t)1; };
      uint64_t mine = 0, total;
      for (int i = first; i < end; ++i) mine += part(i);
      mine = block_prefix<N, uint64_t>(mine, s.wave_u, total) + (BY_MASS ? before_mass : before_count);
      for (int i = first; i < end; ++i) {
        const uint64_t next = mine + part(i);
        if (mine < want && next >= want) s.bin = i;  // one element
        mine = next;
      }
      __syncthreads();
      // its key and how many of that key's elements come up to it
      const int last = s.bin;
      const uint32_t key = (uint32_t)(s.cand[last] >> 32);
      uint32_t ties = 0;
      for (int i = first; i < min(end, last + 1); ++i) ties += (uint32_t)(s.cand[i] >> 32) == key;
      ties = block_sum<N, uint32_t>(ties, s.wave_c);
      if (t == 0) s.border = Border{key, (int)ties};
      __syncthreads();
      return;
    }
    // too many: the range of keys in the bin
    uint32_t kmin = 0xffffffffu, kmax = 0;
    for (int g = threadIdx.x; g < row.groups; g += N) {
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

// ---------------------------------------------------------------------------
// a row's options and what the launches hand on
// ---------------------------------------------------------------------------
struct RowOptions {
  double temp, top_p, min_p, u;
  int64_t top_k;
  bool greedy, by_k, by_p, by_min;
  __device__ __forceinline__ RowOptions(const Args& a, int64_t r) {
    temp = a.o.temperature ? (double)a.o.temperature[r] : a.o.temperature_all;
    top_k = a.o.top_k ? (int64_t)a.o.top_k[r] : a.o.top_k_all;
    top_p = a.o.top_p ? (double)a.o.top_p[r] : a.o.top_p_all;
    min_p = a.o.min_p ? (double)a.o.min_p[r] : a.o.min_p_all;
    min_p = min_p > 0. ? fmin(min_p, 1.) : 0.;  // NaN: none
    u = a.uniform_wide ? ((const double*)a.uniform)[r] : (double)((const float*)a.uniform)[r];
    u = u < 0. ? 0. : u;
    greedy = !(temp > 0.) || top_k == 1;
    by_k = !greedy && top_k > 0 && top_k < a.vocab;
    by_p = !greedy && top_p < 1.;
    by_min = !greedy && min_p > 0.;
  }
  __device__ __forceinline__ bool plain() const { return !greedy && !by_k && !by_p && !by_min; }
};

constexpr int kSums = kThreads / 64;
constexpr int kBinParts = 8;  // work-groups a row for its histogram, at most

struct SliceStats {
  float top, low;  // -inf / +inf: no logit above -inf
  int at;          // first index of the maximum
  int nan;
};

// Per row: the bins that hold the borders.
struct Bins {
  int lo, hi, k;          // border of p in [lo, hi], of k in k (or lo = hi = k, or none: kBins)
  uint32_t k_before;      // elements above bin k
  uint64_t k_mass, lo_mass;  // mass above bins k and lo
  uint64_t all_mass;
};

// The launches' workspace, of `rows` rows, `slices` slices and `parts` shares of a row's
// histogram.  From `bins` on only where some row of the call has a top_k or top_p: null otherwise.
struct Space {
  SliceStats* stats;  // [rows][slices]
  double* sums;       // [rows][slices][kSums]: of a slice's waves (without filters the first alone)
  Bins* bins;         // [rows]
  uint64_t* mass;     // [rows][parts][kBins]
  uint32_t* count;    // [rows][parts][kBins]
  uint64_t* cand;     // [rows][kCandidates]
  uint32_t* n_cand;   // [rows]
  int slices, parts;
};

// the row's maximum, lowest logit and NaN from its slices (every thread reads them all: few)
struct RowStats {
  float top, low;
  int at;
  bool nan;
  __device__ __forceinline__ RowStats(const SliceStats* s, int slices) {
    top = -inf();
    low = inf();
    at = 0x7fffffff;
    int any = 0;
    const int lane = threadIdx.x & 63;
    for (int i = lane; i < slices; i += 64) {
      const SliceStats x = s[i];
      any |= x.nan;
      low = fminf(low, x.low);
      if (x.top > top) {  // slices in index order: the first of equal ones
        top = x.top;
        at = x.at;
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
      low = fminf(low, __shfl_xor(low, o, 64));
      any |= __shfl_xor(any, o, 64);
    }
    nan = any != 0;
  }
  __device__ __forceinline__ bool empty() const { return nan || top == -inf(); }
};

// ---------------------------------------------------------------------------
// maxima: one slice, held in registers; a row without filters gets its slice's sum of
// weights, relative to the slice's own maximum, from the same read.  With filters bound by the
// launch and the read (64 rows of 151936 fp32 logits: 9 us, 4.4 TB/s), without by the fp64
// weights' instructions (512 bf16 rows of 151936: 69 us, 2.3 TB/s; the read alone is 30 at a copy's rate).
// ---------------------------------------------------------------------------
template <typename T, bool BINS>
__global__ __launch_bounds__(kMaxThreads, 5) void maxima_kernel(Args a, Space sp) {
  constexpr int N = kMaxThreads, WAVES = N / 64, GROUPS = kSliceGroups / N;
  __shared__ double table[kTable], per_wave[WAVES];
  __shared__ float tops[WAVES], lows[WAVES];
  __shared__ int ats[WAVES];
  const int64_t r = blockIdx.y;
  const int slice = blockIdx.x, t = threadIdx.x;
  if (BINS && slice == 0 && t == 0) sp.n_cand[r] = 0;
  const RowOptions o(a, r);
  const Row<T> row(a.logits, a.ld, r, a.vocab);
  float x[GROUPS][kGroup];
  float top = -inf(), low = inf();
  bool nan = false;
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const int g = slice * kSliceGroups + i * N + t;
    if (g < row.groups) {
      row.load_raw(g, x[i]);
    } else {
#pragma unroll
      for (int j = 0; j < kGroup; ++j) x[i][j] = -inf();
    }
  }
#pragma unroll
  for (int i = 0; i < GROUPS; ++i)
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      nan |= x[i][j] != x[i][j];
      top = fmaxf(top, x[i][j]);
    }
  if (BINS) {  // the bins' range
#pragma unroll
    for (int i = 0; i < GROUPS; ++i)
#pragma unroll
      for (int j = 0; j < kGroup; ++j) low = fminf(low, x[i][j] == -inf() ? inf() : x[i][j]);
  }
  int at = 0x7fffffff;
  if (o.greedy) {  // the first index of the thread's maximum
#pragma unroll
    for (int i = GROUPS - 1; i >= 0; --i)
#pragma unroll
      for (int j = kGroup - 1; j >= 0; --j)
        if (x[i][j] == top) at = row.first(slice * kSliceGroups + i * N + t) + j;
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    const float xo = __shfl_xor(top, d, 64);
    const int ao = __shfl_xor(at, d, 64);
    if (xo > top || (xo == top && ao < at)) {
      top = xo;
      at = ao;
    }
    low = fminf(low, __shfl_xor(low, d, 64));
  }
  if ((t & 63) == 0) {
    tops[t >> 6] = top;
    lows[t >> 6] = low;
    ats[t >> 6] = at;
  }
  const bool any = __syncthreads_or(nan);
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (tops[w] > top || (tops[w] == top && ats[w] < at)) {
      top = tops[w];
      at = ats[w];
    }
    low = fminf(low, lows[w]);
  }
  if (t == 0) sp.stats[r * sp.slices + slice] = SliceStats{top, low, at, any};
  if (!o.plain()) return;
  if (any || top == -inf()) {
    if (t == 0) sp.sums[(r * sp.slices + slice) * kSums] = 0.;
    return;
  }
  fill_table(table);
  const Weights w = weights_of(table, top, low, o.temp, a.fixed);
  double sum = 0.;
  if (top < inf()) {
#pragma unroll
    for (int i = 0; i < GROUPS; ++i)
#pragma unroll
      for (int j = 0; j < kGroup; ++j) sum += w.of_finite(x[i][j]);
  } else {
#pragma unroll
    for (int i = 0; i < GROUPS; ++i)
#pragma unroll
      for (int j = 0; j < kGroup; ++j) sum += x[i][j] == inf() ? 1. : 0.;
  }
  sum = block_sum<N, double>(sum, per_wave);
  if (t == 0) sp.sums[(r * sp.slices + slice) * kSums] = sum;
}

// ---------------------------------------------------------------------------
// bins: a work-group's share of the row into a histogram of its own, counts where top_k
// asks for them and mass where top_p does.  (Shares added to one histogram by atomics, or added
// up by every gather work-group, cost as much as the logits; a last work-group that adds them
// waits for the XCDs' caches to be written back.)  Bound by the weights' instructions and
// the histogram's LDS atomics (bank conflicts 14 % of the LDS cycles): 17 us at 64 rows of 151936
// with top_p, 38 at 333 of 50257 with every option.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kThreads) void bins_kernel(Args a, Space sp) {
  __shared__ double table[kTable];
  __shared__ uint32_t count[kBins];
  __shared__ uint64_t mass[kBins];
  const int64_t r = blockIdx.y;
  const int t = threadIdx.x;
  const RowOptions o(a, r);
  if (!o.by_k && !o.by_p) return;
  const RowStats s(sp.stats + r * sp.slices, sp.slices);
  if (s.empty()) return;
  for (int i = t; i < kBins; i += kThreads) {
    count[i] = 0;
    mass[i] = 0;
  }
  fill_table(table);
  const Weights w = weights_of(table, s.top, s.low, o.temp, a.fixed);
  const Row<T> row(a.logits, a.ld, r, a.vocab);
  // no branch in a group's eight, so that their chains overlap: -inf falls into the last bin with nothing
  for (int g = blockIdx.x * kThreads + t; g < row.groups; g += gridDim.x * kThreads) {
    float x[kGroup];
    row.load_raw(g, x);
    int b[kGroup];
#pragma unroll
    for (int j = 0; j < kGroup; ++j) b[j] = w.bin(x[j]);
    if (o.by_k) {
#pragma unroll
      for (int j = 0; j < kGroup; ++j) atomicAdd(&count[b[j]], x[j] == -inf() ? 0u : 1u);
    }
    if (o.by_p) {
      uint64_t m[kGroup];
#pragma unroll
      for (int j = 0; j < kGroup; ++j) m[j] = w.fixed_of(x[j]);
#pragma unroll
      for (int j = 0; j < kGroup; ++j) atomicAdd((unsigned long long*)&mass[b[j]], (unsigned long long)m[j]);
    }
  }
  __syncthreads();
  const int64_t base = (r * sp.parts + blockIdx.x) * kBins;
  for (int i = t; i < kBins; i += kThreads) {
    if (o.by_k) sp.count[base + i] = count[i];
    if (o.by_p) sp.mass[base + i] = mass[i];
  }
}

// ---------------------------------------------------------------------------
// search: the border bins from a row's shares of the histogram, consecutive bins a thread.
// A launch of its own, or for few rows the beginning of every gather work-group: a launch less
// (one row: gather and search 8.5 + 12.5 -> 15.9 us, the pass 47 -> 45), where over many rows the
// shares read again by each cost more (64 rows: gather 27 -> 42 us against a search of 9.6).
// ---------------------------------------------------------------------------
constexpr int kFewRows = 4;
__device__ __forceinline__ void search_bins(const Space& sp, int64_t r, const RowOptions& o, Bins& found) {
  __shared__ uint64_t wave_m[kThreads / 64];
  __shared__ uint32_t wave_c[kThreads / 64];
  __shared__ uint64_t bin_mass;  // of bin k
  constexpr int PER = kBins / kThreads;
  const int t = threadIdx.x;
  const int parts = sp.parts;
  const uint32_t* count = sp.count + r * parts * kBins;
  const uint64_t* mass = sp.mass + r * parts * kBins;
  if (t == 0) found = Bins{kBins, kBins, kBins, 0, 0, 0, 0};
  uint32_t c[PER] = {}, cs = 0;
  uint64_t m[PER] = {}, ms = 0;
  // all loads before the first use: other XCDs wrote them
  uint32_t cp[kBinParts][PER] = {};
  uint64_t mp[kBinParts][PER] = {};
#pragma unroll
  for (int part = 0; part < kBinParts; ++part) {
    if (part < parts) {
      const int base = part * kBins + PER * t;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (o.by_k) cp[part][i] = count[base + i];
        if (o.by_p) mp[part][i] = mass[base + i];
      }
    }
  }
#pragma unroll
  for (int part = 0; part < kBinParts; ++part)
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      c[i] += cp[part][i];
      m[i] += mp[part][i];
    }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    cs += c[i];
    ms += m[i];
  }
  uint32_t all_c;
  uint64_t all_m;
  const uint32_t c0 = block_prefix<kThreads, uint32_t>(cs, wave_c, all_c);
  const uint64_t m0 = block_prefix<kThreads, uint64_t>(ms, wave_m, all_m);
  if (t == 0) found.all_mass = all_m;
  const bool cut = o.by_k && (uint64_t)o.top_k < all_c;  // else there are no more than k
  if (cut) {
    uint32_t cc = c0;
    uint64_t mm = m0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (cc < (uint64_t)o.top_k && cc + c[i] >= (uint64_t)o.top_k) {
        found.k = PER * t + i;
        found.k_before = cc;
        found.k_mass = mm;
        bin_mass = m[i];
        if (!o.by_p) {
          found.lo = found.hi = found.k;
          found.lo_mass = mm;
        }
      }
      cc += c[i];
      mm += m[i];
    }
  }
  __syncthreads();
  if (o.by_p) {
    // p times the mass of the first k: between what is above bin k and that with all of bin k
    uint64_t most = all_m, least = all_m;
    if (cut) {
      least = found.k_mass;
      most = least + bin_mass;
    }
    auto goal = [&](uint64_t total) {
      const double x = ceil(o.top_p * (double)total);
      return x > 1. ? (uint64_t)x : (uint64_t)1;
    };
    const uint64_t lo = goal(least), hi = goal(most);
    uint64_t mm = m0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (mm < lo && mm + m[i] >= lo) {
        found.lo = PER * t + i;
        found.lo_mass = mm;
      }
      if (mm < hi && mm + m[i] >= hi) found.hi = PER * t + i;
      mm += m[i];
    }
    __syncthreads();
  }
}

__global__ __launch_bounds__(kThreads) void search_kernel(Args a, Space sp) {
  __shared__ Bins found;
  const int64_t r = blockIdx.x;
  const RowOptions o(a, r);
  if (!o.by_k && !o.by_p) return;
  if (RowStats(sp.stats + r * sp.slices, sp.slices).empty()) return;  // it has no histogram
  search_bins(sp, r, o, found);
  __syncthreads();
  if (threadIdx.x == 0) sp.bins[r] = found;
}

// ---------------------------------------------------------------------------
// gather: per slice the sum of the weights above the border bins, and their logits.  21 us
// at 64 rows of 151936, 28 at 333 of 50257, 13 with the search at one row.
// ---------------------------------------------------------------------------
template <typename T, bool SEARCH>
__global__ __launch_bounds__(kThreads, SEARCH ? 4 : 8) void gather_kernel(Args a, Space sp) {
  __shared__ Bins found;
  __shared__ double table[kTable];
  __shared__ uint64_t cand[kCandidates];
  __shared__ uint32_t n_cand, cand_at;
  const int64_t r = blockIdx.y;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const RowOptions o(a, r);
  if (o.greedy || o.plain()) return;
  const RowStats s(sp.stats + r * sp.slices, sp.slices);
  if (s.empty()) return;
  if (t == 0) n_cand = 0;
  fill_table(table);
  const Weights w = weights_of(table, s.top, s.low, o.temp, a.fixed);
  if (SEARCH && (o.by_k || o.by_p)) {
    search_bins(sp, r, o, found);
    __syncthreads();
    if (blockIdx.x == 0 && t == 0) sp.bins[r] = found;  // the draw's
  }
  const Bins f = !o.by_k && !o.by_p ? Bins{kBins, kBins, kBins, 0, 0, 0, 0} : SEARCH ? found : sp.bins[r];
  const Row<T> row(a.logits, a.ld, r, a.vocab);
  for (int slice = blockIdx.x; slice < sp.slices; slice += gridDim.x) {
    double sum = 0.;
#pragma unroll
    for (int q = 0; q < kSliceGroups / kThreads; ++q) {
      const int g = slice * kSliceGroups + q * kThreads + t;
      if (g >= row.groups) break;
      float x[kGroup];
      row.load(g, x);
      int b[kGroup], least = kBins;
      bool found_one = false;
#pragma unroll
      for (int j = 0; j < kGroup; ++j) {
        b[j] = x[j] == -inf() ? kBins : w.bin(x[j]);
        least = min(least, b[j]);
        found_one |= b[j] < kBins && ((b[j] >= f.lo && b[j] <= f.hi) || b[j] == f.k);
      }
      if (least < f.lo) {
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
          const double y = w.of(x[j]);
          sum += b[j] < f.lo && y >= o.min_p ? y : 0.;
        }
      }
      if (found_one) {
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
          if (b[j] >= kBins || !((b[j] >= f.lo && b[j] <= f.hi) || b[j] == f.k)) continue;
          const uint32_t at = atomicAdd(&n_cand, 1u);
          if (at < (uint32_t)kCandidates)
            cand[at] = ((uint64_t)key_of(x[j]) << 32) | (0xffffffffu - (uint32_t)(row.first(g) + j));
        }
      }
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
    if (lane == 0) sp.sums[(r * sp.slices + slice) * kSums + wave] = sum;  // the draw adds them: no barrier per slice
  }
  // the work-group's candidates to the row's, from one atomic (their order does not matter)
  __syncthreads();
  const uint32_t mine = n_cand;
  if (mine == 0) return;
  if (t == 0) cand_at = atomicAdd(&sp.n_cand[r], mine);
  __syncthreads();
  for (uint32_t i = t; i < mine; i += kThreads)
    if (cand_at + i < (uint32_t)kCandidates && i < (uint32_t)kCandidates) sp.cand[r * kCandidates + cand_at + i] = cand[i];
}

// The token within a slice: the first in index order whose running sum of `weight(x, index)`
// exceeds s.target (an infinite target: the last with any).  A thread takes consecutive groups.
template <typename T, int N, typename F>
__device__ __forceinline__ void draw_token(const Args& a, int64_t r, const Row<T>& row, int slice, F&& weight, Scratch<N>& s) {
  constexpr int PER = kSliceGroups / N;
  const int g0 = slice * kSliceGroups + PER * (int)threadIdx.x;
  double y[PER][kGroup], sum = 0.;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    float x[kGroup];
    const int g = g0 + q, i0 = row.first(g);
    if (g < row.groups) row.load(g, x);
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      y[q][j] = g < row.groups && x[j] != -inf() ? weight(x[j], i0 + j) : 0.;
      sum += y[q][j];
    }
  }
  double all;
  double run = block_prefix<N, double>(sum, s.wave_d, all);
  const double target = s.target;
  int hit = -1, last = -1;
  double hit_y = 0., last_y = 0.;
#pragma unroll
  for (int q = 0; q < PER; ++q)
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      run += y[q][j];
      if (y[q][j] > 0.) {
        last = row.first(g0 + q) + j;
        last_y = y[q][j];
        if (hit < 0 && run > target) {
          hit = last;
          hit_y = last_y;
        }
      }
    }
  // the first hit of the work-group, or (by rounding) the slice's last kept logit
  if (threadIdx.x == 0) {
    s.token = 0x7fffffff;
    s.n_cand = -1;
  }
  __syncthreads();
  // (lanes are in index order: a wave's first lane with a hit, its last with any)
  const uint64_t hits = __builtin_amdgcn_ballot_w64(hit >= 0), lasts = __builtin_amdgcn_ballot_w64(last >= 0);
  const int lane = threadIdx.x & 63;
  if (hit >= 0 && lane == __ffsll((unsigned long long)hits) - 1) atomicMin(&s.token, hit);
  if (last >= 0 && lane == 63 - __clzll((long long)lasts)) atomicMax(&s.n_cand, last);
  __syncthreads();
  const bool none = s.token == 0x7fffffff;
  const int token = none ? s.n_cand : s.token;
  if (token >= 0 && token == (none ? last : hit)) {
    a.tokens[r] = token;
    a.logprobs[r] = (float)log((none ? last_y : hit_y) * s.scale / s.total);
  }
}

// The first wave: the slice that u times the total falls into (s.bin), what is left of the
// target there (s.target) and the total, from s.slice_sum.  A lane takes consecutive slices.
template <int N> __device__ __forceinline__ void pick_slice(Scratch<N>& s, int slices, double u) {
  const int lane = threadIdx.x, per = (slices + 63) / 64;
  const int b = min(slices, lane * per), e = min(slices, b + per);
  double sum = 0.;
  for (int i = b; i < e; ++i) sum += s.slice_sum[i];
  double incl = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(incl, o, 64);
    if (lane >= o) incl += y;
  }
  const double total = __shfl(incl, 63, 64), prev = __shfl_up(incl, 1, 64);
  const double target = u * total;
  double before = lane ? prev : 0., left = 0.;
  int pick = -1, last = 0;
  for (int i = b; i < e; ++i) {
    if (s.slice_sum[i] > 0.) last = i;
    if (pick < 0 && before + s.slice_sum[i] > target) {
      pick = i;
      left = target - before;
    }
    before += s.slice_sum[i];
  }
  const uint64_t found = __builtin_amdgcn_ballot_w64(pick >= 0);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) last = max(last, __shfl_xor(last, o, 64));
  const int from = found ? __ffsll((unsigned long long)found) - 1 : 0;
  pick = __shfl(pick, from, 64);
  left = __shfl(left, from, 64);
  if (lane == 0) {
    s.bin = found ? pick : last;  // u of 1 or more, or NaN: the last one
    s.target = found ? left : __builtin_huge_val();
    s.total = total;
    s.scale = 1.;
  }
}

// A row whose border bins hold too many logits, by its work-group alone: see find_border.  Logits
// that are all equal, or close together in a row whose range a mask of the lowest finite value
// stretches (the bins are then 1/32 octave wide).  A launch of such rows takes, with 151936 fp32
// tokens, T = 5 and top_p (top_k 50000 and top_p): 64 rows masked by -inf, none of them slow, 76
// (100) us, masked by the lowest value 135 (662), all equal 501 (454); 512 rows 309 (361), 388
// (1139), 1129 (1179).
template <typename T, int N>
__device__ __forceinline__ void slow_row(const Args& a, int64_t r, const Row<T>& row, const RowOptions& o, const Weights& w, int slices,
                         Scratch<N>& s) {
  const int t = threadIdx.x;
  Border border{key_of(-inf()), 0};
  if (o.by_k) {
    find_border<T, N, false>(row, w, (uint64_t)o.top_k, nullptr, s);
    border = s.border;
  }
  if (o.by_p) {
    // the mass of what top_k keeps, then the border of p times it
    uint64_t mass = 0;
    for (int g = t; g < row.groups; g += N) {
      float x[kGroup];
      row.load(g, x);
#pragma unroll
      for (int j = 0; j < kGroup; ++j)
        if (x[j] != -inf() && key_of(x[j]) > border.key) mass += w.fixed_of(x[j]);
    }
    uint64_t total = block_sum<N, uint64_t>(mass, s.wave_u);
    if (border.ties) total += border.ties * w.fixed_of(of_key(border.key));
    // the smallest whole mass that is p times the total or more; at least the first element
    const double goal = ceil(o.top_p * (double)total);
    const uint64_t want = goal > 1. ? (uint64_t)goal : 1;
    const Border limit = border;
    __syncthreads();
    find_border<T, N, true>(row, w, want, o.by_k ? &limit : nullptr, s);
    border = s.border;
  }
  const float border_x = of_key(border.key);
  const double tie_weight = border.ties ? w.of(border_x) : 0.;
  const bool tie_kept = border.ties && tie_weight >= o.min_p;
  auto above = [&](float x) { return x != -inf() && key_of(x) > border.key; };
  constexpr int PER = kSliceGroups / N;
  // kept mass and ties per slice
  for (int i = 0; i < slices; ++i) {
    double m = 0.;
    uint32_t ties = 0;
    for (int q = 0; q < PER; ++q) {
      const int g = i * kSliceGroups + q * N + t;
      if (g >= row.groups) break;
      float x[kGroup];
      row.load(g, x);
#pragma unroll
      for (int j = 0; j < kGroup; ++j) {
        if (above(x[j])) {
          const double y = w.of(x[j]);
          m += y >= o.min_p ? y : 0.;
        } else if (tie_kept && x[j] == border_x) {
          ++ties;
        }
      }
    }
    m = block_sum<N, double>(m, s.wave_d);
    if (tie_kept) ties = block_sum<N, uint32_t>(ties, s.wave_c);
    if (t == 0) {
      s.slice_sum[i] = m;
      s.slice_add[i] = ties;
    }
  }
  __syncthreads();
  if (t == 0) {
    uint32_t left = tie_kept ? (uint32_t)border.ties : 0;
    for (int i = 0; i < slices; ++i) {
      const uint32_t n = min(left, (uint32_t)s.slice_add[i]);
      s.slice_add[i] = n;
      left -= n;
      s.slice_sum[i] += n * tie_weight;
    }
  }
  __syncthreads();
  if (t < 64) pick_slice(s, slices, o.u);
  __syncthreads();
  // the slice's first ties, by their rank in it (a thread takes consecutive groups, as the draw does)
  const int slice = s.bin;
  uint32_t ties = 0;
  for (int q = 0; tie_kept && q < PER; ++q) {
    const int g = slice * kSliceGroups + PER * t + q;
    if (g >= row.groups) break;
    float x[kGroup];
    row.load(g, x);
#pragma unroll
    for (int j = 0; j < kGroup; ++j) ties += x[j] == border_x;
  }
  uint32_t all_ties, rank = block_prefix<N, uint32_t>(ties, s.wave_c, all_ties);
  const uint32_t take = (uint32_t)s.slice_add[slice];
  draw_token<T, N>(a, r, row, slice, [&](float x, int) {
    if (above(x)) {
      const double y = w.of(x);
      return y >= o.min_p ? y : 0.;
    }
    return tie_kept && x == border_x && rank++ < take ? tie_weight : 0.;
  }, s);
}

// draw: one work-group a row.  Latency: the sort of its candidates, the sum over the slices and
// the one slice read again follow one another: 11 us at one row, 18 at 64, 13 at 512 without filters.
template <typename T>
__global__ __launch_bounds__(kDrawThreads) void draw_kernel(Args a, Space sp) {
  constexpr int N = kDrawThreads;
  __shared__ Scratch<N> s;
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x;
  const RowOptions o(a, r);
  const SliceStats* stats = sp.stats + r * sp.slices;
  each<N>(sp.slices, [&](int i) {
    const double* sums = sp.sums + (r * sp.slices + i) * kSums;
    double sum = sums[0];
    if (!o.plain())
#pragma unroll
      for (int q = 1; q < kSums; ++q) sum += sums[q];
    s.slice_sum[i] = sum;
    s.slice_add[i] = 0;
  });
  const RowStats rs(stats, sp.slices);
  if (rs.empty()) {  // nothing to draw
    if (t == 0) {
      a.tokens[r] = -1;
      a.logprobs[r] = __builtin_nanf("");
    }
    return;
  }
  if (o.greedy) {
    if (t == 0) {
      a.tokens[r] = rs.at;
      a.logprobs[r] = 0.f;
    }
    return;
  }
  fill_table(s.table);
  const Row<T> row(a.logits, a.ld, r, a.vocab);
  const Weights w = weights_of(s.table, rs.top, rs.low, o.temp, a.fixed);
  if (o.plain()) {
    // slices' sums are relative to their own maxima
    each<N>(sp.slices, [&](int i) { s.slice_sum[i] *= w.of(stats[i].top); });
    __syncthreads();
    if (t < 64) pick_slice(s, sp.slices, o.u);
    __syncthreads();
    const float top = stats[s.bin].top;
    const double scale = w.of(top);
    __syncthreads();
    if (t == 0) {
      s.scale = scale;
      s.target /= scale;
    }
    __syncthreads();
    const Weights v = weights_of(s.table, top, rs.low, o.temp, a.fixed);
    draw_token<T, N>(a, r, row, s.bin, [&](float x, int) { return v.of(x); }, s);
    return;
  }
  uint64_t border = 0;  // the last kept (key, index); 0: no border
  if (o.by_k || o.by_p) {
    const Bins f = sp.bins[r];
    const int have = (int)min(sp.n_cand[r], (uint32_t)kCandidates + 1);
    if (have > kCandidates) {
      slow_row<T, N>(a, r, row, o, w, sp.slices, s);
      return;
    }
    if (have) {
      each<N>(have, [&](int i) { s.cand[i] = sp.cand[r * kCandidates + i]; });
      sort_candidates<N>(s, have);
      // a thread takes consecutive candidates
      const int per = (have + N - 1) / N, b = min(have, per * t), e = min(have, b + per);
      auto logit = [&](int i) { return of_key((uint32_t)(s.cand[i] >> 32)); };
      // the last of the first k: in bin k's group, which ends the candidates
      int last = have - 1;
      uint64_t mass_k = 0;
      if (f.k < kBins) {
        uint32_t before_k = 0;
        for (int i = b; i < e; ++i) before_k += w.bin(logit(i)) < f.k;
        before_k = block_sum<N, uint32_t>(before_k, s.wave_c);
        last = (int)before_k + (int)(o.top_k - (int64_t)f.k_before) - 1;
        if (o.by_p) {
          uint64_t kept = 0;
          for (int i = max(b, (int)before_k); i < min(e, last + 1); ++i) kept += w.fixed_of(logit(i));
          mass_k = f.k_mass + block_sum<N, uint64_t>(kept, s.wave_u);
        }
      } else {
        mass_k = f.all_mass;
      }
      if (o.by_p) {
        // p times the mass of the first k, reached in the bins [lo, hi], which begin the candidates
        const double goal = ceil(o.top_p * (double)mass_k);
        const uint64_t want = goal > 1. ? (uint64_t)goal : 1;
        uint64_t mine = 0, all;
        for (int i = b; i < e; ++i) mine += w.fixed_of(logit(i));
        uint64_t run = block_prefix<N, uint64_t>(mine, s.wave_u, all) + f.lo_mass;
        if (t == 0) s.bin = last;  // where p times the mass rounds past it
        __syncthreads();
        for (int i = b; i < e; ++i) {
          const uint64_t next = run + w.fixed_of(logit(i));
          if (run < want && next >= want) s.bin = i;  // one element
          run = next;
        }
        __syncthreads();
        last = s.bin;
      }
      border = s.cand[last];
      // the kept candidates' mass, by slice
      for (int i = b; i < min(e, last + 1); ++i) {
        const float x = logit(i);
        if (!(w.of(x) >= o.min_p)) continue;
        const int idx = (int)(0xffffffffu - (uint32_t)s.cand[i]);
        atomicAdd((unsigned long long*)&s.slice_add[(idx + row.lead) / kSlice], (unsigned long long)w.fixed_of(x));
      }
    }
  }
  __syncthreads();
  const double unit = 1. / a.fixed;  // a power of two
  each<N>(sp.slices, [&](int i) { s.slice_sum[i] += (double)s.slice_add[i] * unit; });
  __syncthreads();
  if (t < 64) pick_slice(s, sp.slices, o.u);
  __syncthreads();
  draw_token<T, N>(a, r, row, s.bin, [&](float x, int i) {
    const uint64_t me = ((uint64_t)key_of(x) << 32) | (0xffffffffu - (uint32_t)i);
    if (me < border) return 0.;
    const double y = w.of(x);
    return y >= o.min_p ? y : 0.;
  }, s);
}

int slices_of(int64_t vocab) {
  return (int)((((vocab + 2 * kGroup - 2) / kGroup) + kSliceGroups - 1) / kSliceGroups);  // of a row at any alignment
}
int64_t up16(int64_t b) { return (b + 15) / 16 * 16; }

// Work-groups a row, for about 1024 in the launch, and no more than the slices fill evenly (19 slices over 16
// work-groups end when the three that have two do: 10 of two).
int64_t per_row(int64_t rows, int64_t slices, int64_t most) {
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>({most, slices, (1024 + rows / 2) / rows}));
  const int64_t each = (slices + parts - 1) / parts;
  return (slices + each - 1) / each;
}

int64_t space_of(int64_t rows, int64_t vocab, bool bins, int64_t parts, char* base, Space* sp) {
  const int64_t slices = slices_of(vocab);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* p = base + at;
    at += up16(bytes);
    return p;
  };
  Space s{};
  s.slices = (int)slices;
  s.parts = (int)parts;
  s.stats = (SliceStats*)take(rows * slices * (int64_t)sizeof(SliceStats));
  s.sums = (double*)take(rows * slices * kSums * 8);
  if (bins) {
    s.bins = (Bins*)take(rows * (int64_t)sizeof(Bins));
    s.mass = (uint64_t*)take(rows * parts * kBins * 8);
    s.count = (uint32_t*)take(rows * parts * kBins * 4);
    s.cand = (uint64_t*)take(rows * kCandidates * 8);
    s.n_cand = (uint32_t*)take(rows * 4);
  }
  if (sp) *sp = s;
  return at;
}

// How a call's rows are cut into sets of launches of equal size (but the last), so that a set's workspace stays below
// about kSpaceBytes (filters over 151936 tokens: 2277 rows; a histogram of several parts comes with few rows), and
// the parts of a row's histogram in all of them.
constexpr int64_t kSpaceBytes = 128 << 20;
struct Sets {
  int64_t rows, parts, bytes;
  Sets(int64_t all, int64_t vocab, bool bins) {
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(4096, kSpaceBytes / space_of(1, vocab, bins, 1, nullptr, nullptr)));
    const int64_t sets = (all + most - 1) / most;
    rows = (all + sets - 1) / sets;
    parts = per_row(rows, slices_of(vocab), kBinParts);
    bytes = space_of(rows, vocab, bins, parts, nullptr, nullptr);
  }
};

template <typename T>
void launch(const Args& a, const Space& sp, int64_t rows, bool filters, bool bins, hipStream_t s) {
  const dim3 grid((unsigned)sp.slices, (unsigned)rows), block(kMaxThreads);
  {
    TimedLaunch timed_("sampling.maxima_kernel", s);
    if (bins) hipLaunchKernelGGL((maxima_kernel<T, true>), grid, block, 0, s, a, sp);
    else hipLaunchKernelGGL((maxima_kernel<T, false>), grid, block, 0, s, a, sp);
  }
  if (bins) {
    TimedLaunch timed_("sampling.bins_kernel", s);
    hipLaunchKernelGGL(bins_kernel<T>, dim3((unsigned)sp.parts, (unsigned)rows), dim3(kThreads), 0, s, a, sp);
  }
  if (bins && rows > kFewRows) {
    TimedLaunch timed_("sampling.search_kernel", s);
    hipLaunchKernelGGL(search_kernel, dim3((unsigned)rows), dim3(kThreads), 0, s, a, sp);
  }
  if (filters) {
    TimedLaunch timed_("sampling.gather_kernel", s);
    const dim3 gathers((unsigned)per_row(rows, sp.slices, sp.slices), (unsigned)rows), threads(kThreads);
    if (bins && rows <= kFewRows) hipLaunchKernelGGL((gather_kernel<T, true>), gathers, threads, 0, s, a, sp);
    else hipLaunchKernelGGL((gather_kernel<T, false>), gathers, threads, 0, s, a, sp);
  }
  {
    TimedLaunch timed_("sampling.draw_kernel", s);
    hipLaunchKernelGGL(draw_kernel<T>, dim3((unsigned)rows), dim3(kDrawThreads), 0, s, a, sp);
  }
}

}  // namespace sample
}  // namespace ts

extern "C" {

int64_t ts_sample_workspace(int64_t rows, int64_t vocab, int filters) {
  using namespace ts::sample;
  return rows > 0 && vocab > 0 && vocab <= kMaxVocab ? Sets(rows, vocab, filters != 0).bytes : 0;
}

int ts_sample(const void* logits, int64_t ld_logits, int64_t rows, int64_t vocab, const void* uniform,
              int uniform_dtype, const float* temperature, double temperature_all, const int32_t* top_k,
              int64_t top_k_all, const float* top_p, double top_p_all, const float* min_p, double min_p_all,
              int64_t* tokens, float* logprobs, void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
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
  a.fixed = (double)(1ull << std::min(62 - bits, 50));  // vocab weights of at most 1 stay below 2^62
  a.tokens = tokens;
  a.logprobs = logprobs;
  const bool by_min = min_p || min_p_all > 0;
  const bool bins = top_k || top_p || (top_k_all > 1 && top_k_all < vocab) || top_p_all < 1;
  const Sets sets(rows, vocab, bins);
  TS_CHECK_ARG(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= sets.bytes,
               "ts_sample: workspace of %lld bytes, need %lld", (long long)workspace_bytes, (long long)sets.bytes);
  hipStream_t s = (hipStream_t)stream;
  const int64_t size = dtype == TS_F32 ? 4 : 2;
  for (int64_t r0 = 0; r0 < rows; r0 += sets.rows) {
    const int64_t n = std::min(sets.rows, rows - r0);
    Args b = a;
    b.logits = (const char*)logits + r0 * ld_logits * size;
    b.uniform = (const char*)uniform + r0 * (a.uniform_wide ? 8 : 4);
    if (temperature) b.o.temperature += r0;
    if (top_k) b.o.top_k += r0;
    if (top_p) b.o.top_p += r0;
    if (min_p) b.o.min_p += r0;
    b.tokens += r0;
    b.logprobs += r0;
    Space sp;
    space_of(n, vocab, bins, sets.parts, (char*)workspace, &sp);
    if (dtype == TS_F32) launch<float>(b, sp, n, bins || by_min, bins, s);
    else if (dtype == TS_F16) launch<ts::f16>(b, sp, n, bins || by_min, bins, s);
    else launch<ts::bf16>(b, sp, n, bins || by_min, bins, s);
  }
  return ts::check_launch("ts_sample");
}

}  // extern "C"
