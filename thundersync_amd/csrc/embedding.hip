// Embedding lookup with a scale, and the table's gradient by sorted tokens, for gfx950.
//
//   out[n] = scale W[ids[n]]        dW[v] = scale sum over n with ids[n] = v of dout[n]
//
// Lookup: bandwidth-bound, 16 bytes a lane.  Gradient: the tokens' positions are sorted by
// id (stable, so equal ids keep the token order), and chunks of sorted positions add
// up their rows of dout in fp32; an id whose positions end inside the chunk is written once,
// one that a chunk border cuts leaves fp32 partial rows that join_kernel adds in chunk
// order.  No atomics on values: the same bits every time.  Rows of the table that no token
// names are zeros.  Bound by the write of the [V, D] gradient where tokens are few.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "timing.h"
#include "../../include/thundersync_hip.h"

namespace ts {
namespace embed {

constexpr int kThreads = 256;
constexpr int64_t kMaxBlocks = 1 << 23;  // of kThreads along one axis: a launch takes fewer than 2^32 threads there
constexpr int64_t kMaxTokens = 1 << 28;  // of a gradient: every tile of its sort reads all tiles' counts
constexpr int kChunk = 32;      // sorted positions per work-group of the reduction, at most
constexpr int kDigitBits = 9, kBins = 1 << kDigitBits;
constexpr int kRounds = 8, kWaves = kThreads / 64, kSortTile = kThreads * kRounds;

template <typename T> constexpr int kVec = 16 / sizeof(T);

// VEC elements as fp32, and back with one rounding
template <typename T, int VEC> __device__ __forceinline__ void load_vec(const T* p, float (&x)[VEC]) {
  if constexpr (VEC == 1) {
    x[0] = to_f(*p);
  } else if constexpr (sizeof(T) == 2) {
    load8(p, x);
  } else {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i];
  }
}
template <typename T, int VEC> __device__ __forceinline__ void store_vec(T* p, const float (&x)[VEC]) {
  if constexpr (VEC == 1) *p = from_f<T>(x[0]);
  else if constexpr (sizeof(T) == 2) store8(p, x);
  else *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
}

// ---------------------------------------------------------------------------
// lookup; a token id outside [0, vocab) gives a row of NaN.  Bound by HBM: 65536 fp32 rows of
// 1024 in 81 us (268 MB written, 166 MB fetched: 5.4 TB/s), 16384 bf16 rows of 4096 in 46 us.
// ---------------------------------------------------------------------------
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void lookup_kernel(const int64_t* __restrict__ ids, int64_t n,
                                                          const T* __restrict__ w, int64_t ldw, int64_t vocab, int dim,
                                                          float scale, T* __restrict__ out) {
  for (int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; row < n; row += (int64_t)gridDim.x * blockDim.y) {
    const int64_t id = ids[row];
    const bool ok = id >= 0 && id < vocab;
    for (int d = (blockIdx.y * blockDim.x + threadIdx.x) * VEC; d < dim; d += gridDim.y * blockDim.x * VEC) {
      float x[VEC];
      if (ok) load_vec<T, VEC>(w + id * ldw + d, x);
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = ok ? x[i] * scale : __builtin_nanf("");
      store_vec<T, VEC>(out + row * dim + d, x);
    }
  }
}

// ---------------------------------------------------------------------------
// stable sort of the positions by id, kDigitBits at a time from the low end, in tiles of
// kSortTile.  The key of a token that takes no part (outside the vocabulary, or the padding
// id) is `vocab`.  A pass is two launches, of the tiles' digit counts and of their placement,
// or with one tile all passes are one launch in LDS.  The sort occupies a few CUs, so the
// rest of each launch's grid writes its share of the gradient's zeros: a training batch's
// sort (16384 tokens, 48 us by itself) then costs nothing beside them.  The four launches that
// write a [151936, 4096] bf16 gradient's 1.24 GB of zeros take 225 us (5.5 TB/s); the one launch
// of 500 tokens, with [50257, 2560]'s 257 MB, 37 us (6.9 TB/s).
// ---------------------------------------------------------------------------
struct SortArgs {
  const int64_t* ids;     // first pass: key from the ids, position the index
  const uint32_t* key_in; // later passes
  const uint32_t* pos_in;
  uint32_t* key_out;
  uint32_t* pos_out;
  uint32_t* hist;         // [tiles][kBins]
  int64_t n;
  int64_t vocab, padding;
  int tiles, shift;
  // this launch's zeros: 16-byte words [zero0, zero1) of `zero`, and the bytes behind the last
  u32x4* zero;
  int64_t zero0, zero1;
  unsigned char* tail;
  int tail_bytes;
};

__device__ __forceinline__ void write_zeros(const SortArgs& a, int block, int blocks) {
  const int64_t step = (int64_t)blocks * kThreads;
  for (int64_t i = a.zero0 + (int64_t)block * kThreads + threadIdx.x; i < a.zero1; i += step)
    a.zero[i] = u32x4{0, 0, 0, 0};
  if (block == 0 && (int)threadIdx.x < a.tail_bytes) a.tail[threadIdx.x] = 0;
}

__device__ __forceinline__ uint32_t key_at(const SortArgs& a, int64_t i) {
  if (!a.ids) return a.key_in[i];
  const int64_t id = a.ids[i];
  return id < 0 || id >= a.vocab || id == a.padding ? (uint32_t)a.vocab : (uint32_t)id;
}

// Lanes of the wave whose digit equals this lane's, among the `on` ones.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, bool on) {
  uint64_t m = __builtin_amdgcn_ballot_w64(on);
#pragma unroll
  for (int b = 0; b < kDigitBits; ++b) {
    const uint64_t set = __builtin_amdgcn_ballot_w64((digit >> b) & 1);
    m &= (digit >> b) & 1 ? set : ~set;
  }
  return m;
}

// A tile's elements are kRounds x 64 consecutive ones a wave, 64 at a time.  base[wave][digit]
// holds the wave's counts, then (with each digit's first place in `first`) the place of the
// wave's first element of the digit.
struct Places {
  uint32_t base[kWaves][kBins];
  uint32_t wave_sum[kWaves];
};
__device__ __forceinline__ void count_digits(Places& p, const uint32_t (&key)[kRounds], const bool (&on)[kRounds],
                                             int shift) {
  const int wave = threadIdx.x >> 6;
  for (int b = threadIdx.x; b < kWaves * kBins; b += kThreads) (&p.base[0][0])[b] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
    if (on[r]) atomicAdd(&p.base[wave][(key[r] >> shift) & (kBins - 1)], 1u);
  __syncthreads();
}
// two consecutive digits a thread: `all` of each in the whole sort, `before` in earlier tiles
__device__ __forceinline__ void place_digits(Places& p, const uint32_t (&all)[2], const uint32_t (&before)[2]) {
  static_assert(kBins == 2 * kThreads, "two digits a thread");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t incl = all[0] + all[1];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(incl, o, 64);
    if (lane >= o) incl += y;
  }
  if (lane == 63) p.wave_sum[wave] = incl;
  __syncthreads();
  uint32_t first = incl - all[0] - all[1];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) first += w < wave ? p.wave_sum[w] : 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int b = 2 * threadIdx.x + i;
    uint32_t at = first + (i ? all[0] : 0) + before[i];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const uint32_t c = p.base[w][b];
      p.base[w][b] = at;
      at += c;
    }
  }
  __syncthreads();
}
// an element's place is its digit's base for the wave plus the earlier elements with the digit
template <typename F>
__device__ __forceinline__ void put_digits(Places& p, const uint32_t (&key)[kRounds], const bool (&on)[kRounds],
                                           int shift, F&& put) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint32_t digit = (key[r] >> shift) & (kBins - 1);
    const uint64_t same = same_digit(digit, on[r]);
    const uint64_t before = same & ((1ull << lane) - 1);
    if (on[r]) put(r, p.base[wave][digit] + (uint32_t)__popcll(before));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (on[r] && before == 0) p.base[wave][digit] += (uint32_t)__popcll(same);  // the digit's first lane
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

__global__ __launch_bounds__(kThreads) void sort_count_kernel(SortArgs a) {
  if ((int)blockIdx.x >= a.tiles) return write_zeros(a, (int)blockIdx.x - a.tiles, (int)gridDim.x - a.tiles);
  __shared__ uint32_t bins[kBins];
  for (int b = threadIdx.x; b < kBins; b += kThreads) bins[b] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * kSortTile;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = i0 + r * kThreads + threadIdx.x;
    if (i < a.n) atomicAdd(&bins[(key_at(a, i) >> a.shift) & (kBins - 1)], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kThreads) a.hist[(int64_t)blockIdx.x * kBins + b] = bins[b];
}

// Each tile adds up the tiles' counts itself (two digits a thread, rows of 2 KB): for the
// tiles of a batch less than a launch that would scan them.
__global__ __launch_bounds__(kThreads) void sort_place_kernel(SortArgs a) {
  if ((int)blockIdx.x >= a.tiles) return write_zeros(a, (int)blockIdx.x - a.tiles, (int)gridDim.x - a.tiles);
  __shared__ Places p;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i0 = (int64_t)blockIdx.x * kSortTile + wave * (kRounds * 64) + lane;
  uint32_t key[kRounds], pos[kRounds];
  bool on[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = i0 + 64 * r;
    on[r] = i < a.n;
    key[r] = on[r] ? key_at(a, i) : 0;
    pos[r] = on[r] ? (a.ids ? (uint32_t)i : a.pos_in[i]) : 0;
  }
  uint32_t all[2] = {}, before[2] = {};
#pragma unroll 8
  for (int tile = 0; tile < a.tiles; ++tile) {
    const u32x2 c = *reinterpret_cast<const u32x2*>(a.hist + (int64_t)tile * kBins + 2 * threadIdx.x);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      all[i] += c[i];
      before[i] += tile < (int)blockIdx.x ? c[i] : 0;
    }
  }
  count_digits(p, key, on, a.shift);
  place_digits(p, all, before);
  put_digits(p, key, on, a.shift, [&](int r, uint32_t at) {
    a.key_out[at] = key[r];
    a.pos_out[at] = pos[r];
  });
}

// at most kSortTile tokens: every pass in LDS
__global__ __launch_bounds__(kThreads) void sort_tile_kernel(SortArgs a) {
  if ((int)blockIdx.x >= a.tiles) return write_zeros(a, (int)blockIdx.x - a.tiles, (int)gridDim.x - a.tiles);
  __shared__ Places p;
  __shared__ uint32_t keys[kSortTile], places[kSortTile];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i0 = wave * (kRounds * 64) + lane, n = (int)a.n;
  uint32_t key[kRounds], pos[kRounds];
  bool on[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    pos[r] = i0 + 64 * r;
    on[r] = (int)pos[r] < n;
    key[r] = on[r] ? key_at(a, pos[r]) : 0;
  }
  for (int shift = 0; shift == 0 || (a.vocab >> shift) > 0; shift += kDigitBits) {
    if (shift) {
#pragma unroll
      for (int r = 0; r < kRounds; ++r)
        if (on[r]) {
          key[r] = keys[i0 + 64 * r];
          pos[r] = places[i0 + 64 * r];
        }
    }
    count_digits(p, key, on, shift);  // (its barriers also end the reads above)
    uint32_t all[2] = {};
    const uint32_t before[2] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int w = 0; w < kWaves; ++w) all[i] += p.base[w][2 * threadIdx.x + i];
    place_digits(p, all, before);
    put_digits(p, key, on, shift, [&](int r, uint32_t at) {
      keys[at] = key[r];
      places[at] = pos[r];
    });
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += kThreads) {
    a.key_out[i] = keys[i];
    a.pos_out[i] = places[i];
  }
}

// ---------------------------------------------------------------------------
// sums of the rows of dout over runs of equal ids.  A work-group takes a chunk of sorted
// positions and, with few rows of output a chunk, is bound by the latency of its gathered rows:
// eight rows are loaded ahead of the sums.  65536 fp32 rows of 1024: 96 us (333 MB, 3.5 TB/s);
// 16384 bf16 rows of 4096: 70 us; 500: 6 us.  The join: 12, 9 and 4 us.
// ---------------------------------------------------------------------------
struct ReduceArgs {
  const uint32_t* key;  // sorted ids
  const uint32_t* pos;
  int64_t n;
  uint32_t vocab;       // the key of tokens that take no part
  int64_t ldd;          // row stride of dout
  int dim;
  float scale;
  int chunk;            // sorted positions per work-group
  float* part;          // [chunks][2][dim]: the run that began earlier, the run that goes on
};

template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void reduce_kernel(ReduceArgs a, const T* __restrict__ dout,
                                                          T* __restrict__ dw) {
  __shared__ uint32_t key[kChunk + 2], pos[kChunk];  // key[0], key[count + 1]: the neighbours'
  const int64_t i0 = (int64_t)blockIdx.x * a.chunk;
  const int count = (int)min((int64_t)a.chunk, a.n - i0);
  const int t = threadIdx.x;
  if (t < count) pos[t] = a.pos[i0 + t];
  // `vocab` stands for no neighbour: runs of it are skipped anyway
  if (t < count + 2) key[t] = i0 + t >= 1 && i0 + t <= a.n ? a.key[i0 + t - 1] : a.vocab;
  __syncthreads();
  const int d = (blockIdx.y * kThreads + t) * VEC;
  if (d >= a.dim) return;
  float acc[VEC] = {};
  bool earlier = key[0] == key[1];
  // U rows at a time, the next U in flight while these are added; a row past the chunk or of a
  // token that takes no part is the chunk's first again
  constexpr int U = 8;
  struct alignas(sizeof(T) * VEC) Raw {
    T v[VEC];
  };
  auto fetch = [&](int j0, Raw (&x)[U]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u < count && key[j0 + u + 1] != a.vocab ? j0 + u : 0;
      x[u] = *reinterpret_cast<const Raw*>(dout + pos[j] * a.ldd + d);
    }
  };
  // false: nothing follows
  auto add = [&](int j0, const Raw (&x)[U]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u;
      if (j >= count) return false;
      const uint32_t id = key[j + 1];
      if (id == a.vocab) return false;  // sorted last
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += to_f(x[u].v[i]);
      const bool last = j + 1 == count;
      if (!last && key[j + 2] == id) continue;
      const bool goes_on = last && key[j + 2] == id;
      if (earlier || goes_on) {
        float* q = a.part + ((int64_t)blockIdx.x * 2 + (earlier ? 0 : 1)) * a.dim + d;
#pragma unroll
        for (int i = 0; i < VEC; ++i) q[i] = acc[i];
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] *= a.scale;
        store_vec<T, VEC>(dw + (int64_t)id * a.dim + d, acc);
      }
      earlier = false;
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
    }
    return true;
  };
  Raw x[U], y[U];
  fetch(0, x);
  for (int j0 = 0; j0 < count; j0 += 2 * U) {
    fetch(j0 + U, y);
    if (!add(j0, x)) return;
    fetch(j0 + 2 * U, x);
    if (!add(j0 + U, y)) return;
  }
}

// the runs that chunk borders cut: the chunk a run begins in adds its parts in chunk order
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void join_kernel(ReduceArgs a, T* __restrict__ dw) {
  const int64_t c = blockIdx.x, first = c * a.chunk, next = first + a.chunk;
  if (next >= a.n) return;  // the last chunk: its last run goes nowhere
  const uint32_t id = a.key[next - 1];
  if (id == a.vocab || a.key[next] != id) return;
  if (a.key[first] == id && first > 0 && a.key[first - 1] == id) return;  // began earlier
  // the first chunk that the run does not reach past, kThreads of them looked at at a time (one
  // after the other the look-ups of a frequent token's 150 chunks took longer than their sums)
  __shared__ int ends;
  int64_t end = c + 2;
  while (true) {
    if (threadIdx.x == 0) ends = kThreads;
    __syncthreads();
    const int64_t e = end + threadIdx.x;
    if (e * a.chunk >= a.n || a.key[e * a.chunk - 1] != id || a.key[e * a.chunk] != id) atomicMin(&ends, (int)threadIdx.x);
    __syncthreads();
    end += ends;
    if (ends < kThreads) break;
    __syncthreads();
  }
  const int d = (blockIdx.y * kThreads + threadIdx.x) * VEC;
  if (d >= a.dim) return;
  float acc[VEC];
  const float* q = a.part + (c * 2 + 1) * a.dim + d;
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = q[i];
#pragma unroll 16
  for (int64_t e = c + 1; e < end; ++e) {
    const float* r = a.part + e * 2 * a.dim + d;
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] += r[i];
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] *= a.scale;
  store_vec<T, VEC>(dw + (int64_t)id * a.dim + d, acc);
}

bool ok16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int64_t tiles_of(int64_t n) { return (n + kSortTile - 1) / kSortTile; }
// Few tokens: chunks of 8, for work-groups enough
int chunk_of(int64_t n) { return n <= 4096 ? 8 : kChunk; }
int64_t chunks_of(int64_t n) { return (n + chunk_of(n) - 1) / chunk_of(n); }
int64_t up16(int64_t b) { return (b + 15) / 16 * 16; }

// the workspace: two (key, position) buffers, the digit counts, the partial rows
struct Workspace {
  int64_t key[2], pos[2], hist, part, bytes;
  Workspace(int64_t n, int64_t dim) {
    int64_t at = 0;
    auto take = [&](int64_t bytes_) {
      const int64_t r = at;
      at += up16(bytes_);
      return r;
    };
    for (int i = 0; i < 2; ++i) {
      key[i] = take(4 * n);
      pos[i] = take(4 * n);
    }
    hist = take(4 * (int64_t)kBins * tiles_of(n));
    part = take(8 * chunks_of(n) * dim);
    bytes = at;
  }
};

template <typename T>
void launch_lookup(const int64_t* ids, int64_t n, const void* w, int64_t ldw, int64_t vocab, int64_t dim, float scale,
                   void* out, hipStream_t s) {
  const bool vec = ok16(w) && ok16(out) && dim % kVec<T> == 0 && ldw % kVec<T> == 0;
  const int64_t lanes = vec ? dim / kVec<T> : dim;
  int tx = 1;
  while (tx < kThreads && tx < lanes) tx *= 2;
  const dim3 block((unsigned)tx, (unsigned)(kThreads / tx));
  const dim3 grid((unsigned)std::min<int64_t>((n + block.y - 1) / block.y, kMaxBlocks), (unsigned)((lanes + tx - 1) / tx));
  if (vec)
    hipLaunchKernelGGL((lookup_kernel<T, kVec<T>>), grid, block, 0, s, ids, n, (const T*)w, ldw, vocab, (int)dim, scale,
                       (T*)out);
  else
    hipLaunchKernelGGL((lookup_kernel<T, 1>), grid, block, 0, s, ids, n, (const T*)w, ldw, vocab, (int)dim, scale,
                       (T*)out);
}

template <typename T>
void launch_sums(const ReduceArgs& a, const void* dout, void* dw, hipStream_t s) {
  const bool vec = ok16(dout) && ok16(dw) && a.dim % kVec<T> == 0 && a.ldd % kVec<T> == 0;
  const int64_t lanes = vec ? a.dim / kVec<T> : a.dim;
  const dim3 grid((unsigned)chunks_of(a.n), (unsigned)((lanes + kThreads - 1) / kThreads));
  {
    TimedLaunch timed_("embedding.reduce_kernel", s);
    if (vec) hipLaunchKernelGGL((reduce_kernel<T, kVec<T>>), grid, dim3(kThreads), 0, s, a, (const T*)dout, (T*)dw);
    else hipLaunchKernelGGL((reduce_kernel<T, 1>), grid, dim3(kThreads), 0, s, a, (const T*)dout, (T*)dw);
  }
  if (grid.x == 1) return;
  TimedLaunch timed_("embedding.join_kernel", s);
  if (vec) hipLaunchKernelGGL((join_kernel<T, kVec<T>>), grid, dim3(kThreads), 0, s, a, (T*)dw);
  else hipLaunchKernelGGL((join_kernel<T, 1>), grid, dim3(kThreads), 0, s, a, (T*)dw);
}

}  // namespace embed
}  // namespace ts

using namespace ts::embed;

extern "C" {

int ts_embedding_fwd(const int64_t* ids, int64_t n, const void* weight, int64_t ld_weight, int64_t vocab, int64_t dim,
                     float scale, void* out, int dtype, void* stream) {
  TS_CHECK_ARG(dtype == TS_F32 || dtype == TS_F16 || dtype == TS_BF16, "ts_embedding_fwd: dtype %d", dtype);
  TS_CHECK_ARG(n >= 0 && n < (1ll << 31) && vocab >= 0 && vocab < (1ll << 31) && dim >= 1 && dim < (1 << 20) &&
                   ld_weight >= dim,
               "ts_embedding_fwd: bad shape n=%lld vocab=%lld dim=%lld", (long long)n, (long long)vocab,
               (long long)dim);
  if (n == 0) return TS_OK;
  TS_CHECK_ARG(ids && out && (weight || vocab == 0), "ts_embedding_fwd: null pointer");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("embedding.lookup_kernel", s);
    if (dtype == TS_F32) launch_lookup<float>(ids, n, weight, ld_weight, vocab, dim, scale, out, s);
    else if (dtype == TS_F16) launch_lookup<ts::f16>(ids, n, weight, ld_weight, vocab, dim, scale, out, s);
    else launch_lookup<ts::bf16>(ids, n, weight, ld_weight, vocab, dim, scale, out, s);
  }
  return ts::check_launch("ts_embedding_fwd");
}

int64_t ts_embedding_bwd_workspace(int64_t n, int64_t dim) {
  return n > 0 && dim > 0 ? Workspace(n, dim).bytes : 0;
}

int ts_embedding_bwd(const int64_t* ids, int64_t n, const void* grad_out, int64_t ld_grad, int64_t vocab, int64_t dim,
                     int64_t padding, float scale, void* grad_weight, void* workspace, int64_t workspace_bytes,
                     int dtype, void* stream) {
  TS_CHECK_ARG(dtype == TS_F32 || dtype == TS_F16 || dtype == TS_BF16, "ts_embedding_bwd: dtype %d", dtype);
  TS_CHECK_ARG(n >= 0 && n < kMaxTokens && vocab >= 0 && vocab < (1ll << 31) - 1 && dim >= 1 && dim < (1 << 20),
               "ts_embedding_bwd: bad shape n=%lld vocab=%lld dim=%lld", (long long)n, (long long)vocab,
               (long long)dim);
  if (vocab == 0) return TS_OK;
  TS_CHECK_ARG(grad_weight && ok16(grad_weight), "ts_embedding_bwd: grad_weight null or not 16-byte aligned");
  hipStream_t s = (hipStream_t)stream;
  const int64_t bytes = vocab * dim * (dtype == TS_F32 ? 4 : 2);
  TS_CHECK_ARG(n == 0 || (ids && grad_out && ld_grad >= 0), "ts_embedding_bwd: null pointer");
  TS_CHECK_ARG(n == 0 || (workspace && ok16(workspace) && workspace_bytes >= ts_embedding_bwd_workspace(n, dim)),
               "ts_embedding_bwd: workspace of %lld bytes, need %lld", (long long)workspace_bytes,
               (long long)ts_embedding_bwd_workspace(n, dim));
  const Workspace ws(n, dim);
  char* base = (char*)workspace;
  SortArgs a{};
  a.ids = ids;
  a.n = n;
  a.vocab = vocab;
  a.padding = padding;
  a.tiles = (int)tiles_of(n);
  a.hist = (uint32_t*)(base + ws.hist);
  a.zero = (ts::u32x4*)grad_weight;
  int passes = 1;
  while ((vocab >> (passes * kDigitBits)) > 0) ++passes;
  // launch i of `launches` writes its share of the zeros, the last one the bytes behind the last whole word
  const int launches = a.tiles <= 1 ? 1 : 2 * passes;
  auto share = [&](int i) {
    a.zero0 = bytes / 16 * i / launches;
    a.zero1 = bytes / 16 * (i + 1) / launches;
    a.tail = (unsigned char*)grad_weight + bytes / 16 * 16;
    a.tail_bytes = i + 1 == launches ? (int)(bytes % 16) : 0;
    const int64_t blocks = std::min<int64_t>((a.zero1 - a.zero0 + kThreads - 1) / kThreads, 4096);
    return dim3((unsigned)(a.tiles + std::max<int64_t>(blocks, 1)));
  };
  if (a.tiles <= 1) {
    a.key_out = (uint32_t*)(base + ws.key[0]);
    a.pos_out = (uint32_t*)(base + ws.pos[0]);
    ts::TimedLaunch timed_("embedding.sort_tile_kernel", s);
    const dim3 grid = share(0);
    hipLaunchKernelGGL(sort_tile_kernel, grid, dim3(kThreads), 0, s, a);
    a.key_in = a.key_out;
    a.pos_in = a.pos_out;
  } else {
    for (int pass = 0; pass < passes; ++pass) {
      a.shift = pass * kDigitBits;
      a.key_out = (uint32_t*)(base + ws.key[pass % 2]);
      a.pos_out = (uint32_t*)(base + ws.pos[pass % 2]);
      {
        ts::TimedLaunch timed_("embedding.sort_count_kernel", s);
        const dim3 grid = share(2 * pass);
        hipLaunchKernelGGL(sort_count_kernel, grid, dim3(kThreads), 0, s, a);
      }
      {
        ts::TimedLaunch timed_("embedding.sort_place_kernel", s);
        const dim3 grid = share(2 * pass + 1);
        hipLaunchKernelGGL(sort_place_kernel, grid, dim3(kThreads), 0, s, a);
      }
      a.ids = nullptr;
      a.key_in = a.key_out;
      a.pos_in = a.pos_out;
    }
  }
  const int st = ts::check_launch("ts_embedding_bwd (sort)");
  if (st != TS_OK || n == 0) return st;
  ReduceArgs r;
  r.key = a.key_in;
  r.pos = a.pos_in;
  r.n = n;
  r.vocab = (uint32_t)vocab;
  r.ldd = ld_grad;
  r.dim = (int)dim;
  r.scale = scale;
  r.chunk = chunk_of(n);
  r.part = (float*)(base + ws.part);
  if (dtype == TS_F32) launch_sums<float>(r, grad_out, grad_weight, s);
  else if (dtype == TS_F16) launch_sums<ts::f16>(r, grad_out, grad_weight, s);
  else launch_sums<ts::bf16>(r, grad_out, grad_weight, s);
  return ts::check_launch("ts_embedding_bwd");
}

}  // extern "C"
