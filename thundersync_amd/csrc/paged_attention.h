// What the kernels of attention over a paged cache share: their arguments, how a call's work is cut into items, and
// the reads of a page in matrix-instruction layout.
#pragma once

#include "paged.h"
#include "timing.h"

namespace ts {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float neg_inf() { return -__builtin_huge_valf(); }

// Where a sequence's work lies in its kernel's, written by the work-group that begins it.
struct Plan {
  int32_t start, blocks;  // of its first tile, and of each tile
  int32_t per;            // blocks of a work-group
  int32_t kernel;
};
constexpr int64_t kMaxKeys = 1 << 30;  // of a sequence

struct AttnArgs {
  Batch batch;
  const char* query;  // rows of head_dim elements
  int64_t token_stride, head_stride;
  char* out;          // [tokens][heads][head_dim]
  const char *key, *value;
  const float *key_scale, *value_scale;
  int64_t key_page_stride, value_page_stride;  // bytes
  int64_t pages;
  float scale;        // log2 units
  int32_t heads, kv_heads, group, head_dim, page_shift;
  int32_t few_rows;   // sequences of more query rows (tokens x group) are the chunk kernel's; 0: none are
  int32_t jobs[2];    // work-groups of each KV head that a kernel's work is dealt to, at least
  int32_t tile_rows[2];
  int64_t slots[2];
  Plan* plan;         // [seqs], or null where no tile can be cut
  float* part[2];     // of each kernel: [slots][rows][row] unnormalised sums
  float* stats[2];    // [slots][rows][2]: reference point (log2 units) and sum
};

// The kernel's only argument, read from its segment where it is used: over a loop of tiles its 50 words would not fit
// the scalar registers beside the tile's own.
__device__ __forceinline__ AttnArgs arguments() {
  typedef const __attribute__((address_space(4))) uint32_t* Words;
  Words p = (Words)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  uint32_t w[sizeof(AttnArgs) / 4];
#pragma unroll
  for (int i = 0; i < (int)(sizeof(AttnArgs) / 4); ++i) w[i] = p[i];
  AttnArgs a;
  __builtin_memcpy(&a, w, sizeof(a));
  // known to be global memory again: reads through pointers that may be any kind wait for LDS too
  auto global = [](auto*& x) __attribute__((always_inline)) {
    typedef std::remove_reference_t<decltype(*x)> E;
    x = (E*)(__attribute__((address_space(1))) E*)(uint64_t)x;
  };
  global(a.batch.table);
  global(a.batch.lengths);
  global(a.batch.offsets);
  global(a.query);
  global(a.out);
  global(a.key);
  global(a.value);
  global(a.key_scale);
  global(a.value_scale);
  global(a.plan);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    global(a.part[i]);
    global(a.stats[i]);
  }
  return a;
}

// How a kernel's work is dealt out.  A tile (query rows of one KV head, of one sequence) is kTileCost blocks for its
// start and end and one for each kBlockKeys keys; a KV head's tiles follow one another, and each of its work-groups
// takes as many blocks in a row, ending tiles and beginning others on the way, so that all end together however lengths
// differ.  A tile that a border cuts leaves partial rows: slot 2 j of work-group j where it began before, 2 j + 1 where it
// ends behind.  Work-groups are as many as the device holds at once, and fewer where they would get less than kLeast
// blocks.  64 sequences of 100 to 6000 keys, 24/4 heads of 256, five rows each: 132 us in slices of equal length a sequence,
// 114 dealt like this; 128 of 8192, 32/8 heads of 128: 370 us, 411 dealt to four times as many.
//
// Lengths are known on the device alone: every work-group works its part out itself, 64 sequences at a time.
constexpr int kBlockKeys = 128, kTileCost = 3;
template <int KERNEL> constexpr int kLeast = KERNEL == 0 ? 4 : 5;
// Waves a SIMD: a step's loads and the accumulators are 3 ROW / 8 registers, of 16 bits 5 ROW / 8, and one wave fewer
// with nothing spilled is faster (rows of 128: 256 sequences of 256 to 16384 keys 737 us at three, 796 at four; 16 bits, 64
// of 100 to 6000: 151 us at two, 161 at three).
__host__ __device__ constexpr int few_occupancy(bool wide, int row, int tiles) {
  const int size = row * tiles;
  return size <= 64 ? 3 : wide ? 2 : size <= 128 ? 3 : 2;
}
__host__ __device__ constexpr int chunk_occupancy(int row) { return row <= 64 ? 4 : 2; }

__device__ __forceinline__ int wave_prefix(int x, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  return x;
}

// Keys that a sequence's tiles go over: a key past the page table ruins the rows that see it, once.
__device__ __forceinline__ int keys_of(const AttnArgs& a, const Seq& q) {
  return (int)min((int64_t)q.len, ((int64_t)a.batch.width << a.page_shift) + 16);
}
__device__ __forceinline__ int blocks_of(const AttnArgs& a, const Seq& q) {
  return kTileCost + (int)((uint32_t)(keys_of(a, q) + kBlockKeys - 1) / kBlockKeys);
}
template <int KERNEL>
__device__ __forceinline__ int tiles_of(const AttnArgs& a, const Seq& q, int tile_rows) {
  const int64_t rows = (int64_t)q.n * a.group;
  const bool many = a.few_rows > 0 && rows > a.few_rows;
  return many == (KERNEL == 1) ? (int)((rows + tile_rows - 1) / tile_rows) : 0;
}
// A border less than kSnap blocks inside a tile moves to the nearer end of it: a tile that is cut costs a start, an end
// and a partial tile more.
constexpr int kSnap = 4;
__device__ __forceinline__ int snapped(int border, int in_tile, int blocks) {
  if (2 * in_tile <= blocks) return in_tile < kSnap ? border - in_tile : border;
  return blocks - in_tile < kSnap ? border + blocks - in_tile : border;
}

// A work-group's place in its kernel's work.  Everything is read from one lane, so that it is uniform to the compiler
// too and pages are looked up by scalar loads.
template <int KERNEL> struct Cursor {
  Seq seq;
  int s, tile, tiles, blocks;  // of the sequence
  int from;                    // block of the tile
  int left;                    // blocks of the work-group
  int per, job, head;
  int end;                     // of the work-group's blocks

  // false if the work-group has none; `past` is then by how many it is past the last that has
  __device__ __forceinline__ bool begin(const AttnArgs& a, int tile_rows, int id, int lane, int& past) {
    const Batch& b = a.batch;
    // the first 64 sequences are read once
    Seq q{0, 0, 0};
    int count = 0;
    auto read = [&](int s0) __attribute__((always_inline)) {
      count = 0;
      if (s0 + lane < b.seqs) {
        q = seq_of(b, s0 + lane);
        count = tiles_of<KERNEL>(a, q, tile_rows) * blocks_of(a, q);
      }
    };
    int total = 0;
    for (int s0 = (b.seqs - 1) & ~63; s0 >= 0; s0 -= 64) {
      read(s0);
      total += count;
    }
    total = __builtin_amdgcn_readlane(wave_prefix(total, lane), 63);
    per = max((int)((uint32_t)(total + a.jobs[KERNEL] - 1) / (uint32_t)a.jobs[KERNEL]), kLeast<KERNEL>);
    job = (uint32_t)id / (uint32_t)a.kv_heads;
    head = id - job * a.kv_heads;
    const int used = (uint32_t)(total + per - 1) / (uint32_t)per;
    past = id - used * a.kv_heads;
    if (job >= used) return false;
    const int borders[2] = {job * per, min((job + 1) * per, total)};
    int start = 0, stop = borders[1] == total ? total : 0, before = 0;
    bool found = false;
    for (int s0 = 0; s0 < b.seqs; s0 += 64) {
      if (s0 > 0) read(s0);
      const int upto = wave_prefix(count, lane) + before;
      const int all = __builtin_amdgcn_readlane(upto, 63);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int border = borders[k];
        if (border < before || border >= all) continue;
        const int at = __ffsll((unsigned long long)__ballot(upto > border)) - 1;
        const int size = __builtin_amdgcn_readlane(blocks_of(a, q), at);
        const int in = border - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(count, at));
        const int nth = (uint32_t)in / (uint32_t)size, x = in - nth * size, to = snapped(border, x, size);
        if (k == 1) {
          stop = to;
          continue;
        }
        start = to;
        enter(a, tile_rows, s0, at, q);
        tile = nth;
        from = x + to - border;
        found = true;
      }
      if (found && stop > 0) break;
      before = all;
    }
    end = stop;
    left = stop - start;
    if (!found || left <= 0) {
      past = -1;  // nothing, but rows behind the last sequence are others'
      return false;
    }
    if (from == blocks) {
      from = 0;
      if (++tile >= tiles && !skip(a, tile_rows, lane)) return false;
    }
    return true;
  }
  // One wave finds the work-group's place and the next tile and the others read it in LDS, where it is also kept while a
  // tile is computed, for scalar registers are short.
  struct Kept {
    int word[12 + 4];
  };
  __device__ __forceinline__ void put(Kept& to, bool some, int past) const {
    static_assert(sizeof(Cursor) <= sizeof(int) * 14, "a cursor and two words");
    if (threadIdx.x == 0) {
      __builtin_memcpy(to.word, this, sizeof(Cursor));
      to.word[14] = some;
      to.word[15] = past;
    }
  }
  __device__ __forceinline__ bool take(const Kept& kept, int* past = nullptr) {
    asm volatile("" ::: "memory");
    int w[sizeof(Cursor) / 4];
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Cursor) / 4); ++i) w[i] = __builtin_amdgcn_readfirstlane(kept.word[i]);
    __builtin_memcpy(this, w, sizeof(Cursor));
    if (past) *past = __builtin_amdgcn_readfirstlane(kept.word[15]);
    return __builtin_amdgcn_readfirstlane(kept.word[14]) != 0;
  }
  // the sequence that lane `at` of a chunk of 64 has read
  __device__ __forceinline__ void enter(const AttnArgs& a, int tile_rows, int s0, int at, const Seq& q) {
    s = s0 + __builtin_amdgcn_readfirstlane(at);
    seq.len = __builtin_amdgcn_readlane(q.len, at);
    seq.row0 = __builtin_amdgcn_readlane(q.row0, at);
    seq.n = __builtin_amdgcn_readlane(q.n, at);
    tiles = tiles_of<KERNEL>(a, seq, tile_rows);
    blocks = blocks_of(a, seq);
    tile = from = 0;
  }
  // The keys of the tile that are the work-group's; whether it has all of it; else the slot of its partial rows.
  __device__ __forceinline__ void piece(const AttnArgs& a, int& begin, int& end) const {
    const int keys = keys_of(a, seq);
    begin = min(keys, max(from - kTileCost, 0) * kBlockKeys);
    end = min(keys, max(min(blocks, from + left) - kTileCost, 0) * kBlockKeys);
  }
  __device__ __forceinline__ bool whole() const { return from == 0 && left >= blocks; }
  __device__ __forceinline__ int slot(int kv_heads) const { return (2 * job + (from == 0)) * kv_heads + head; }
  // To the next tile; false at the work-group's end.
  __device__ __forceinline__ bool next(const AttnArgs& a, int tile_rows, int lane) {
    left -= min(blocks, from + left) - from;
    if (left <= 0) return false;
    from = 0;
    return ++tile < tiles || skip(a, tile_rows, lane);
  }
  // To the next sequence that has tiles.
  __device__ __forceinline__ bool skip(const AttnArgs& a, int tile_rows, int lane) {
    for (int s0 = s + 1; s0 < a.batch.seqs; s0 += 64) {
      Seq q{0, 0, 0};
      if (s0 + lane < a.batch.seqs) q = seq_of(a.batch, s0 + lane);
      const uint64_t which = __ballot(tiles_of<KERNEL>(a, q, tile_rows) > 0);
      if (which) {
        enter(a, tile_rows, s0, __ffsll((unsigned long long)which) - 1, q);
        return true;
      }
    }
    return false;
  }
};

// Weights are rounded to the element type for the product with the values, half a step each, as in packed attention: in fp32
// there is no matrix instruction of this rate.  That is 1.4e-3 of an output's size in bf16 and 1.4e-4 in fp16, beside 1.7e-3
// and 2.1e-4 of the output's own rounding.  Their sum is of the unrounded ones, in fp32.  A row's reference point is its
// largest score when it last moved, in fp16 kLift below it: weights go up to 2^(kLift + kSlack), below 65504, and half of
// fp16's smallest number is 2^-32 of the largest, not 2^-25, which many small weights beside a large one would be lost to.
constexpr float kSlack = 8.f;  // log2 units by which scores may pass the largest before the reference point moves
template <typename T> constexpr float kLift = std::is_same_v<T, f16> ? 7.f : 0.f;
template <typename T> constexpr float kSlackSum = std::is_same_v<T, f16> ? 32768.f : 256.f;  // 2^(kLift + kSlack)

// Two 16-bit values without those that are not finite, and ones in the place of these.
template <typename T> constexpr uint32_t kOneOf = std::is_same_v<T, f16> ? 0x3c00u : 0x3f80u;
template <typename T> __device__ __forceinline__ void split_finite(uint32_t x, uint32_t& fine, uint32_t& flag) {
  constexpr uint32_t top = std::is_same_v<T, f16> ? 0x7c00u : 0x7f80u;
  const bool lo = (x & top) == top, hi = (x >> 16 & top) == top;
  fine = (lo ? 0u : x & 0xffffu) | (hi ? 0u : x & 0xffff0000u);
  flag = (lo ? kOneOf<T> : 0u) | (hi ? kOneOf<T> << 16 : 0u);
}

// host side
struct Sizes {
  int64_t groups[2];  // work-groups of each kernel, at most (0: not launched)
  int64_t slots[2];   // partial tiles, at most
  int64_t rows[2];    // of a tile
  int64_t jobs[2];
  int64_t blocks[2];  // of a KV head, at most
  int64_t bytes;
};
Sizes sizes_of(const ts_paged_cache& c, const ts_paged_batch& b, int64_t tokens, int64_t heads);
void launch_few(const AttnArgs& a, const Sizes& z, int dtype, bool wide, int row, hipStream_t s);
void launch_chunks(const AttnArgs& a, const Sizes& z, int dtype, bool wide, int row, hipStream_t s);

}  // namespace paged
}  // namespace ts
