// What the kernels of attention over a paged cache share: their arguments, how a call's work is cut into items, and
// the reads of a page in matrix-instruction layout.
#pragma once

#include "paged.h"
#include "timing.h"

namespace ts {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float neg_inf() { return -__builtin_huge_valf(); }

// Where a sequence's partial rows lie, written by the work-group of its first item: slot (unit0 + slice * tiles
// + tile) * kv_heads + head of its kernel's, `rows` query rows a tile.
struct Plan {
  int32_t unit0, slices, rows, kernel;
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
  int32_t target[2];  // items that a kernel's work is cut into, at least
  Plan* plan;         // [seqs]
  float* part[2];     // of each kernel: [slots][rows][row] unnormalised sums
  float* stats[2];    // [slots][rows][2]: reference point (log2 units) and sum
};

// Items: (sequence, tile of ROWS query rows of a KV head, slice of its keys, KV head).  A slice is as long as cuts all
// of a kernel's keys into `target` of them, about what the device holds at once, or, where these are longer than
// kSliceLong keys, into up to four times as many, so that a last round of them costs less; a multiple of kSliceStep and no
// shorter than kSliceLeast, so that long and short sequences of a batch share the device evenly.  One sequence of 125000
// keys, 8 KV heads: 59 us in 1024 items, 64 in 2048, 76 in 4096; 256 sequences of 256 to 16384: 835, 802 and 780.  Lengths are known on the device alone:
// every wave works the plan out itself, 64 sequences at a time, and takes the item of its work-group.
// Items number at most kv_heads * (keys / slice + tiles); those of sequences with several slices, which leave partial
// rows, at most twice kv_heads * keys / slice (each such sequence has at most twice its length in slices).
constexpr int kSliceStep = 128;
template <int KERNEL> constexpr int kSliceLong = KERNEL == 0 ? 4096 : 2048;
template <int KERNEL> constexpr int kSliceLeast = KERNEL == 0 ? 256 : 512;

struct Item {
  Seq seq;
  int s, head, tile, slice, slices, rows;
  int unit, part;  // among all of the kernel's (tile, slice), and among those that leave partial rows
  int begin, end;  // keys
};

__device__ __forceinline__ int wave_prefix(int x, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  return x;
}

// Keys that a sequence's items go over: a key past the page table ruins the rows that see it, once.
__device__ __forceinline__ int keys_of(const AttnArgs& a, const Seq& q) {
  return (int)min((int64_t)q.len, ((int64_t)a.batch.width << a.page_shift) + 16);
}

template <int KERNEL>
__device__ __forceinline__ int tiles_of(const AttnArgs& a, const Seq& q, int tile_rows) {
  const int64_t rows = (int64_t)q.n * a.group;
  const bool many = a.few_rows > 0 && rows > a.few_rows;
  return many == (KERNEL == 1) ? (int)((rows + tile_rows - 1) / tile_rows) : 0;
}

// The work-group's item; false if it has none, and `past` is then by how many it is past the last.
template <int KERNEL>
__device__ __forceinline__ bool find_item(const AttnArgs& a, int tile_rows, int id, int lane, Item& it, int& past) {
  const Batch& b = a.batch;
  float work = 0.f;  // keys of all tiles; a rounded sum is the same in every wave
  for (int s0 = 0; s0 < b.seqs; s0 += 64)
    if (s0 + lane < b.seqs) {
      const Seq q = seq_of(b, s0 + lane);
      work += (float)keys_of(a, q) * (float)tiles_of<KERNEL>(a, q, tile_rows);
    }
  work = wave_sum(work);
  float each = work * (float)a.kv_heads / (float)a.target[KERNEL];
  each = fmaxf(fminf(each, (float)kSliceLong<KERNEL>), each * 0.25f);
  // read from one lane, as what follows is: uniform to the compiler too, so that pages are looked up by scalar loads
  const int slice = __builtin_amdgcn_readfirstlane(
      max(kSliceLeast<KERNEL>, (int)fminf(each / kSliceStep + 1.f, (float)(kMaxKeys / kSliceStep)) * kSliceStep));
  const int unit = id / a.kv_heads;
  int before = 0, parts_before = 0;
  for (int s0 = 0; s0 < b.seqs; s0 += 64) {
    int slices = 0, count = 0;
    Seq q{0, 0, 0};
    if (s0 + lane < b.seqs) {
      q = seq_of(b, s0 + lane);
      slices = max(1, (keys_of(a, q) + slice - 1) / slice);
      count = tiles_of<KERNEL>(a, q, tile_rows) * slices;
    }
    const int upto = wave_prefix(count, lane) + before;
    const int parts = wave_prefix(slices > 1 ? count : 0, lane) + parts_before;
    const int all = __builtin_amdgcn_readlane(upto, 63);
    if (unit < all) {
      const int at = __ffsll((unsigned long long)__ballot(upto > unit)) - 1;
      it.s = __builtin_amdgcn_readfirstlane(s0 + at);
      it.seq.len = __builtin_amdgcn_readlane(q.len, at);
      it.seq.row0 = __builtin_amdgcn_readlane(q.row0, at);
      it.seq.n = __builtin_amdgcn_readlane(q.n, at);
      it.slices = __builtin_amdgcn_readlane(slices, at);
      it.unit = unit;
      it.head = id - unit * a.kv_heads;
      const int of = __builtin_amdgcn_readlane(count, at);
      const int in = unit - (__builtin_amdgcn_readlane(upto, at) - of);
      it.part = __builtin_amdgcn_readlane(parts, at) - of + in;
      const int tiles = of / it.slices;  // of one slice side by side: they read the same keys
      it.slice = in / tiles;
      it.tile = in - it.slice * tiles;
      it.rows = it.seq.n * a.group;
      const int keys = keys_of(a, it.seq);
      it.begin = min(it.slice * slice, keys);
      it.end = min(it.begin + slice, keys);
      return true;
    }
    before = all;
    parts_before = __builtin_amdgcn_readlane(parts, 63);
  }
  past = id - before * a.kv_heads;
  return false;
}

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
  int64_t items[2];  // at most, of each kernel (0: not launched)
  int64_t slots[2];  // those that leave partial rows
  int64_t rows[2];   // of a tile
  int64_t target[2];
  int64_t bytes;
};
Sizes sizes_of(const ts_paged_cache& c, const ts_paged_batch& b, int64_t tokens, int64_t heads);
void launch_few(const AttnArgs& a, const Sizes& z, int dtype, bool wide, int row, hipStream_t s);
void launch_chunks(const AttnArgs& a, const Sizes& z, int dtype, bool wide, int row, hipStream_t s);

}  // namespace paged
}  // namespace ts
