// Appending keys and values to a paged cache, with the position rotation on the way, for gfx950.
//
//   position of new token i of a sequence's n:  p = length - n + i
//   rotation of a row's first `rotary` elements by the table's row p, cos | sin, in fp32:
//     a' = a cos_j - b sin_j,  b' = b cos_j + a sin_j   for the pairs (a, b) = (x_j, x_{j + rotary/2}),
//     or (x_{2j}, x_{2j+1}) where interleaved
//   query rows are rotated into an output of their own, key rows into the cache; value rows go there as they are
//   8 bits: one scale 2^e, the smallest with most <= 448 * 2^e over the new tokens of a block of 16 tokens and
//   head (in fp16 not below 2^-15), no smaller than before where the block holds older tokens; these are then written by the new scale (a
//   power of two, so that only e4m3's subnormal codes can lose bits).
//
// Bound by HBM where tokens are many (each row is read and written once) and by latency where they
// are few.  One launch: its first work-groups take the blocks of an 8-bit cache, the others rows.  16 prompts of 1024
// tokens, 32 + 2 * 8 heads of 128, 8 bits: 87 us for 370 MB, 4.3 TB/s; a token for each of 64 sequences: 7 us.
#include <algorithm>

#include "paged.h"
#include "timing.h"

namespace ts {
namespace paged {

constexpr int kThreads = 256;
constexpr int kBatch = 4;  // head rows in flight a thread: 37 us for ragged parts of prompts, one at a time 47

int check_cache(const ts_paged_cache* c, const char* what) {
  TS_CHECK_ARG(c && c->key && c->value, "%s: null cache", what);
  TS_CHECK_ARG(c->dtype == TS_F16 || c->dtype == TS_BF16, "%s: cache dtype %d", what, c->dtype);
  TS_CHECK_ARG(c->bits == 8 || c->bits == 16, "%s: a cache of %d bits", what, c->bits);
  TS_CHECK_ARG((c->key_scale && c->value_scale) == (c->bits == 8), "%s: scales of a cache of %d bits", what, c->bits);
  TS_CHECK_ARG(c->row == 64 || c->row == 128 || c->row == 192 || c->row == 256, "%s: rows of %d", what, c->row);
  TS_CHECK_ARG(c->head_dim >= 8 && c->head_dim <= c->row && c->head_dim % 8 == 0, "%s: head dim %d in rows of %d",
               what, c->head_dim, c->row);
  TS_CHECK_ARG(c->page_size >= 16 && c->page_size <= 256 && (c->page_size & (c->page_size - 1)) == 0,
               "%s: pages of %d tokens", what, c->page_size);
  TS_CHECK_ARG(c->kv_heads >= 1 && c->kv_heads <= 1024, "%s: %d KV heads", what, c->kv_heads);
  const int64_t page = (int64_t)c->kv_heads * c->page_size * c->row;
  TS_CHECK_ARG(c->pages >= 0 && c->pages < (1ll << 31) && c->key_page_stride >= page && c->value_page_stride >= page &&
                   c->key_page_stride % 16 == 0 && c->value_page_stride % 16 == 0,
               "%s: %lld pages at strides %lld, %lld", what, (long long)c->pages, (long long)c->key_page_stride,
               (long long)c->value_page_stride);
  TS_CHECK_ARG((((uintptr_t)c->key | (uintptr_t)c->value) & 15) == 0, "%s: cache not 16-byte aligned", what);
  return TS_OK;
}

int check_batch(const ts_paged_batch* b, int64_t tokens, const char* what) {
  TS_CHECK_ARG(b && b->seqs >= 0 && b->seqs <= kMaxSeqs && tokens >= 0 && tokens < kMaxTokens && b->width >= 0 &&
                   b->width < (1ll << 24) && b->ld_table >= 0,
               "%s: bad batch", what);
  TS_CHECK_ARG(b->offsets || b->seqs == tokens, "%s: %lld rows for %lld sequences of one token", what,
               (long long)tokens, (long long)b->seqs);
  TS_CHECK_ARG(b->seqs == 0 || (b->lengths && (b->table || b->width == 0)), "%s: null pointer", what);
  return TS_OK;
}

struct Rows {
  const char* ptr;  // [tokens][heads], rows of head_dim 16-bit elements
  int64_t token_stride, head_stride;
  int32_t heads;
};

struct Args {
  Batch batch;
  Rows query, key, value;
  char* query_out;       // [tokens][heads][head_dim]
  char *key_pages, *value_pages;
  float *key_scale, *value_scale;
  int64_t key_page_stride, value_page_stride;
  const float* rotary;   // [rotary_rows][rotary]
  const int32_t* positions;
  int64_t pages;
  int32_t rotary_rows, rotary_dim;
  int32_t kv_heads, head_dim, row, page_shift;
  int32_t interleaved;
  int32_t block_units;   // work-groups of the first part
  int32_t heads_each;    // head rows a thread of the second part takes
  int64_t row_items;
};

// Chunk pair j of a row (eight elements each): rotated against each other where half-split.
__device__ __forceinline__ void chunk_pair(const Args& a, int j, int& c0, int& c1) {
  const int r = a.rotary_dim >> 4;
  if (a.interleaved || j >= r) {
    c0 = 2 * j;
    c1 = 2 * j + 1;
  } else {
    c0 = j;
    c1 = j + r;
  }
}

// cos and sin of chunk pair j at `pos`; a position past the table gives NaN
__device__ __forceinline__ void angles(const Args& a, int pos, int j, float (&c)[8], float (&s)[8]) {
  if (pos >= 0 && pos < a.rotary_rows) {
    const float* p = a.rotary + (int64_t)pos * a.rotary_dim + 8 * j;
    load8(p, c);
    load8(p + (a.rotary_dim >> 1), s);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = s[i] = __builtin_nanf("");
  }
}

// a c + b s rounded once: what the products and their sum lose is added at the end.  Of the 33.5 million keys of 16 prompts of
// 1024 tokens none goes to another code than in 64 bits; 3 to 8 did where a product was rounded before (87 us, then 85).
__device__ __forceinline__ float rounded_once(float a, float c, float b, float s) {
#pragma clang fp contract(off)
  const float p = a * c, q = b * s, sum = p + q, second = sum - p;
  const float lost = ((p - (sum - second)) + (q - second)) + (__builtin_fmaf(a, c, -p) + __builtin_fmaf(b, s, -q));
  return fabsf(sum) < __builtin_huge_valf() ? sum + lost : sum;
}
template <bool ONCE>
__device__ __forceinline__ void rotate(const Args& a, float (&x)[8], float (&y)[8], const float (&c)[8],
                                       const float (&s)[8]) {
  auto turn = [](float& u, float& v, float cos, float sin) __attribute__((always_inline)) {
    const float p = u, q = v;
    u = ONCE ? rounded_once(p, cos, q, -sin) : p * cos - q * sin;
    v = ONCE ? rounded_once(q, cos, p, sin) : q * cos + p * sin;
  };
  if (a.interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      turn(x[2 * i], x[2 * i + 1], c[i], s[i]);
      turn(y[2 * i], y[2 * i + 1], c[4 + i], s[4 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) turn(x[i], y[i], c[i], s[i]);
  }
}

// The unit-th block of 16 tokens that the call writes: its sequence and the positions
// [first, last] that it gets.  Every wave scans the sequences itself, 64 at a time.
__device__ __forceinline__ bool find_block(const Batch& b, int unit, int lane, int& s, int& first, int& last,
                                           Seq& q) {
  if (!b.offsets) {  // a token each
    if (unit >= b.seqs) return false;
    s = unit;
    q = seq_of(b, s);
    first = last = q.len - 1;
    return q.len > 0;
  }
  int before = 0;
  for (int s0 = 0; s0 < b.seqs; s0 += 64) {
    int count = 0;
    if (s0 + lane < b.seqs) {
      const Seq x = seq_of(b, s0 + lane);
      const int from = max(x.len - x.n, 0);
      count = x.len > from ? ((x.len - 1) >> 4) - (from >> 4) + 1 : 0;
    }
    int upto = count;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(upto, d, 64);
      if (lane >= d) upto += y;
    }
    const int all = __builtin_amdgcn_readlane(upto, 63);
    if (unit < before + all) {
      const uint64_t past = __ballot(before + upto > unit);
      const int at = __ffsll((unsigned long long)past) - 1;
      s = s0 + at;
      const int skip = unit - before - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(count, at));
      q = seq_of(b, s);
      const int from = max(q.len - q.n, 0);
      const int block = (from >> 4) + skip;
      first = max(from, block << 4);
      last = min(q.len - 1, (block << 4) + 15);
      return true;
    }
    before += all;
  }
  return false;
}

// One wave: the new tokens of a block of 16, of one head, of keys or values.
template <typename T, int ROW>
__device__ __forceinline__ void append_block(const Args& a, int unit, int lane) {
  constexpr int kPairs = ROW / 16, kEach = ROW / 64;  // chunk pairs of a row, and of a lane
  const int tensors = 2 * a.kv_heads;
  const int which = unit % tensors, head = which >> 1;
  const bool is_value = which & 1;
  int s, first, last;
  Seq q;
  if (!find_block(a.batch, unit / tensors, lane, s, first, last, q)) return;
  const int page = page_of(a.batch, s, first, a.page_shift, a.pages);
  if (page < 0) return;
  const int page_size = 1 << a.page_shift;
  const int slot0 = first & (page_size - 1), block = slot0 >> 4;
  const Rows& in = is_value ? a.value : a.key;
  char* codes = (is_value ? a.value_pages : a.key_pages) +
                (int64_t)page * (is_value ? a.value_page_stride : a.key_page_stride) +
                ((int64_t)head * page_size + 16 * block) * a.row;
  float* scale = (is_value ? a.value_scale : a.key_scale) + ((int64_t)page * a.kv_heads + head) * (page_size >> 4) + block;
  const int held = first & 15, count = last - first + 1;
  float x[kEach][2][8], most = 0.f;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int item = lane + 64 * k, t = item / kPairs, j = item % kPairs;
    if (t >= count || 16 * j >= a.head_dim) continue;
    const int row = q.row0 + (first + t) - (q.len - q.n);
    int c0, c1;
    chunk_pair(a, j, c0, c1);
    if (is_value) {
      c0 = 2 * j;
      c1 = 2 * j + 1;
    }
    const T* p = (const T*)in.ptr + (int64_t)row * in.token_stride + (int64_t)head * in.head_stride;
    load8(p + 8 * c0, x[k][0]);
    if (8 * c1 < a.head_dim) load8(p + 8 * c1, x[k][1]);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) x[k][1][i] = 0.f;
    if (!is_value && 16 * j < a.rotary_dim) {
      float c[8], sn[8];
      angles(a, a.positions ? a.positions[row] : first + t, j, c, sn);
      // a key on the other side of a border between codes is off by up to 1/8 of its size
      rotate<true>(a, x[k][0], x[k][1], c, sn);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float m = fabsf(x[k][h][i]);
        if (m < __builtin_huge_valf()) most = fmaxf(most, m);
      }
  }
  most = wave_max(most);
  const int old = held ? exponent_of(*scale) : kMinExponent;
  const int e = max(old, exponent_for<T>(most));
  if (held && e > old) {
    // the older tokens by the new scale
    const float ratio = two_to(max(old - e, -126));
    for (int i = lane; i < held * (ROW / 4); i += 64) {
      uint32_t* p = (uint32_t*)codes + i;
      float v[4];
      codes_to_f(*p, v);
      *p = codes4(v[0] * ratio, v[1] * ratio, v[2] * ratio, v[3] * ratio);
    }
  }
  const float inverse = two_to(-e), limit = code_limit<T>(e);
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int item = lane + 64 * k, t = item / kPairs, j = item % kPairs;
    if (t >= count || 16 * j >= a.head_dim) continue;
    int c0, c1;
    chunk_pair(a, j, c0, c1);
    if (is_value) {
      c0 = 2 * j;
      c1 = 2 * j + 1;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = h ? c1 : c0;
      if (8 * c >= a.head_dim) continue;
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = code_value(x[k][h][i], inverse, limit);
      *(u32x2*)(codes + (held + t) * ROW + 8 * c) =
          u32x2{codes4(y[0], y[1], y[2], y[3]), codes4(y[4], y[5], y[6], y[7])};
    }
  }
  if (lane == 0) *scale = two_to(e);
}

// ROW: an 8-bit cache's row, 0 for 16 bits
template <typename T, int ROW>
__global__ __launch_bounds__(kThreads) void append_kernel(Args a) {
  constexpr bool WIDE = ROW == 0;
  const int lane = threadIdx.x & 63;
  if ((int)blockIdx.x < a.block_units) {
    if constexpr (!WIDE) {
      const int unit = (int)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
      append_block<T, ROW>(a, unit, lane);
    }
    return;
  }
  // rows: chunk pair j of every groups-th head row of one token
  const int64_t item = ((int64_t)blockIdx.x - a.block_units) * kThreads + threadIdx.x;
  if (item >= a.row_items) return;
  const int pairs = (a.head_dim + 15) >> 4;
  const int heads = a.query.heads + (WIDE ? 2 * a.kv_heads : 0);
  const int groups = (heads + a.heads_each - 1) / a.heads_each;
  const int j = (int)(item % pairs);
  const int group = (int)(item / pairs % groups), t = (int)(item / ((int64_t)pairs * groups));
  const int s = seq_of_row(a.batch, t);
  int pos = -1, page = -1;
  if (s < a.batch.seqs) {
    const Seq q = seq_of(a.batch, s);
    if (t >= q.row0 && t < q.row0 + q.n) pos = q.len - q.n + (t - q.row0);  // else a row before the first sequence
    if (WIDE && pos >= 0) page = page_of(a.batch, s, pos, a.page_shift, a.pages);
  }
  const int slot = pos & ((1 << a.page_shift) - 1);
  int c0, c1;
  chunk_pair(a, j, c0, c1);
  float c[8], sn[8];
  const bool turns = 16 * j < a.rotary_dim;
  if (turns && pos >= 0) angles(a, a.positions ? a.positions[t] : pos, j, c, sn);
  // kBatch rows are asked for before the first is written
  for (int h0 = group; h0 < heads; h0 += kBatch * groups) {
    u32x4 v0[kBatch], v1[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int h = h0 + k * groups;
      v0[k] = v1[k] = u32x4{0, 0, 0, 0};
      if (h >= heads || pos < 0) continue;  // a row of no sequence
      const bool is_query = h < a.query.heads, is_value = h >= a.query.heads + a.kv_heads;
      const T* p = (const T*)(is_query ? a.query.ptr : is_value ? a.value.ptr : a.key.ptr) +
                   t * (is_query ? a.query.token_stride : is_value ? a.value.token_stride : a.key.token_stride) +
                   (is_query ? h : (h - a.query.heads) % a.kv_heads) *
                       (is_query ? a.query.head_stride : is_value ? a.value.head_stride : a.key.head_stride);
      const int b0 = is_value ? 2 * j : c0, b1 = is_value ? 2 * j + 1 : c1;
      v0[k] = *(const u32x4*)(p + 8 * b0);
      if (8 * b1 < a.head_dim) v1[k] = *(const u32x4*)(p + 8 * b1);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int h = h0 + k * groups;
      if (h >= heads) continue;
      const bool is_query = h < a.query.heads, is_value = h >= a.query.heads + a.kv_heads;
      if (!is_query && page < 0) continue;
      const int head = is_query ? h : (h - a.query.heads) % a.kv_heads;
      T* o = is_query ? (T*)a.query_out + ((int64_t)t * a.query.heads + head) * a.head_dim
                      : (T*)(is_value ? a.value_pages : a.key_pages) +
                            (int64_t)page * (is_value ? a.value_page_stride : a.key_page_stride) +
                            (((int64_t)head << a.page_shift) + slot) * a.row;
      const int b0 = is_value ? 2 * j : c0, b1 = is_value ? 2 * j + 1 : c1;
      if (turns && !is_value && pos >= 0) {
        float x[8], y[8];
        load8((const T*)&v0[k], x);
        load8((const T*)&v1[k], y);
        rotate<false>(a, x, y, c, sn);
        store8((T*)&v0[k], x);
        store8((T*)&v1[k], y);
      }
      *(u32x4*)(o + 8 * b0) = v0[k];
      if (8 * b1 < a.head_dim) *(u32x4*)(o + 8 * b1) = v1[k];
    }
  }
}

// What the codes stand for, eight of a row a thread: 100 MB in 23 us, 4.3 TB/s.
template <typename T>
__global__ __launch_bounds__(kThreads) void values_kernel(const char* key, const char* value, const float* key_scale,
                                                          const float* value_scale, int64_t key_stride,
                                                          int64_t value_stride, char* key_out, char* value_out,
                                                          int64_t items, int chunks, int head_dim, int row,
                                                          int heads_page) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < 2 * items; i += (int64_t)gridDim.x * kThreads) {
    const bool is_value = i >= items;
    const int64_t at = is_value ? i - items : i;
    const int c = (int)(at % chunks);
    const int64_t line = at / chunks;  // (page, head, token)
    const int64_t page = line / heads_page;
    const int in_page = (int)(line - page * heads_page);
    const char* p = (is_value ? value : key) + page * (is_value ? value_stride : key_stride) + (int64_t)in_page * row + 8 * c;
    const u32x2 v = *(const u32x2*)p;
    const float s = (is_value ? value_scale : key_scale)[line >> 4];
    *(u32x4*)((is_value ? value_out : key_out) + (line * head_dim + 8 * c) * 2) =
        u32x4{widen2<T, false>(v[0], s), widen2<T, true>(v[0], s), widen2<T, false>(v[1], s), widen2<T, true>(v[1], s)};
  }
}

}  // namespace paged
}  // namespace ts

extern "C" {

int ts_paged_append(const ts_paged_cache* cache, const ts_paged_batch* batch, int64_t tokens, const void* query,
                    int64_t query_token_stride, int64_t query_head_stride, int64_t heads, void* query_out,
                    const void* key, int64_t key_token_stride, int64_t key_head_stride, const void* value,
                    int64_t value_token_stride, int64_t value_head_stride, const float* rotary, int64_t rotary_rows,
                    int64_t rotary_dim, int interleaved, const int32_t* positions, void* stream) {
  using namespace ts::paged;
  if (int e = check_cache(cache, "ts_paged_append")) return e;
  if (int e = check_batch(batch, tokens, "ts_paged_append")) return e;
  TS_CHECK_ARG(heads >= 0 && heads <= (1 << 16), "ts_paged_append: %lld query heads", (long long)heads);
  TS_CHECK_ARG(rotary_dim >= 0 && rotary_dim <= cache->head_dim && rotary_dim % 16 == 0 &&
                   (rotary_dim == 0 || (rotary && rotary_rows >= 0 && rotary_rows < (1ll << 31))),
               "ts_paged_append: rotation of %lld of %d elements", (long long)rotary_dim, cache->head_dim);
  if (tokens == 0) return TS_OK;
  TS_CHECK_ARG(key && value && (heads == 0 || (query && query_out)), "ts_paged_append: null pointer");
  TS_CHECK_ARG((((uintptr_t)query | (uintptr_t)query_out | (uintptr_t)key | (uintptr_t)value | (uintptr_t)rotary) & 15) == 0 &&
                   (query_token_stride | query_head_stride | key_token_stride | key_head_stride | value_token_stride |
                    value_head_stride) % 8 == 0,
               "ts_paged_append: rows not 16-byte aligned");
  Args a{};
  a.batch = batch_of(*batch, tokens);
  a.query = Rows{(const char*)query, query_token_stride, query_head_stride, (int32_t)heads};
  a.key = Rows{(const char*)key, key_token_stride, key_head_stride, cache->kv_heads};
  a.value = Rows{(const char*)value, value_token_stride, value_head_stride, cache->kv_heads};
  a.query_out = (char*)query_out;
  a.key_pages = (char*)cache->key;
  a.value_pages = (char*)cache->value;
  a.key_scale = cache->key_scale;
  a.value_scale = cache->value_scale;
  a.key_page_stride = cache->key_page_stride;
  a.value_page_stride = cache->value_page_stride;
  a.rotary = rotary;
  a.rotary_rows = (int32_t)rotary_rows;
  a.rotary_dim = (int32_t)rotary_dim;
  a.positions = positions;
  a.pages = cache->pages;
  a.kv_heads = cache->kv_heads;
  a.head_dim = cache->head_dim;
  a.row = cache->row;
  a.page_shift = shift_of(cache->page_size);
  a.interleaved = interleaved;
  const bool wide = cache->bits == 16;
  // blocks of 16 tokens that n tokens of a sequence touch: at most n / 16 + 2, and n
  const int64_t blocks = wide ? 0 : std::min(tokens, tokens / 16 + 2 * batch->seqs);
  const int64_t block_units = (blocks * 2 * cache->kv_heads + kThreads / 64 - 1) / (kThreads / 64);
  const int64_t rows = heads + (wide ? 2 * cache->kv_heads : 0);
  const int64_t pairs = (cache->head_dim + 15) / 16;
  // Threads take as many head rows of a token as leave about 2^18 of them: the angles are loaded once for these.
  a.heads_each = (int32_t)std::max<int64_t>(1, std::min<int64_t>(8, tokens * rows * pairs >> 18));
  a.row_items = tokens * pairs * ((rows + a.heads_each - 1) / a.heads_each);
  const int64_t grid = block_units + (a.row_items + kThreads - 1) / kThreads;
  TS_CHECK_ARG(grid < (1 << 24), "ts_paged_append: %lld tokens of %lld heads: grid too large", (long long)tokens,
               (long long)(heads + 2 * cache->kv_heads));
  a.block_units = (int32_t)block_units;
  if (grid == 0) return TS_OK;
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("paged.append_kernel", s);
    switch (wide ? 0 : cache->row) {
      case 0: TS_LAUNCH_E_T(cache->dtype, append_kernel, 0, dim3((unsigned)grid), dim3(kThreads), 0, s, a); break;
      case 64: TS_LAUNCH_E_T(cache->dtype, append_kernel, 64, dim3((unsigned)grid), dim3(kThreads), 0, s, a); break;
      case 128: TS_LAUNCH_E_T(cache->dtype, append_kernel, 128, dim3((unsigned)grid), dim3(kThreads), 0, s, a); break;
      case 192: TS_LAUNCH_E_T(cache->dtype, append_kernel, 192, dim3((unsigned)grid), dim3(kThreads), 0, s, a); break;
      default: TS_LAUNCH_E_T(cache->dtype, append_kernel, 256, dim3((unsigned)grid), dim3(kThreads), 0, s, a);
    }
  }
  return ts::check_launch("ts_paged_append");
}

int ts_paged_values(const ts_paged_cache* cache, void* key_out, void* value_out, void* stream) {
  using namespace ts::paged;
  if (int e = check_cache(cache, "ts_paged_values")) return e;
  TS_CHECK_ARG(cache->bits == 8, "ts_paged_values: a 16-bit cache holds its values");
  const int heads_page = cache->kv_heads * cache->page_size, chunks = cache->head_dim / 8;
  const int64_t items = cache->pages * heads_page * chunks;
  if (items == 0) return TS_OK;
  TS_CHECK_ARG(key_out && value_out && (((uintptr_t)key_out | (uintptr_t)value_out) & 15) == 0,
               "ts_paged_values: outputs null or not 16-byte aligned");
  const int64_t grid = std::min<int64_t>((2 * items + kThreads - 1) / kThreads, 1 << 20);
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("paged.values_kernel", s);
    TS_LAUNCH_E(cache->dtype, values_kernel, dim3((unsigned)grid), dim3(kThreads), 0, s, (const char*)cache->key,
                (const char*)cache->value, cache->key_scale, cache->value_scale, cache->key_page_stride,
                cache->value_page_stride, (char*)key_out, (char*)value_out, items, chunks, cache->head_dim, cache->row,
                heads_page);
  }
  return ts::check_launch("ts_paged_values");
}

}  // extern "C"
