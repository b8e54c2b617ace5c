// Attention of a call's rows over the keys of a paged cache, for gfx950: the entry, and the join of partial rows.
//
//   row of new token i of a sequence's n, query head h: o = sum_k w_k v_k / sum_k w_k, w_k = exp(scale q . k_k - m),
//   over the keys of KV head h / group at positions 0 .. length - n + i; a row without keys is zero
//
// paged_attention_few.hip takes the sequences with few query rows, paged_attention_chunk.hip those with many.
#include <algorithm>

#include "paged_attention.h"

namespace ts {
namespace paged {

// Where the partial rows of one row (token t, query head h) lie: part p at place(p).  parts is 1 where there is nothing to
// join: the row has been written.
struct Parts {
  const float *part, *stats;
  int owner, inner, parts, rows, at;  // at: the row of its tile, of its KV head
  int kv_heads, head;

  __device__ __forceinline__ int64_t place(int p) const {
    return ((int64_t)(p == 0 ? 2 * owner + 1 : 2 * (inner + p - 1)) * kv_heads + head) * rows + at;
  }
};
__device__ __forceinline__ Parts parts_of(const AttnArgs& a, int t, int h, int s) {
  bool mine = s < a.batch.seqs;
  Seq q{0, 0, 0};
  if (mine) q = seq_of(a.batch, s);
  mine = mine && t >= q.row0 && t < q.row0 + q.n;
  Plan plan{0, 1, 1, 0};
  if (mine) plan = a.plan[s];
  // a plan that no work-group wrote (lengths or offsets changed under the call) reads nothing out of the workspace
  mine = mine && plan.per > 0 && plan.blocks > 0 && plan.start >= 0 && (plan.kernel & ~1) == 0;
  if (!mine) plan = Plan{0, 1, 1, 0};
  Parts y;
  y.rows = plan.kernel ? a.tile_rows[1] : a.tile_rows[0];
  y.kv_heads = a.kv_heads;
  y.head = h / a.group;
  const int row = (t - q.row0) * a.group + h % a.group, tile = row / y.rows;
  y.at = row - tile * y.rows;
  // the work-group that begins the tile: the last whose border lies before it or has moved to its start; those that begin
  // inside, from `inner` on: their borders have not moved
  const int first = plan.start + tile * plan.blocks, last = first + plan.blocks;
  y.owner = (first + min(kSnap - 1, plan.blocks / 2)) / plan.per;
  y.inner = (first + kSnap + plan.per - 1) / plan.per;
  y.parts = mine ? 1 + max(0, (last - kSnap) / plan.per - y.inner + 1) : 1;
  const int64_t slots = plan.kernel ? a.slots[1] : a.slots[0];
  if (min(y.owner, y.inner) < 0 || ((int64_t)max(y.owner, y.inner + y.parts - 2) + 1) * 2 * a.kv_heads > slots) y.parts = 1;
  y.part = plan.kernel ? a.part[1] : a.part[0];
  y.stats = plan.kernel ? a.stats[1] : a.stats[0];
  return y;
}

// o = sum_p acc_p 2^(m_p - M) / sum_p l_p 2^(m_p - M) over a row's parts in order, M the largest m.
//
// Few rows: WAVES waves a row, each every WAVES-th part, then the waves in order.
template <typename T, int ROW, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void merge_kernel(AttnArgs a) {
  constexpr int N = ROW / 64;
  __shared__ float s_acc[WAVES][ROW], s_sum[WAVES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = (int)blockIdx.x / a.heads, h = (int)blockIdx.x - t * a.heads;
  const Parts y = parts_of(a, t, h, __builtin_amdgcn_readfirstlane(seq_of_row(a.batch, t)));
  if (y.parts <= 1) return;
  float acc[N], sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  float most = neg_inf();
  for (int p = lane; p < y.parts; p += 64) most = fmaxf(most, y.stats[2 * y.place(p)]);
  most = wave_max(most);
  const float ref = most == neg_inf() ? 0.f : most;
#pragma unroll 4
  for (int p = wave; p < y.parts; p += WAVES) {
    const int64_t at = y.place(p);
    const float w = fast_exp2(y.stats[2 * at] - ref);
    sum = fmaf(y.stats[2 * at + 1], w, sum);
    const float* x = y.part + at * ROW + N * lane;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = fmaf(x[i], w, acc[i]);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) s_acc[wave][N * lane + i] = acc[i];
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= a.head_dim) return;
  float l = 0.f, o = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    l += s_sum[w];
    o += s_acc[w][d];
  }
  ((T*)a.out)[((int64_t)t * a.heads + h) * a.head_dim + d] = from_f<T>(o * (l > 0.f ? 1.f / l : 0.f));
}

// Many rows: 16 lanes a row.
constexpr int kMergeLanes = 16, kMergeThreads = 256;
template <typename T, int ROW>
__global__ __launch_bounds__(kMergeThreads) void merge_kernel(AttnArgs a) {
  constexpr int N = ROW / kMergeLanes;
  const int lane = threadIdx.x % kMergeLanes;
  const int id = ((int)blockIdx.x * kMergeThreads + (int)threadIdx.x) / kMergeLanes;
  const int t = (uint32_t)id / (uint32_t)a.heads, h = id - t * a.heads;
  const Parts y = parts_of(a, t, h, t < a.batch.tokens ? seq_of_row(a.batch, t) : a.batch.seqs);
  const int parts = y.parts > 1 ? y.parts : 0;
  float most = neg_inf();
  for (int p = lane; p < parts; p += kMergeLanes) most = fmaxf(most, y.stats[2 * y.place(p)]);
#pragma unroll
  for (int d = 1; d < kMergeLanes; d <<= 1) most = fmaxf(most, __shfl_xor(most, d, 64));
  if (parts == 0) return;
  const float ref = most == neg_inf() ? 0.f : most;
  f32x4 acc[N / 4];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < N / 4; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int p = 0; p < parts; ++p) {
    const int64_t at = y.place(p);
    const float w = fast_exp2(y.stats[2 * at] - ref);
    sum = fmaf(y.stats[2 * at + 1], w, sum);
    const f32x4* x = (const f32x4*)(y.part + at * ROW + N * lane);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const f32x4 v = x[i];
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[i][k] = fmaf(v[k], w, acc[i][k]);
    }
  }
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
  T* out = (T*)a.out + ((int64_t)t * a.heads + h) * a.head_dim + N * lane;
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    if (N * lane + 4 * i >= a.head_dim) continue;
    T v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = from_f<T>(acc[i][k] * inv);
    __builtin_memcpy(__builtin_assume_aligned(out + 4 * i, 8), v, 8);
  }
}

// Sixteen waves a row where rows are few and may have many parts, 16 lanes where they are many: 32 rows of 123 parts 7.7 us
// (four waves 9.8), 768 of a few parts 6.2 (sixteen waves 8.7), 65536 of three 17.5, 4.9 TB/s (a wave a row 39).
constexpr int64_t kFewMerged = 64, kManyMerged = 2048;
template <typename T, int ROW> void launch_merge(const AttnArgs& a, hipStream_t s) {
  ts::TimedLaunch timed_("paged.merge_kernel", s);
  const int64_t rows = (int64_t)a.batch.tokens * a.heads;
  if (rows <= kFewMerged) hipLaunchKernelGGL((merge_kernel<T, ROW, 16>), dim3((unsigned)rows), dim3(1024), 0, s, a);
  else if (rows < kManyMerged) hipLaunchKernelGGL((merge_kernel<T, ROW, 4>), dim3((unsigned)rows), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((merge_kernel<T, ROW>), dim3((unsigned)((rows + 15) / 16)), dim3(kMergeThreads), 0, s, a);
}
template <typename T> void launch_merge(const AttnArgs& a, int row, hipStream_t s) {
  switch (row) {
    case 64: launch_merge<T, 64>(a, s); break;
    case 128: launch_merge<T, 128>(a, s); break;
    case 192: launch_merge<T, 192>(a, s); break;
    default: launch_merge<T, 256>(a, s);
  }
}

// Sequences of up to 32 query rows a KV head are the few kernel's.
constexpr int kFewRows = 32;

Sizes sizes_of(const ts_paged_cache& c, const ts_paged_batch& b, int64_t tokens, int64_t heads) {
  Sizes z{};
  const int64_t group = heads / c.kv_heads, keys = b.width * c.page_size + 16;
  const bool ragged = b.offsets != nullptr, chunks = ragged && tokens * group > kFewRows;
  // 32 rows a tile would not fit the registers beside wide rows' loads: their sequences of more than 16 rows are read twice
  z.rows[0] = (ragged || group > 16) && c.row <= 128 ? 32 : 16;
  z.rows[1] = 128;
  // work-groups of a KV head that the device's 256 CUs hold at once (four waves each, eight of chunks of 256-wide rows)
  const int64_t held[2] = {256 * few_occupancy(c.bits == 16, c.row, (int)z.rows[0] / 16),
                           256 * chunk_occupancy(c.row) / (c.row > 192 ? 2 : 1)};
  for (int k = 0; k < 2; ++k) z.jobs[k] = std::max<int64_t>(1, held[k] / c.kv_heads);
  const int64_t seqs = std::min(b.seqs, tokens);
  const int64_t tiles[2] = {
      !ragged ? seqs * ((group + z.rows[0] - 1) / z.rows[0]) : seqs * (kFewRows / z.rows[0]),
      chunks ? tokens * group / z.rows[1] + std::min(seqs, tokens * group / (kFewRows + 1)) : 0};
  int64_t plan = 0;
  for (int k = 0; k < 2; ++k) {
    z.blocks[k] = tiles[k] * (kTileCost + (keys + kBlockKeys - 1) / kBlockKeys);
    const int64_t least = k ? kLeast<1> : kLeast<0>;
    const int64_t jobs = std::min((z.blocks[k] + least - 1) / least, z.jobs[k]);
    z.groups[k] = jobs * c.kv_heads;
    z.slots[k] = jobs > 1 ? 2 * z.groups[k] : 0;
    if (z.slots[k]) plan = (b.seqs * (int64_t)sizeof(Plan) + 255) / 256 * 256;
    z.bytes += z.slots[k] * z.rows[k] * (c.row + 2) * 4;
  }
  z.bytes += plan;
  return z;
}

}  // namespace paged
}  // namespace ts

extern "C" {

int64_t ts_paged_attention_workspace(const ts_paged_cache* cache, const ts_paged_batch* batch, int64_t tokens,
                                     int64_t heads) {
  using namespace ts::paged;
  if (check_cache(cache, "ts_paged_attention_workspace") || check_batch(batch, tokens, "ts_paged_attention_workspace") ||
      heads < 1 || heads % cache->kv_heads)
    return 0;
  return sizes_of(*cache, *batch, tokens, heads).bytes;
}

int ts_paged_attention(const ts_paged_cache* cache, const ts_paged_batch* batch, int64_t tokens, const void* query,
                       int64_t token_stride, int64_t head_stride, int64_t heads, float scale, void* out,
                       void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace ts::paged;
  if (int e = check_cache(cache, "ts_paged_attention")) return e;
  if (int e = check_batch(batch, tokens, "ts_paged_attention")) return e;
  TS_CHECK_ARG(heads >= 1 && heads <= (1 << 16) && heads % cache->kv_heads == 0, "ts_paged_attention: %lld heads over %d",
               (long long)heads, cache->kv_heads);
  TS_CHECK_ARG(__builtin_isfinite(scale * kLog2e), "ts_paged_attention: scale %g", (double)scale);
  if (tokens == 0) return TS_OK;
  TS_CHECK_ARG(query && out && cache->pages > 0, "ts_paged_attention: null pointer, or a cache without pages");
  TS_CHECK_ARG((((uintptr_t)query | (uintptr_t)out) & 15) == 0 && (token_stride | head_stride) % 8 == 0,
               "ts_paged_attention: rows not 16-byte aligned");
  const Sizes z = sizes_of(*cache, *batch, tokens, heads);
  // 2^24 work-groups of 256 threads wrap a launch; blocks are counted in 32 bits
  TS_CHECK_ARG(tokens * heads < (1ll << 24) && std::max(z.groups[0], z.groups[1]) + tokens / 16 < (1ll << 23) &&
                   batch->width * cache->page_size <= kMaxKeys && std::max(z.blocks[0], z.blocks[1]) < (1ll << 30),
               "ts_paged_attention: %lld rows of %lld heads over %lld sequences of %lld pages: too large", (long long)tokens,
               (long long)heads, (long long)batch->seqs, (long long)batch->width);
  TS_CHECK_ARG(z.bytes == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= z.bytes),
               "ts_paged_attention: workspace of %lld bytes, need %lld", (long long)workspace_bytes, (long long)z.bytes);
  AttnArgs a{};
  a.batch = batch_of(*batch, tokens);
  if (batch->width == 0) {  // a table that may be read, though none of it is used
    a.batch.table = batch->lengths;
    a.batch.ld_table = 0;
  }
  a.query = (const char*)query;
  a.token_stride = token_stride;
  a.head_stride = head_stride;
  a.out = (char*)out;
  a.key = (const char*)cache->key;
  a.value = (const char*)cache->value;
  a.key_scale = cache->key_scale;
  a.value_scale = cache->value_scale;
  a.key_page_stride = cache->key_page_stride * (cache->bits / 8);
  a.value_page_stride = cache->value_page_stride * (cache->bits / 8);
  a.pages = cache->pages;
  a.scale = scale * kLog2e;
  a.heads = (int32_t)heads;
  a.kv_heads = cache->kv_heads;
  a.group = (int32_t)(heads / cache->kv_heads);
  a.head_dim = cache->head_dim;
  a.page_shift = shift_of(cache->page_size);
  a.few_rows = z.groups[1] ? kFewRows : 0;
  char* at = (char*)workspace;
  const bool merges = z.slots[0] || z.slots[1];
  if (merges) {
    a.plan = (Plan*)at;
    at += (batch->seqs * (int64_t)sizeof(Plan) + 255) / 256 * 256;
  }
  for (int k = 0; k < 2; ++k) {
    a.jobs[k] = (int32_t)z.jobs[k];
    a.tile_rows[k] = (int32_t)z.rows[k];
    a.slots[k] = z.slots[k];
    a.part[k] = (float*)at;
    a.stats[k] = a.part[k] + z.slots[k] * z.rows[k] * cache->row;
    at = (char*)(a.stats[k] + z.slots[k] * z.rows[k] * 2);
  }
  hipStream_t s = (hipStream_t)stream;
  launch_few(a, z, cache->dtype, cache->bits == 16, cache->row, s);
  if (z.groups[1]) launch_chunks(a, z, cache->dtype, cache->bits == 16, cache->row, s);
  if (merges) {
    if (cache->dtype == TS_F16) launch_merge<ts::f16>(a, cache->row, s);
    else launch_merge<ts::bf16>(a, cache->row, s);
  }
  return ts::check_launch("ts_paged_attention");
}

}  // extern "C"
