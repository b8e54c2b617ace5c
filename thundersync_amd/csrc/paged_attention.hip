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

// o = sum_p acc_p 2^(m_p - M) / sum_p l_p 2^(m_p - M) over a row's slices, M the largest m: a work-group a row, its
// waves every fourth slice, then the waves in order.
template <typename T, int ROW>
__global__ __launch_bounds__(256) void merge_kernel(AttnArgs a) {
  constexpr int N = ROW / 64;
  __shared__ float s_acc[4][ROW], s_stat[4][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
  const int s = seq_of_row(a.batch, t);
  if (s >= a.batch.seqs) return;
  const Seq q = seq_of(a.batch, s);
  if (t < q.row0 || t >= q.row0 + q.n) return;
  const Plan plan = a.plan[s];
  if (plan.slices <= 1) return;
  const int head = h / a.group, row = (t - q.row0) * a.group + h % a.group, tile = row / plan.rows;
  const float *part = a.part[plan.kernel], *stats = a.stats[plan.kernel];
  const int tiles = (q.n * a.group + plan.rows - 1) / plan.rows;
  const int64_t step = (int64_t)tiles * a.kv_heads * plan.rows;
  const int64_t at = ((int64_t)(plan.unit0 + tile) * a.kv_heads + head) * plan.rows + row % plan.rows;
  float most = neg_inf();
  for (int p = lane; p < plan.slices; p += 64) most = fmaxf(most, stats[2 * (at + p * step)]);
  most = wave_max(most);
  const float ref = most == neg_inf() ? 0.f : most;
  float acc[N], sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int p = wave; p < plan.slices; p += 4) {
    const int64_t i0 = at + p * step;
    const float w = fast_exp2(stats[2 * i0] - ref);
    sum = fmaf(stats[2 * i0 + 1], w, sum);
    const float* x = part + i0 * ROW + N * lane;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = fmaf(x[i], w, acc[i]);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) s_acc[wave][N * lane + i] = acc[i];
  if (lane == 0) s_stat[wave][0] = sum;
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= a.head_dim) return;
  const float l = (s_stat[0][0] + s_stat[1][0]) + (s_stat[2][0] + s_stat[3][0]);
  const float o = (s_acc[0][d] + s_acc[1][d]) + (s_acc[2][d] + s_acc[3][d]);
  ((T*)a.out)[((int64_t)t * a.heads + h) * a.head_dim + d] = from_f<T>(o * (l > 0.f ? 1.f / l : 0.f));
}

// Sequences of up to 32 query rows a KV head are the few kernel's.
constexpr int kFewRows = 32;

Sizes sizes_of(const ts_paged_cache& c, const ts_paged_batch& b, int64_t tokens, int64_t heads) {
  Sizes z{};
  const int64_t group = heads / c.kv_heads, keys = b.width * c.page_size + 16;
  const bool ragged = b.offsets != nullptr, chunks = ragged && tokens * group > kFewRows;
  // 32 rows a tile would not fit the registers beside wide rows' loads
  z.rows[0] = (ragged || group > 16) && c.row <= 128 ? 32 : 16;
  z.rows[1] = 128;
  z.target[0] = c.row * z.rows[0] <= 128 * 16 ? 1024 : 512;
  z.target[1] = 512;
  const int64_t seqs = std::min(b.seqs, tokens);
  const int64_t tiles[2] = {
      !ragged ? seqs * ((group + z.rows[0] - 1) / z.rows[0]) : seqs * (kFewRows / z.rows[0]),
      chunks ? tokens * group / z.rows[1] + std::min(seqs, tokens * group / (kFewRows + 1)) : 0};
  const int64_t least[2] = {kSliceLeast<0>, kSliceLeast<1>}, longest[2] = {kSliceLong<0>, kSliceLong<1>};
  int64_t plan = 0;
  for (int k = 0; k < 2; ++k) {
    const int64_t most = c.kv_heads * tiles[k] * ((keys + least[k] - 1) / least[k]);
    // kv_heads * keys / slice, for any lengths (a rounded slice may be short of its length by 2^-20)
    const int64_t cut = std::max(z.target[k], std::min(4 * z.target[k], c.kv_heads * tiles[k] * keys / longest[k])) * 65 / 64;
    z.items[k] = std::min(most, cut + c.kv_heads * (tiles[k] + 1));
    z.slots[k] = keys <= least[k] ? 0 : std::min(most, 2 * (cut + c.kv_heads));
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
  TS_CHECK_ARG(__builtin_isfinite(scale), "ts_paged_attention: scale %g", (double)scale);
  if (tokens == 0) return TS_OK;
  TS_CHECK_ARG(query && out, "ts_paged_attention: null pointer");
  TS_CHECK_ARG((((uintptr_t)query | (uintptr_t)out) & 15) == 0 && (token_stride | head_stride) % 8 == 0,
               "ts_paged_attention: rows not 16-byte aligned");
  const Sizes z = sizes_of(*cache, *batch, tokens, heads);
  // 2^24 work-groups of 256 threads wrap a launch; a slice of 2^30 keys has to be enough for `target` of them
  TS_CHECK_ARG(tokens * heads < (1ll << 24) && std::max(z.items[0], z.items[1]) + tokens / 16 < (1ll << 24) - 1 &&
                   batch->width * cache->page_size <= kMaxKeys &&
                   (double)batch->width * cache->page_size * (double)(z.items[0] + z.items[1]) < 1e11,
               "ts_paged_attention: %lld rows of %lld heads over %lld sequences of %lld pages: too large", (long long)tokens,
               (long long)heads, (long long)batch->seqs, (long long)batch->width);
  TS_CHECK_ARG(z.bytes == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= z.bytes),
               "ts_paged_attention: workspace of %lld bytes, need %lld", (long long)workspace_bytes, (long long)z.bytes);
  AttnArgs a{};
  a.batch = batch_of(*batch, tokens);
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
  a.few_rows = z.items[1] ? kFewRows : 0;
  char* at = (char*)workspace;
  const bool merges = z.slots[0] || z.slots[1];
  if (merges) {
    a.plan = (Plan*)at;
    at += (batch->seqs * (int64_t)sizeof(Plan) + 255) / 256 * 256;
  }
  for (int k = 0; k < 2; ++k) {
    a.target[k] = (int32_t)z.target[k];
    a.part[k] = (float*)at;
    a.stats[k] = a.part[k] + z.slots[k] * z.rows[k] * cache->row;
    at = (char*)(a.stats[k] + z.slots[k] * z.rows[k] * 2);
  }
  hipStream_t s = (hipStream_t)stream;
  launch_few(a, z, cache->dtype, cache->bits == 16, cache->row, s);
  if (z.items[1]) launch_chunks(a, z, cache->dtype, cache->bits == 16, cache->row, s);
  if (merges) {
    ts::TimedLaunch timed_("paged.merge_kernel", s);
    const dim3 grid((unsigned)(tokens * heads)), block(256);
    switch (cache->row) {
      case 64: TS_LAUNCH_E_T(cache->dtype, merge_kernel, 64, grid, block, 0, s, a); break;
      case 128: TS_LAUNCH_E_T(cache->dtype, merge_kernel, 128, grid, block, 0, s, a); break;
      case 192: TS_LAUNCH_E_T(cache->dtype, merge_kernel, 192, grid, block, 0, s, a); break;
      default: TS_LAUNCH_E_T(cache->dtype, merge_kernel, 256, grid, block, 0, s, a);
    }
  }
  return ts::check_launch("ts_paged_attention");
}

}  // extern "C"
