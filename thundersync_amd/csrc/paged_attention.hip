// Attention of a call's rows over the keys of a paged cache, for gfx950.
//
//   row of new token i of a sequence's n, query head h: o = sum_k w_k v_k / sum_k w_k, w_k = exp(scale q . k_k - m),
//   over the keys of KV head h / group at positions 0 .. length - n + i; a row without keys is zero
#include <algorithm>

#include "paged.h"
#include "timing.h"

namespace ts {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
  Batch batch;
  const char* query;  // rows of head_dim elements
  int64_t token_stride, head_stride;
  char* out;          // [tokens][heads][head_dim]
  const char *key, *value;
  const float *key_scale, *value_scale;
  int64_t key_page_stride, value_page_stride;
  int64_t pages;
  float scale;        // log2 units
  int32_t heads, kv_heads, head_dim, page_shift;
};

// A wave a row: lanes hold ROW / 64 elements each.
template <typename T, bool WIDE, int ROW>
__device__ __forceinline__ void load_row(const char* page, int head, int slot, int page_shift, const float* scale, int lane,
                                         float (&x)[ROW / 64]) {
  constexpr int N = ROW / 64;
  const int64_t at = ((int64_t)head << page_shift) + slot;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t e = at * ROW + lane * N + i;
    if constexpr (WIDE) x[i] = to_f(((const T*)page)[e]);
    else x[i] = __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t*)page)[e], 0) * scale[at >> 4];
  }
}

template <typename T, bool WIDE, int ROW>
__global__ __launch_bounds__(256) void simple_kernel(AttnArgs a) {
  constexpr int N = ROW / 64;
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= (int64_t)a.batch.tokens * a.heads) return;
  const int t = (int)(unit / a.heads), h = (int)(unit % a.heads), hk = h / (a.heads / a.kv_heads);
  float q[N], acc[N], m = -__builtin_huge_valf(), l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = lane * N + i;
    q[i] = d < a.head_dim ? to_f(((const T*)a.query)[t * a.token_stride + h * a.head_stride + d]) * a.scale : 0.f;
    acc[i] = 0.f;
  }
  const int s = seq_of_row(a.batch, t);
  int last = -1;
  if (s < a.batch.seqs) {
    const Seq seq = seq_of(a.batch, s);
    last = seq.len - seq.n + (t - seq.row0);
  }
  bool bad = false;
  for (int k = 0; k <= last; ++k) {
    const int page = page_of(a.batch, s, k, a.page_shift, a.pages);
    if (page < 0) {
      bad = true;
      break;
    }
    const int slot = k & ((1 << a.page_shift) - 1);
    const int64_t scales = ((int64_t)page * a.kv_heads << a.page_shift) >> 4;
    float x[N], dot = 0.f;
    load_row<T, WIDE, ROW>(a.key + page * a.key_page_stride * (WIDE ? 2 : 1), hk, slot, a.page_shift,
                           a.key_scale + scales, lane, x);
#pragma unroll
    for (int i = 0; i < N; ++i) dot += q[i] * x[i];
    dot = wave_sum(dot);
    const float mn = fmaxf(m, dot), ref = mn == -__builtin_huge_valf() ? 0.f : mn;
    const float w = fast_exp2(dot - ref), r = fast_exp2(m - ref);
    m = mn;
    l = l * r + w;
    load_row<T, WIDE, ROW>(a.value + page * a.value_page_stride * (WIDE ? 2 : 1), hk, slot, a.page_shift,
                           a.value_scale + scales, lane, x);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = acc[i] * r + w * x[i];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = lane * N + i;
    if (d < a.head_dim)
      ((T*)a.out)[((int64_t)t * a.heads + h) * a.head_dim + d] =
          from_f<T>(bad ? __builtin_nanf("") : last < 0 ? 0.f : acc[i] / l);
  }
}

template <typename T, bool WIDE>
void launch_rows(const AttnArgs& a, int row, hipStream_t s) {
  const dim3 grid((unsigned)(((int64_t)a.batch.tokens * a.heads + 3) / 4)), block(256);
  ts::TimedLaunch timed_("paged.attention_kernel", s);
  switch (row) {
    case 64: hipLaunchKernelGGL((simple_kernel<T, WIDE, 64>), grid, block, 0, s, a); break;
    case 128: hipLaunchKernelGGL((simple_kernel<T, WIDE, 128>), grid, block, 0, s, a); break;
    case 192: hipLaunchKernelGGL((simple_kernel<T, WIDE, 192>), grid, block, 0, s, a); break;
    default: hipLaunchKernelGGL((simple_kernel<T, WIDE, 256>), grid, block, 0, s, a);
  }
}

}  // namespace paged
}  // namespace ts

extern "C" {

int64_t ts_paged_attention_workspace(const ts_paged_cache* cache, const ts_paged_batch* batch, int64_t tokens,
                                     int64_t heads) {
  return 0;
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
  TS_CHECK_ARG(tokens * heads < (1ll << 25), "ts_paged_attention: %lld rows of %lld heads: grid too large",
               (long long)tokens, (long long)heads);
  AttnArgs a;
  a.batch = batch_of(*batch, tokens);
  a.query = (const char*)query;
  a.token_stride = token_stride;
  a.head_stride = head_stride;
  a.out = (char*)out;
  a.key = (const char*)cache->key;
  a.value = (const char*)cache->value;
  a.key_scale = cache->key_scale;
  a.value_scale = cache->value_scale;
  a.key_page_stride = cache->key_page_stride;
  a.value_page_stride = cache->value_page_stride;
  a.pages = cache->pages;
  a.scale = scale * kLog2e;
  a.heads = (int32_t)heads;
  a.kv_heads = cache->kv_heads;
  a.head_dim = cache->head_dim;
  a.page_shift = shift_of(cache->page_size);
  hipStream_t s = (hipStream_t)stream;
  if (cache->dtype == TS_F16) {
    if (cache->bits == 16) launch_rows<ts::f16, true>(a, cache->row, s);
    else launch_rows<ts::f16, false>(a, cache->row, s);
  } else {
    if (cache->bits == 16) launch_rows<ts::bf16, true>(a, cache->row, s);
    else launch_rows<ts::bf16, false>(a, cache->row, s);
  }
  return ts::check_launch("ts_paged_attention");
}

}  // extern "C"
