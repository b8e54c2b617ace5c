// What the kernels over a paged cache share: its description, the batch of sequences that a call
// appends or reads, and the 8-bit form of its values.
//
// A page holds page_size consecutive tokens of one sequence, head after head: rows of `row`
// elements (head_dim of them used, the rest zero), [pages][kv_heads][page_size][row].  An 8-bit
// cache holds e4m3 codes and an fp32 scale, a power of two, for each kScaleTokens tokens of a
// page and head, [pages][kv_heads][page_size / kScaleTokens]: a value is code * scale exactly, in
// bf16 and fp16 too, so that whatever reads it goes on as with a 16-bit cache.
#pragma once

#include "common.h"
#include "../../include/thundersync_hip.h"

namespace ts {
namespace paged {

constexpr int kScaleTokens = 16;
constexpr int64_t kMaxSeqs = 1 << 20;
constexpr int64_t kMaxTokens = 1ll << 31;

struct Batch {
  const int32_t* table;    // page ids, `width` a sequence
  int64_t ld_table;
  int32_t width;
  const int32_t* lengths;  // tokens of a sequence, the call's own among them
  const int32_t* offsets;  // first row of each sequence's tokens in the call, or null: one each
  int32_t seqs;
  int32_t tokens;          // rows of the call
};

struct Seq {
  int len;   // tokens in the cache with the call's own; 0: none
  int row0;  // its rows of the call
  int n;
};

// Rows outside the call's are no sequence's, whatever the offsets say.
__device__ __forceinline__ Seq seq_of(const Batch& b, int s) {
  Seq q;
  q.len = max(b.lengths[s], 0);
  if (b.offsets) {
    q.row0 = min(max(b.offsets[s], 0), b.tokens);
    q.n = min(max(b.offsets[s + 1], q.row0), b.tokens) - q.row0;
  } else {
    q.row0 = s;
    q.n = 1;
  }
  return q;
}

// The sequence of row `t`, the first whose rows end past it; seqs if none does.
__device__ __forceinline__ int seq_of_row(const Batch& b, int t) {
  if (!b.offsets) return t;
  int lo = 0, hi = b.seqs;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (b.offsets[mid + 1] > t) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// The page of position `pos`, or -1: past the table, or no page of the cache.
__device__ __forceinline__ int page_of(const Batch& b, int s, int pos, int page_shift, int64_t pages) {
  const int at = pos >> page_shift;
  if (at >= b.width) return -1;
  const int page = b.table[(int64_t)s * b.ld_table + at];
  return page >= 0 && page < pages ? page : -1;
}

// Scales are powers of two within these exponents, so that code * scale and value / scale are
// exact in fp32, and code * scale in the element type: codes below the normal ones have steps of 2^-9 of the
// scale, fp16 has steps of 2^-24 (values of the type lose nothing by it: they have no smaller steps to keep).
constexpr int kMinExponent = -118, kMaxExponent = 120;
template <typename T> constexpr int kLeastExponent = std::is_same_v<T, f16> ? -15 : kMinExponent;
__device__ __forceinline__ float two_to(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ int exponent_of(float scale) { return (int)(__float_as_uint(scale) >> 23) - 127; }

// The smallest exponent e with most <= 448 * 2^e (448 = 1.75 * 2^8: e4m3's largest value).
template <typename T> __device__ __forceinline__ int exponent_for(float most) {
  const uint32_t u = __float_as_uint(most);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(kLeastExponent<T>, min(kMaxExponent, e));
}

// The largest code of a block: below the top of the element type all of e4m3, at it the largest
// whose value the type still holds (65504 rounds to 65536 otherwise).
template <typename T> __device__ __forceinline__ float code_limit(int e) {
  return e >= (std::is_same_v<T, f16> ? 8 : 120) ? 240.f : 448.f;
}

// x / 2^e within the limit; infinities and NaN become NaN, e4m3 has no infinity
__device__ __forceinline__ float code_value(float x, float inverse, float limit) {
  const float y = fminf(fmaxf(x * inverse, -limit), limit);
  return fabsf(x) < __builtin_huge_valf() ? y : __builtin_nanf("");
}

// two codes to two T values times a power of two, four codes from four floats
template <typename T, bool HI> __device__ __forceinline__ uint32_t widen2(uint32_t codes, float scale) {
  uint32_t r;
  if constexpr (std::is_same_v<T, f16>) {
    const auto h = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HI);
    __builtin_memcpy(&r, &h, 4);
  } else {
    const auto h = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HI);
    __builtin_memcpy(&r, &h, 4);
  }
  return r;
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
__device__ __forceinline__ void codes_to_f(uint32_t c, float (&x)[4]) {
  x[0] = __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
  x[1] = __builtin_amdgcn_cvt_f32_fp8((int)c, 1);
  x[2] = __builtin_amdgcn_cvt_f32_fp8((int)c, 2);
  x[3] = __builtin_amdgcn_cvt_f32_fp8((int)c, 3);
}

// host side
int check_cache(const ts_paged_cache* c, const char* what);
int check_batch(const ts_paged_batch* b, int64_t tokens, const char* what);
inline Batch batch_of(const ts_paged_batch& b, int64_t tokens) {
  return Batch{b.table, b.ld_table, (int32_t)b.width, b.lengths, b.offsets, (int32_t)b.seqs, (int32_t)tokens};
}
inline int shift_of(int page_size) { return __builtin_ctz((unsigned)page_size); }

}  // namespace paged
}  // namespace ts
