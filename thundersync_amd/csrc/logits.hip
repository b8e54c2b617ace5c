// Adjusting logits before a token is drawn, for gfx950.
//
//   z1 = z / r if z > 0, else z r       for tokens that the row's history holds
//   z2 = z1 - f count - p               for tokens that occur `count` > 0 times in its generated part
//   z3 = z2 + sum of the row's biases of the token, in their order
//   out = z3, or -inf where the row's mask has a 0        in fp32, rounded once
//
// A work-group takes a slice of a row's vocabulary.  It counts the history's tokens of its slice in
// LDS (one word a token: generated occurrences, whether it occurs at all, whether it has a bias), then passes
// over the slice once.  Counts are whole numbers and biases are added in their order, so the result does not
// depend on the order of the atomics.
#include <algorithm>

#include "common.h"
#include "timing.h"
#include "../../include/thundersync_hip.h"

namespace ts {
namespace logits {

constexpr int kThreads = 512;
constexpr int kSlice = 8192;  // tokens of a work-group
constexpr uint32_t kSeen = 1u << 31, kBiased = 1u << 30, kCount = kBiased - 1;

struct Args {
  const char* logits;
  char* out;
  int64_t ld, ld_out;
  int32_t vocab;
  const void* history;
  int64_t ld_history;
  int32_t history_width;
  const int32_t *lengths, *prompts;
  const float *repetition, *frequency, *presence;  // per row, or null
  float repetition_all, frequency_all, presence_all;
  const void* bias_ids;
  const float* bias;
  int64_t ld_bias_ids, ld_bias;
  int32_t biases;
  const uint32_t* allowed;
  int64_t ld_allowed;
  const int32_t* allowed_rows;  // the mask's row of each row (negative: none), or null
  int64_t masks;
};

// A row's token list, in 64 or 32 bits.
template <typename I> __device__ __forceinline__ int64_t id_at(const void* p, int64_t i) { return ((const I*)p)[i]; }

template <typename T, typename I>
__global__ __launch_bounds__(kThreads) void adjust_kernel(Args a) {
  __shared__ uint32_t word[kSlice];
  const int slices = (a.vocab + kSlice - 1) / kSlice;
  const int64_t row = blockIdx.x / slices;
  const int v0 = (int)(blockIdx.x % slices) * kSlice, n = min(kSlice, a.vocab - v0);
  const bool words = a.history || a.biases > 0;
  if (words) {
    for (int i = threadIdx.x; i < n; i += kThreads) word[i] = 0;
    __syncthreads();
    if (a.history) {
      const int len = min(max(a.lengths ? a.lengths[row] : a.history_width, 0), a.history_width);
      const int prompt = a.prompts ? a.prompts[row] : 0;
      for (int i = threadIdx.x; i < len; i += kThreads) {
        const int64_t at = id_at<I>(a.history, row * a.ld_history + i) - v0;
        if (at < 0 || at >= n) continue;
        atomicOr(&word[at], kSeen);
        if (i >= prompt) atomicAdd(&word[at], 1u);
      }
    }
    for (int i = threadIdx.x; i < a.biases; i += kThreads) {
      const int64_t at = id_at<I>(a.bias_ids, row * a.ld_bias_ids + i) - v0;
      if (at >= 0 && at < n) atomicOr(&word[at], kBiased);
    }
    __syncthreads();
  }
  float r = a.repetition ? a.repetition[row] : a.repetition_all;
  float f = a.frequency ? a.frequency[row] : a.frequency_all;
  float p = a.presence ? a.presence[row] : a.presence_all;
  if (!(r > 0.f)) r = 1.f;
  if (f != f) f = 0.f;
  if (p != p) p = 0.f;
  const uint32_t* mask = nullptr;
  bool bad = false;
  if (a.allowed) {
    const int64_t at = a.allowed_rows ? a.allowed_rows[row] : row;
    bad = at >= a.masks;
    if (at >= 0 && !bad) mask = a.allowed + at * a.ld_allowed;
  }
  const T* z = (const T*)a.logits + row * a.ld + v0;
  T* o = (T*)a.out + row * a.ld_out + v0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    float x = to_f(z[i]);
    if (words) {
      const uint32_t w = word[i];
      if (w & kSeen) x = x > 0.f ? x / r : x * r;
      const uint32_t count = w & kCount;
      if (count) x -= f * (float)count + p;
      if (w & kBiased) {
        float add = 0.f;
        for (int k = 0; k < a.biases; ++k)
          if (id_at<I>(a.bias_ids, row * a.ld_bias_ids + k) == v0 + i) add += a.bias[row * a.ld_bias + k];
        x += add;
      }
    }
    if (mask && !((mask[(v0 + i) >> 5] >> (i & 31)) & 1)) x = -__builtin_huge_valf();
    o[i] = from_f<T>(bad ? __builtin_nanf("") : x);
  }
}

}  // namespace logits
}  // namespace ts

extern "C" {

int ts_adjust_logits(const void* logits, int64_t ld_logits, int64_t rows, int64_t vocab, const void* history,
                     int64_t ld_history, int64_t history_width, const int32_t* lengths, const int32_t* prompt_lengths,
                     const float* repetition, float repetition_all, const float* frequency, float frequency_all,
                     const float* presence, float presence_all, const void* bias_ids, int64_t ld_bias_ids,
                     const float* bias, int64_t ld_bias, int64_t biases, const int32_t* allowed, int64_t ld_allowed,
                     const int32_t* allowed_rows, int64_t masks, int id_bytes, void* out, int64_t ld_out, int dtype,
                     void* stream) {
  using namespace ts::logits;
  TS_CHECK_ARG(dtype == TS_F32 || dtype == TS_F16 || dtype == TS_BF16, "ts_adjust_logits: dtype %d", dtype);
  TS_CHECK_ARG(rows >= 0 && rows < (1ll << 31) && vocab >= 1 && vocab <= (1 << 21) && ld_logits >= 0 && ld_out >= vocab,
               "ts_adjust_logits: bad shape rows=%lld vocab=%lld", (long long)rows, (long long)vocab);
  TS_CHECK_ARG(id_bytes == 4 || id_bytes == 8, "ts_adjust_logits: ids of %d bytes", id_bytes);
  TS_CHECK_ARG(history_width >= 0 && history_width < (1 << 30) && biases >= 0 && biases <= 65536 && ld_history >= 0 &&
                   ld_bias_ids >= 0 && ld_bias >= 0 && ld_allowed >= 0 && masks >= 0,
               "ts_adjust_logits: bad lists (history %lld, biases %lld)", (long long)history_width, (long long)biases);
  TS_CHECK_ARG((repetition || repetition_all > 0) && (frequency || frequency_all == frequency_all) &&
                   (presence || presence_all == presence_all),
               "ts_adjust_logits: a penalty that is no number, or a repetition not above 0");
  const int64_t groups = rows * ((vocab + kSlice - 1) / kSlice);
  TS_CHECK_ARG(groups * kThreads < (1ll << 32), "ts_adjust_logits: %lld rows of %lld: grid too large", (long long)rows,
               (long long)vocab);
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(logits && out && (biases == 0 || (bias_ids && bias)), "ts_adjust_logits: null pointer");
  Args a{};
  a.logits = (const char*)logits;
  a.out = (char*)out;
  a.ld = ld_logits;
  a.ld_out = ld_out;
  a.vocab = (int32_t)vocab;
  a.history = history_width > 0 ? history : nullptr;
  a.ld_history = ld_history;
  a.history_width = (int32_t)history_width;
  a.lengths = lengths;
  a.prompts = prompt_lengths;
  a.repetition = repetition;
  a.frequency = frequency;
  a.presence = presence;
  a.repetition_all = repetition_all;
  a.frequency_all = frequency_all;
  a.presence_all = presence_all;
  a.bias_ids = bias_ids;
  a.bias = bias;
  a.ld_bias_ids = ld_bias_ids;
  a.ld_bias = ld_bias;
  a.biases = (int32_t)biases;
  a.allowed = (const uint32_t*)allowed;
  a.ld_allowed = ld_allowed;
  a.allowed_rows = allowed_rows;
  a.masks = masks;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)groups), block(kThreads);
  {
    ts::TimedLaunch timed_("logits.adjust_kernel", s);
#define TS_ADJUST(T)                                                                                    \
  do {                                                                                                  \
    if (id_bytes == 8) hipLaunchKernelGGL((adjust_kernel<T, int64_t>), grid, block, 0, s, a);           \
    else hipLaunchKernelGGL((adjust_kernel<T, int32_t>), grid, block, 0, s, a);                         \
  } while (0)
    if (dtype == TS_F32) TS_ADJUST(float);
    else if (dtype == TS_F16) TS_ADJUST(ts::f16);
    else TS_ADJUST(ts::bf16);
#undef TS_ADJUST
  }
  return ts::check_launch("ts_adjust_logits");
}

}  // extern "C"
