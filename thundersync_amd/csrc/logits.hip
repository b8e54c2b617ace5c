// Adjusting logits before a token is drawn, for gfx950.
//
//   z1 = z / r if z > 0, else z r       for tokens that the row's history holds
//   z2 = z1 - f count - p               for tokens that occur `count` > 0 times in its generated part
//   z3 = z2 + sum of the row's biases of the token, in their order
//   out = z3, or -inf where the row's mask has a 0        in fp32, rounded once
//
// A work-group takes a slice of a row's vocabulary and asks for its logits at once; while they come it counts the
// history's tokens of its slice in LDS (one word a token: generated occurrences, whether it occurs at all, whether it
// has a bias).  Few tokens are touched by a list, so a thread copies its 16 bytes as they are, bits of the mask
// applied, and takes the touched ones among them one by one.  Counts are whole numbers and biases are added in their
// order, so the result does not depend on the order of the atomics.
//
// Bound by memory: 509 rows of 151936 in bf16 with their masks and histories, 341 MB, take 73 us, 4.7 TB/s; 64 rows in
// fp32, 79 MB that the last-level cache holds, 22, of them 14 without a history (each of a row's 19 work-groups counts all of
// it).  One thread an element and a word for each took 256 and 28.
#include <algorithm>

#include "common.h"
#include "timing.h"
#include "../../include/thundersync_hip.h"

namespace ts {
namespace logits {

constexpr int kBiases = 1024;  // of a row
constexpr int kGroups = 512;    // two for each CU

struct Args {
  const char* logits;
  char* out;
  int64_t ld, ld_out;
  int32_t vocab, slice, slices;  // a slice is a multiple of 64 tokens
  int64_t groups;
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

typedef uint32_t Quad __attribute__((ext_vector_type(4)));
typedef Quad AnyQuad __attribute__((aligned(2)));  // rows of odd lengths begin anywhere

template <typename T> struct Raw;
template <> struct Raw<float> { typedef uint32_t type; };
template <> struct Raw<f16> { typedef uint16_t type; };
template <> struct Raw<bf16> { typedef uint16_t type; };

// W: a token's word.  16 bits count histories below 2^14 tokens, and 32768 of them leave room for two work-groups on a
// CU: 509 rows of 151936 with 8192 of history take 73 us, with 32 bits and half the slice 92.
template <typename T, typename I, typename W, int kThreads, int kUnits>
__global__ __launch_bounds__(kThreads) void adjust_kernel(Args a) {
  constexpr int kE = 16 / (int)sizeof(T);  // tokens of a unit
  constexpr int kAhead = 4;                // history tokens that a thread asks for at once
  constexpr int kBits = 8 * (int)sizeof(W), kPer = 32 / kBits;
  constexpr uint32_t kSeen = 1u << (kBits - 1), kBiased = 1u << (kBits - 2), kCount = kBiased - 1;
  typedef typename Raw<T>::type R;
  extern __shared__ uint32_t word[];
  // a row's slices go to the same die, whose L2 then holds the history
  const int64_t group = (int64_t)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (group >= a.groups) return;
  const int64_t row = group / a.slices;
  const int v0 = (int)(group - row * a.slices) * a.slice, n = min(a.slice, a.vocab - v0);
  const int tid = threadIdx.x;
  const R* z = (const R*)a.logits + row * a.ld + v0;
  R* o = (R*)a.out + row * a.ld_out + v0;
  Quad raw[kUnits];
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    const int t = (j * kThreads + tid) * kE;
    if (t + kE <= n) {
      raw[j] = *(const AnyQuad*)(z + t);
    } else {
      raw[j] = Quad{0, 0, 0, 0};
      for (int e = 0; e < kE && t + e < n; ++e) raw[j][e * sizeof(T) / 4] |= (uint32_t)z[t + e] << (e * sizeof(T) % 4 * 8);
    }
  }
  const uint8_t* mask = nullptr;
  bool bad = false;
  if (a.allowed || a.allowed_rows) {  // rows may name a mask where there is none
    const int64_t at = a.allowed_rows ? a.allowed_rows[row] : row;
    bad = at >= a.masks;
    if (at >= 0 && !bad) mask = (const uint8_t*)(a.allowed + at * a.ld_allowed);
  }
  uint32_t bits[kUnits];
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    const int t = (j * kThreads + tid) * kE;
    bits[j] = mask && t < n ? mask[(v0 + t) >> 3] >> (t & 7) : 0xffu;
  }
  const bool words = a.history || a.biases > 0;
  const int quads = a.slice / kPer;  // 32 bits each
  const auto mark = [&](int at, uint32_t v) { return v << (at % kPer * kBits); };
  int32_t* bias_at = (int32_t*)(word + quads);
  float* bias = (float*)(bias_at + a.biases);
  if (words) {
    const I* ids = (const I*)a.history + row * a.ld_history;
    I id[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = j * kThreads + tid;
      id[j] = i < a.history_width ? ids[i] : -1;
    }
    for (int i = tid * 4; i < quads; i += kThreads * 4) *(Quad*)(word + i) = Quad{0, 0, 0, 0};
    for (int i = tid; i < a.biases; i += kThreads) {
      const int64_t at = (int64_t)((const I*)a.bias_ids)[row * a.ld_bias_ids + i] - v0;
      bias_at[i] = at >= 0 && at < n ? (int)at : -1;
      bias[i] = a.bias[row * a.ld_bias + i];
    }
    __syncthreads();
    const int len = a.history ? min(max(a.lengths ? a.lengths[row] : a.history_width, 0), a.history_width) : 0;
    const int prompt = a.prompts ? a.prompts[row] : 0;
    for (int base = 0; base < len; base += kAhead * kThreads) {
      I next[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int64_t i = (int64_t)base + (kAhead + j) * kThreads + tid;
        next[j] = i < len ? ids[i] : -1;
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int i = base + j * kThreads + tid;
        const int64_t at = (int64_t)id[j] - v0;
        if (i < len && id[j] >= 0 && at >= 0 && at < n) {
          if (i >= prompt) atomicAdd(&word[(int)at / kPer], mark((int)at, 1u));
          else atomicOr(&word[(int)at / kPer], mark((int)at, kSeen));
        }
        id[j] = next[j];
      }
    }
    for (int i = tid; i < a.biases; i += kThreads)
      if (bias_at[i] >= 0) atomicOr(&word[bias_at[i] / kPer], mark(bias_at[i], kBiased));
    __syncthreads();
  }
  float r = a.repetition ? a.repetition[row] : a.repetition_all;
  float f = a.frequency ? a.frequency[row] : a.frequency_all;
  float p = a.presence ? a.presence[row] : a.presence_all;
  if (!(r > 0.f)) r = 1.f;
  if (f != f) f = 0.f;
  if (p != p) p = 0.f;
  const uint32_t none = __builtin_bit_cast(R, from_f<T>(-__builtin_huge_valf()));
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    const int t = (j * kThreads + tid) * kE;
    if (t >= n) continue;
    Quad x = raw[j];
    if (words) {
      uint32_t touched = 0;
#pragma unroll
      for (int e = 0; e < kE; e += kPer) {
        const uint32_t w = word[(t + e) / kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) touched |= (W)(w >> k * (kBits % 32)) ? 1u << (e + k) : 0u;
      }
      touched &= bits[j];
      while (touched) {
        const int e = __builtin_ctz(touched);
        touched &= touched - 1;
        const uint32_t w = ((const W*)word)[t + e], count = w & kCount;
        const int d = e * (int)sizeof(T) / 4, shift = e * (int)sizeof(T) % 4 * 8;
        const uint32_t all = d & 2 ? (d & 1 ? x[3] : x[2]) : (d & 1 ? x[1] : x[0]);
        float y = to_f(__builtin_bit_cast(T, (R)(all >> shift)));
        if (w & ~kBiased) y = y > 0.f ? y / r : y * r;
        if (count) y -= f * (float)count + p;
        if (w & kBiased) {
          float add = 0.f;
          for (int k = 0; k < a.biases; ++k)
            if (bias_at[k] == t + e) add += bias[k];
          y += add;
        }
        const uint32_t keep = sizeof(T) == 4 ? 0u : 0xffff0000u >> shift;
        const uint32_t value = (all & keep) | (uint32_t)__builtin_bit_cast(R, from_f<T>(y)) << shift;
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = k == d ? value : x[k];
      }
    }
    if (bad) x = Quad{1, 1, 1, 1} * (__builtin_bit_cast(R, from_f<T>(__builtin_nanf(""))) * (sizeof(T) == 4 ? 1u : 0x10001u));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (sizeof(T) == 4) {
        x[k] = bits[j] >> k & 1 ? x[k] : none;
      } else {
        const uint32_t low = bits[j] >> 2 * k & 1 ? x[k] & 0xffff : none;
        const uint32_t high = bits[j] >> (2 * k + 1) & 1 ? x[k] >> 16 : none;
        x[k] = low | high << 16;
      }
    }
    if (t + kE <= n) {
      *(AnyQuad*)(o + t) = x;
    } else {
      for (int e = 0; e < kE && t + e < n; ++e) o[t + e] = (R)(x[e * sizeof(T) / 4] >> (e * sizeof(T) % 4 * 8));
    }
  }
}

template <typename T, typename I, typename W, int kThreads, int kTokens>
int launch(Args& a, int64_t rows, hipStream_t s) {
  const int most = std::min(kTokens, (16384 - 2 * a.biases) * (4 / (int)sizeof(W)) / 64 * 64);  // 64 KB of words and biases
  // few rows: down to 2048 tokens a slice, until every CU has two (one row: 7.5 us, in slices of 16384 9.5)
  a.slices = std::max((a.vocab + most - 1) / most, std::min((a.vocab + 2047) / 2048, (int)(kGroups / rows)));
  a.slice = ((a.vocab + a.slices - 1) / a.slices + 63) / 64 * 64;
  a.groups = rows * a.slices;
  const int64_t grid = (a.groups + 7) / 8 * 8;
  TS_CHECK_ARG(grid * kThreads < (1ll << 32), "ts_adjust_logits: %lld rows of %d: grid too large", (long long)rows, a.vocab);
  const size_t lds = a.history || a.biases > 0 ? a.slice * sizeof(W) + 8 * (size_t)a.biases : 0;
  TimedLaunch timed_("logits.adjust_kernel", s);
  hipLaunchKernelGGL((adjust_kernel<T, I, W, kThreads, kTokens * (int)sizeof(T) / 16 / kThreads>), dim3((unsigned)grid),
                     dim3(kThreads), lds, s, a);
  return check_launch("ts_adjust_logits");
}

// Every slice reads the row's whole history, so many rows of 16 bits take long slices: of 151936 tokens with 8192 of
// history, 384 rows take 55 us in slices of 32768 and 80 in slices of 8192, 32 rows 12.6 and 14.6, 8 rows 10.4 and 9.6.
// In fp32 the logits are the larger part, and short slices keep more of them in flight: 200 rows with 4096 of history
// take 57 us against 63.
template <typename T, typename I>
int launch_by_rows(Args& a, int64_t rows, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (rows * a.vocab >= (1 << 22)) {
      if (a.history_width < (1 << 14)) return launch<T, I, uint16_t, 1024, 32768>(a, rows, s);
      return launch<T, I, uint32_t, 1024, 16384>(a, rows, s);
    }
  }
  return launch<T, I, uint32_t, 512, 8192>(a, rows, s);
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
  TS_CHECK_ARG(history_width >= 0 && history_width < (1 << 30) && biases >= 0 && biases <= kBiases && ld_history >= 0 &&
                   ld_bias_ids >= 0 && ld_bias >= 0 && ld_allowed >= 0 && masks >= 0,
               "ts_adjust_logits: bad lists (history %lld, biases %lld)", (long long)history_width, (long long)biases);
  TS_CHECK_ARG((repetition || repetition_all > 0) && (frequency || frequency_all == frequency_all) &&
                   (presence || presence_all == presence_all),
               "ts_adjust_logits: a penalty that is no number, or a repetition not above 0");
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(logits && out && (biases == 0 || (bias_ids && bias)) && (allowed || !allowed_rows || masks == 0),
               "ts_adjust_logits: null pointer");
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
  if (id_bytes == 8) {
    if (dtype == TS_F32) return launch_by_rows<float, int64_t>(a, rows, s);
    if (dtype == TS_F16) return launch_by_rows<ts::f16, int64_t>(a, rows, s);
    return launch_by_rows<ts::bf16, int64_t>(a, rows, s);
  }
  if (dtype == TS_F32) return launch_by_rows<float, int32_t>(a, rows, s);
  if (dtype == TS_F16) return launch_by_rows<ts::f16, int32_t>(a, rows, s);
  return launch_by_rows<ts::bf16, int32_t>(a, rows, s);
}

}  // extern "C"
