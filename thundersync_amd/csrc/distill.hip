// Distillation from a teacher's top logits through the head, for gfx950: the per-row
// divergence of the student's softmax over the whole vocabulary from the teacher's over
// its K returned tokens, and its gradient, without a [N, V] block of logits.
//
//   z[n, v] = h[n] . W[v],  q[n] = softmax_v(z[n] / T),  p[n] = softmax over the row's
//   present slots of teacher[n] / T, the slots of one token added together
//   loss[n] = sum_k p_k (log p_k - log q_k),  dz[n, v] = g[n] / T (q_v - p_v)
//
// Forward: teacher_kernel turns each row's slots into (token, p); stats_kernel reduces the
// logits of a 256-row vocabulary tile to (max, sum exp) per token in its MFMA epilogue;
// scores_kernel takes the logits at the slots' tokens as dot products; loss_kernel merges
// the tiles and sums the slots.  Backward, per block of rows: dlogits_kernel recomputes the
// logits and writes the block's q part in the element type, slots_kernel overwrites the
// slots' entries with g / T (q - p) rounded once; the vector-Jacobian products with W and h
// are the fused logprob's.  Bound by the products, as the fused logprob is (its GEMM core).
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "gemm_core.h"
#include "head_tiles.h"
#include "timing.h"
#include "../../include/thundersync_hip.h"

namespace ts {
namespace distill {

using namespace ts::gemm;
using namespace ts::head;

constexpr int kMaxTop = 1024;   // slots per row
constexpr int kRowWaves = 4;    // rows per work-group of the per-row kernels
constexpr int kDead = 0, kLive = 1, kBadId = 2;  // row states

template <typename T> __device__ __forceinline__ T wave_sum_of(T v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}

template <typename T> __device__ __forceinline__ double to_d(T x) { return (double)to_f(x); }
template <> __device__ __forceinline__ double to_d<double>(double x) { return x; }

// ---------------------------------------------------------------------------
// the teacher's distribution: one wave per row.  p is computed in fp64 (K exponentials a
// row) and stored in the compute type C.  Slots of one token are added into the first of
// them, the others become absent; K <= 1024 comparisons a slot, from LDS.
// ---------------------------------------------------------------------------
template <typename L, typename C>
__global__ __launch_bounds__(64 * kRowWaves) void teacher_kernel(const int64_t* __restrict__ ids,
                                                                 const L* __restrict__ teacher, int64_t ld_teacher,
                                                                 int rows, int top, int64_t vocab, double inv_t,
                                                                 int32_t* __restrict__ slot_id, C* __restrict__ slot_p,
                                                                 int pitch, int32_t* __restrict__ state) {
  extern __shared__ __attribute__((aligned(8))) char smem[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double* sp = reinterpret_cast<double*>(smem) + wave * top;
  int32_t* si = reinterpret_cast<int32_t*>(reinterpret_cast<double*>(smem) + kRowWaves * top) + wave * top;
  const int n = blockIdx.x * kRowWaves + wave;
  if (n >= rows) return;  // whole waves; the waves share nothing
  const int64_t* id = ids + (int64_t)n * top;
  const L* x = teacher + (int64_t)n * ld_teacher;
  // present slots: a token id of 0 or more and a logit above -inf (a NaN is present)
  auto present = [&](int k) { return id[k] >= 0 && !(to_d(x[k]) == -__builtin_huge_val()); };
  double m = -__builtin_huge_val();
  int bad = 0, some = 0;
  for (int k = lane; k < top; k += 64)
    if (present(k)) {
      m = fmax(m, to_d(x[k]));
      some = 1;
      bad |= id[k] >= vocab;
    }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    m = fmax(m, __shfl_xor(m, o, kWave));
    some |= __shfl_xor(some, o, kWave);
    bad |= __shfl_xor(bad, o, kWave);
  }
  double s = 0.;
  for (int k = lane; k < top; k += 64) {
    const bool on = present(k);
    const double e = on ? exp((to_d(x[k]) - m) * inv_t) : 0.;
    s += e;
    sp[k] = e;
    si[k] = on && id[k] < vocab ? (int32_t)id[k] : -1;
  }
  s = wave_sum_of(s);
  __builtin_amdgcn_wave_barrier();
  __threadfence_block();
  const double inv_s = some ? 1. / s : 0.;
  for (int k = lane; k < pitch; k += 64) {
    const int mine = k < top ? si[k] : -1;
    double p = 0.;
    bool first = mine >= 0;
    if (first)
      for (int j = 0; j < top; ++j) {
        if (si[j] != mine) continue;
        p += sp[j];
        first = first && j >= k;
      }
    slot_id[(int64_t)n * pitch + k] = first ? mine : -1;
    slot_p[(int64_t)n * pitch + k] = first ? (C)(p * inv_s) : (C)0;
  }
  if (lane == 0) state[n] = !some ? kDead : bad ? kBadId : kLive;
}

// ---------------------------------------------------------------------------
// forward: per (vocabulary tile, token) max and sum exp of z / T
// ---------------------------------------------------------------------------
// (max of z, sum exp((z - max) / T)) of two disjoint sets of logits, either of which may be
// empty (max = -inf, sum 0); unit = log2(e) / T.  A set that holds a NaN has a NaN sum.
__device__ __forceinline__ void merge(float& m, float& s, float mo, float so, float unit) {
  if (mo == neg_inf() || m == neg_inf()) {
    m = fmaxf(m, mo);
    s += so;
    return;
  }
  const float mn = fmaxf(m, mo);
  s = fast_exp2((m - mn) * unit) * s + fast_exp2((mo - mn) * unit) * so;
  m = mn;
}

struct StatsArgs {
  const bf16* h;
  int64_t ldh;
  const bf16* w;
  int64_t ldw;
  int rows, dim, vocab;
  int n_ttiles, n_vtiles;
  float unit;      // log2(e) / T
  float* part_m;   // [n_vtiles][rows]
  float* part_s;
};

template <typename E, class S>
__global__ __launch_bounds__(kGemmThreads, 1) void stats_kernel(StatsArgs p) {
  GEMM_RING_OF(S)
  constexpr int MI = S::MI, NI = S::NI;
  int vt, tt;
  grouped_tile(xcd_logical(blockIdx.x, p.n_ttiles * p.n_vtiles), p.n_vtiles, p.n_ttiles, vt, tt);
  const int v0 = vt * TM, n0 = tt * S::BN;
  f32x16 acc[MI][NI];
  gemm_tile<E, false, false, S>(acc, p.w + (int64_t)v0 * p.ldw, p.ldw, min(TM, p.vocab - v0),
                                p.h + (int64_t)n0 * p.ldh, p.ldh, min(S::BN, p.rows - n0), p.dim, s0, s1, s2, s3);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave % S::WM, wn = wave / S::WM;
  float* xm = reinterpret_cast<float*>(s0);  // [WM - 1][BN] per token, from the waves wm > 0
  float* xs = xm + (S::WM - 1) * S::BN;
  // rows past the vocabulary (last vocabulary tile only) take no part
  if (v0 + TM > p.vocab) {
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int ni = 0; ni < NI; ++ni)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (v0 + a_row<S>(mi, i, lane, wm) >= p.vocab) acc[mi][ni][i] = neg_inf();
  }
  float mk[NI], sk[NI];
#pragma unroll
  for (int ni = 0; ni < NI; ++ni) {
    const int col = b_row<S>(ni, lane, wn);
    float m = neg_inf();
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int i = 0; i < 16; i += 2) m = fmaxf(m, fmaxf(acc[mi][ni][i], acc[mi][ni][i + 1]));
    float sum = 0.f;
    if (m == neg_inf()) {  // nothing, or nothing but -inf and NaN, which a maximum does not show
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (acc[mi][ni][i] != neg_inf()) sum = __builtin_nanf("");
    } else {
      const float m2 = m * p.unit;
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += fast_exp2(fmaf(acc[mi][ni][i], p.unit, -m2));
    }
    const float mo = shfl_xor(m, 32), so = shfl_xor(sum, 32);  // lane ^ 32 holds the other rows
    merge(m, sum, mo, so, p.unit);
    if (wm > 0 && lane < 32) {
      xm[(wm - 1) * S::BN + col] = m;
      xs[(wm - 1) * S::BN + col] = sum;
    }
    mk[ni] = m;
    sk[ni] = sum;
  }
  __syncthreads();
#pragma unroll
  for (int ni = 0; ni < NI; ++ni) {
    const int col = b_row<S>(ni, lane, wn), n = n0 + col;
    if (wm == 0 && lane < 32 && n < p.rows) {
#pragma unroll
      for (int w = 0; w < S::WM - 1; ++w) merge(mk[ni], sk[ni], xm[w * S::BN + col], xs[w * S::BN + col], p.unit);
      p.part_m[(int64_t)vt * p.rows + n] = mk[ni];
      p.part_s[(int64_t)vt * p.rows + n] = sk[ni];
    }
  }
}

// ---------------------------------------------------------------------------
// the logits at the slots: z[n, k] = h[n] . W[slot_id[n, k]], a wave per slot
// ---------------------------------------------------------------------------
template <typename T, typename C>
__global__ __launch_bounds__(256) void scores_kernel(const T* __restrict__ h, int64_t ldh, const T* __restrict__ w,
                                                     int64_t ldw, const int32_t* __restrict__ slot_id, int pitch,
                                                     int top, int dim, C* __restrict__ z) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n = blockIdx.x;
  const T* hr = h + n * ldh;
  for (int k = 4 * blockIdx.y + wave; k < top; k += 4 * gridDim.y) {
    const int id = slot_id[n * pitch + k];
    if (id < 0) continue;
    const T* wr = w + (int64_t)id * ldw;
    C acc = (C)0;
    if constexpr (sizeof(T) == 2) {
      for (int d = 8 * lane; d < dim; d += 512) {
        float a[8], b[8];
        load8(hr + d, a);
        load8(wr + d, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc = fmaf(a[i], b[i], acc);
      }
    } else {
      for (int d = lane; d < dim; d += 64) acc = fma(hr[d], wr[d], acc);
    }
    acc = wave_sum_of(acc);
    if (lane == 0) z[n * pitch + k] = acc;
  }
}

// ---------------------------------------------------------------------------
// loss[n] = sum_k p_k (log p_k - (z_k / T - lse)); lse of z / T.  With TILES the row's lse
// is first merged from the tiles' statistics.  A work-group of 16 waves owns 16 tokens:
// its 64 slots of 16 lanes merge the tiles t = slot, slot + 64, ..., then wave w sums
// token w's slots.
// ---------------------------------------------------------------------------
constexpr int kLossTokens = 16;
template <typename C, bool TILES>
__global__ __launch_bounds__(64 * kLossTokens) void loss_kernel(const float* __restrict__ pm,
                                                                const float* __restrict__ ps, int n_vtiles, int rows,
                                                                float unit, const int32_t* __restrict__ slot_id,
                                                                const C* __restrict__ slot_p,
                                                                const C* __restrict__ slot_z, int pitch, int top,
                                                                const int32_t* __restrict__ state, C inv_t,
                                                                C* __restrict__ lse, C* __restrict__ loss) {
  __shared__ float sm[kLossTokens][kLossTokens], ss[kLossTokens][kLossTokens];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n0 = blockIdx.x * kLossTokens;
  if constexpr (TILES) {
    const int tok = lane & 15, slot = 4 * wave + (lane >> 4), n = n0 + tok;
    float M = neg_inf(), S = 0.f;
    if (n < rows) {
#pragma unroll 4
      for (int t = slot; t < n_vtiles; t += 64) {
        const int64_t o = (int64_t)t * rows + n;
        merge(M, S, pm[o], ps[o], unit);
      }
    }
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) {
      const float mo = shfl_xor(M, o), so = shfl_xor(S, o);
      merge(M, S, mo, so, unit);
    }
    if (lane < 16) {
      sm[wave][tok] = M;
      ss[wave][tok] = S;
    }
    __syncthreads();
  }
  const int n = n0 + wave;
  if (n >= rows) return;
  C l;
  if constexpr (TILES) {
    float M = sm[0][wave], S = ss[0][wave];
#pragma unroll
    for (int v = 1; v < kLossTokens; ++v) merge(M, S, sm[v][wave], ss[v][wave], unit);
    l = (C)(M * inv_t + logf(S));
    if (lane == 0) lse[n] = l;
  } else {
    l = lse[n];
  }
  C sum = (C)0;
  for (int k = lane; k < top; k += 64) {
    const int64_t o = (int64_t)n * pitch + k;
    if (slot_id[o] < 0) continue;
    const C p = slot_p[o];
    if (p == (C)0) continue;
    sum += p * (log(p) - (slot_z[o] * inv_t - l));
  }
  sum = wave_sum_of(sum);
  if (lane == 0) loss[n] = state[n] == kDead ? (C)0 : state[n] == kBadId ? (C)__builtin_nan("") : sum;
}

// ---------------------------------------------------------------------------
// backward: the q part of dlogits, [rows, ld] of E (pad columns 0)
// ---------------------------------------------------------------------------
struct DlArgs {
  const bf16* h;
  int64_t ldh;
  const bf16* w;
  int64_t ldw;
  const float* lse;
  const float* g;
  const int32_t* state;
  int rows, dim, vocab, vocab_pad;
  int n_ttiles, n_vtiles;
  float unit, inv_t;
  bf16* dl;
  int64_t ldl;
};

template <typename E, class S>
__global__ __launch_bounds__(kGemmThreads, 1) void dlogits_kernel(DlArgs p) {
  GEMM_RING_OF(S)
  constexpr int MI = S::MI, NI = S::NI;
  int vt, tt;
  grouped_tile(xcd_logical(blockIdx.x, p.n_ttiles * p.n_vtiles), p.n_vtiles, p.n_ttiles, vt, tt);
  const int v0 = vt * TM, n0 = tt * S::BN;
  f32x16 acc[MI][NI];
  gemm_tile<E, false, false, S>(acc, p.w + (int64_t)v0 * p.ldw, p.ldw, min(TM, p.vocab - v0),
                                p.h + (int64_t)n0 * p.ldh, p.ldh, min(S::BN, p.rows - n0), p.dim, s0, s1, s2, s3);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave % S::WM, wn = wave / S::WM;
  // tokens 64 q .. 64 q + 63 of the tile are staged in ring stage q as [64][OPITCH];
  // a Wide tile does not fit, its waves' two halves of the tokens take turns
  constexpr int PASSES = S::BN > TN ? S::WN : 1, PT = S::BN / PASSES;  // tokens per pass
  static_assert(PT <= 256, "four stages of 64 tokens");
  auto quarter = [&](int q) -> bf16* { return q == 0 ? s0 : q == 1 ? s1 : q == 2 ? s2 : s3; };
  auto values = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
      const int n = min(n0 + b_row<S>(ni, lane, wn), p.rows - 1);
      const float lse2 = p.lse[n] * kLog2e, g = p.g[n] * p.inv_t;
      const bool dead = p.state[n] == kDead;
      const int col = b_row<S>(ni, lane, PASSES > 1 ? 0 : wn);  // token within the pass
      bf16* out = quarter(col >> 6) + (col & 63) * OPITCH;
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          float d[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = 4 * i4 + j;
            d[j] = fast_exp2(fmaf(acc[mi][ni][i], p.unit, -lse2)) * g;
            // a row without a teacher has no gradient, whatever its hidden state holds
            if (dead || v0 + a_row<S>(mi, i, lane, wm) >= p.vocab) d[j] = 0.f;
          }
          *reinterpret_cast<u32x2*>(out + a_row<S>(mi, 4 * i4, lane, wm)) =
              u32x2{pack2<E>(d[0], d[1]), pack2<E>(d[2], d[3])};
        }
      if constexpr (PASSES > 1) __builtin_amdgcn_sched_barrier(0);
    }
  };
  const int vmax = min(TM, p.vocab_pad - v0);
  auto store = [&](int pass) __attribute__((always_inline)) {
#pragma unroll 4
    for (int it = 0; it < (PT * TM / 8) / kGemmThreads; ++it) {
      const int c = it * kGemmThreads + tid;
      const int row = c / (TM / 8), chunk = (c % (TM / 8)) * 8;
      const int n = n0 + pass * PT + row;
      if (n < p.rows && chunk < vmax)
        *reinterpret_cast<u32x4*>(p.dl + (int64_t)n * p.ldl + v0 + chunk) =
            *reinterpret_cast<const u32x4*>(quarter(row >> 6) + (row & 63) * OPITCH + chunk);
    }
  };
  if constexpr (PASSES == 1) {
    values();
    __syncthreads();
    store(0);
  } else {
    static_assert(PASSES <= 2, "two halves");
    if (wn == 0) values();
    __syncthreads();
    store(0);
    __syncthreads();
    if (wn == 1) values();
    __syncthreads();
    store(1);
  }
}

// dl[n, slot_id] = grad_scale g (q - p) with q = exp(logit_scale z - lse), rounded once: the
// slots' entries in full
template <typename T, typename C>
__global__ __launch_bounds__(256) void slots_kernel(const int32_t* __restrict__ slot_id, const C* __restrict__ slot_p,
                                                    const C* __restrict__ slot_z, int pitch, int top, int64_t rows,
                                                    const C* __restrict__ lse, const C* __restrict__ g, C logit_scale,
                                                    C grad_scale, T* __restrict__ dl, int64_t ldl) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t n = i / pitch;
  const int k = (int)(i - n * pitch);
  if (n >= rows || k >= top) return;
  const int id = slot_id[i];
  if (id < 0) return;
  const C d = (exp(slot_z[i] * logit_scale - lse[n]) - slot_p[i]) * (g[n] * grad_scale);
  if constexpr (std::is_same_v<T, C>) dl[n * ldl + id] = d;
  else dl[n * ldl + id] = from_f<T>((float)d);
}

// out[n] = live row ? scale h[n] : 0
template <typename T, typename C>
__global__ __launch_bounds__(256) void rows_kernel(const T* __restrict__ h, int64_t ldh,
                                                   const int32_t* __restrict__ state, int64_t rows, int dim, C scale,
                                                   T* __restrict__ out, int64_t ldo) {
  const int64_t n = blockIdx.x;
  const bool dead = state[n] == kDead;
  for (int d = threadIdx.x; d < dim; d += 256) {
    const T x = h[n * ldh + d];
    if constexpr (std::is_same_v<T, C>) out[n * ldo + d] = dead ? (T)0 : x * scale;
    else out[n * ldo + d] = dead ? from_f<T>(0.f) : scale == (C)1 ? x : from_f<T>(to_f(x) * scale);
  }
}

template <typename L>
void launch_teacher(const int64_t* ids, const void* teacher, int64_t ld, int64_t rows, int top, int64_t vocab,
                    double inv_t, int32_t* slot_id, void* slot_p, int pitch, int32_t* state, bool wide, hipStream_t s) {
  const dim3 grid((unsigned)((rows + kRowWaves - 1) / kRowWaves)), block(64 * kRowWaves);
  const size_t lds = (size_t)kRowWaves * top * (sizeof(double) + sizeof(int32_t));
  if (wide)
    hipLaunchKernelGGL((teacher_kernel<L, double>), grid, block, lds, s, ids, (const L*)teacher, ld, (int)rows, top,
                       vocab, inv_t, slot_id, (double*)slot_p, pitch, state);
  else
    hipLaunchKernelGGL((teacher_kernel<L, float>), grid, block, lds, s, ids, (const L*)teacher, ld, (int)rows, top,
                       vocab, inv_t, slot_id, (float*)slot_p, pitch, state);
}

bool known(int dtype) { return dtype == TS_F32 || dtype == TS_F16 || dtype == TS_BF16 || dtype == TS_F64; }

}  // namespace distill
}  // namespace ts

using namespace ts::distill;

extern "C" {

int ts_distill_teacher(const int64_t* ids, const void* teacher, int64_t ld_teacher, int teacher_dtype, int64_t rows,
                       int64_t top, int64_t vocab, double temperature, int32_t* slot_id, void* slot_p,
                       int64_t pitch, int32_t* state, int dtype, void* stream) {
  TS_CHECK_ARG(known(teacher_dtype) && known(dtype), "ts_distill_teacher: dtypes %d, %d", teacher_dtype, dtype);
  TS_CHECK_ARG(rows >= 0 && rows < (1 << 30) && top > 0 && top <= kMaxTop && vocab > 0 && vocab < (1 << 30) &&
                   pitch >= top && pitch <= kMaxTop && ld_teacher >= top,
               "ts_distill_teacher: bad shape rows=%lld top=%lld (1 .. %d) vocab=%lld", (long long)rows,
               (long long)top, kMaxTop, (long long)vocab);
  TS_CHECK_ARG(temperature > 0 && temperature < __builtin_huge_val(), "ts_distill_teacher: temperature %g",
               temperature);
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(ids && teacher && slot_id && slot_p && state, "ts_distill_teacher: null pointer");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("distill.teacher_kernel", s);
    const bool wide = dtype == TS_F64;
    const double inv = 1. / temperature;
    if (teacher_dtype == TS_F32)
      launch_teacher<float>(ids, teacher, ld_teacher, rows, (int)top, vocab, inv, slot_id, slot_p, (int)pitch, state, wide, s);
    else if (teacher_dtype == TS_F16)
      launch_teacher<ts::f16>(ids, teacher, ld_teacher, rows, (int)top, vocab, inv, slot_id, slot_p, (int)pitch, state, wide, s);
    else if (teacher_dtype == TS_BF16)
      launch_teacher<ts::bf16>(ids, teacher, ld_teacher, rows, (int)top, vocab, inv, slot_id, slot_p, (int)pitch, state, wide, s);
    else
      launch_teacher<double>(ids, teacher, ld_teacher, rows, (int)top, vocab, inv, slot_id, slot_p, (int)pitch, state, wide, s);
  }
  return ts::check_launch("ts_distill_teacher");
}

int64_t ts_distill_fwd_workspace(int64_t rows, int64_t vocab) {
  if (rows <= 0 || vocab <= 0) return 0;
  return 2 * ((vocab + TM - 1) / TM) * rows * (int64_t)sizeof(float);
}

int ts_distill_scores(const void* hidden, int64_t ld_hidden, const void* weight, int64_t ld_weight,
                      const int32_t* slot_id, int64_t pitch, int64_t rows, int64_t top, int64_t dim, void* slot_z,
                      int dtype, void* stream) {
  TS_CHECK_ARG(known(dtype), "ts_distill_scores: dtype %d", dtype);
  TS_CHECK_ARG(rows >= 0 && rows < (1 << 30) && top > 0 && top <= pitch && pitch <= kMaxTop && dim > 0 &&
                   dim < (1 << 20) && ld_hidden >= dim && ld_weight >= dim,
               "ts_distill_scores: bad shape");
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(hidden && weight && slot_id && slot_z, "ts_distill_scores: null pointer");
  TS_CHECK_ARG(dtype == TS_F32 || dtype == TS_F64 ||
                   (ok16(hidden) && ok16(weight) && dim % 8 == 0 && ld_hidden % 8 == 0 && ld_weight % 8 == 0),
               "ts_distill_scores: hidden/weight rows must be 16-byte aligned with dim %% 8 == 0");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("distill.scores_kernel", s);
    const dim3 grid((unsigned)rows, (unsigned)std::min<int64_t>((top + 3) / 4, 8));
#define TS_SCORES(T, C)                                                                                          \
  hipLaunchKernelGGL((scores_kernel<T, C>), grid, dim3(256), 0, s, (const T*)hidden, ld_hidden, (const T*)weight, \
                     ld_weight, slot_id, (int)pitch, (int)top, (int)dim, (C*)slot_z)
    if (dtype == TS_BF16) TS_SCORES(ts::bf16, float);
    else if (dtype == TS_F16) TS_SCORES(ts::f16, float);
    else if (dtype == TS_F32) TS_SCORES(float, float);
    else TS_SCORES(double, double);
#undef TS_SCORES
  }
  return ts::check_launch("ts_distill_scores");
}

int ts_distill_fwd(const void* hidden, int64_t ld_hidden, const void* weight, int64_t ld_weight, int64_t rows,
                   int64_t dim, int64_t vocab, double temperature, const int32_t* slot_id, const float* slot_p,
                   float* slot_z, int64_t pitch, int64_t top, const int32_t* state, float* loss, float* lse,
                   void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  TS_CHECK_ARG(dtype == TS_BF16 || dtype == TS_F16, "ts_distill_fwd: dtype %d (bf16 or fp16)", dtype);
  TS_CHECK_ARG(rows >= 0 && dim > 0 && vocab > 0 && rows < (1 << 30) && vocab < (1 << 30) && dim < (1 << 20) &&
                   top > 0 && top <= pitch && pitch <= kMaxTop,
               "ts_distill_fwd: bad shape rows=%lld dim=%lld vocab=%lld top=%lld", (long long)rows, (long long)dim,
               (long long)vocab, (long long)top);
  TS_CHECK_ARG(temperature > 0 && temperature < __builtin_huge_val(), "ts_distill_fwd: temperature %g", temperature);
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(hidden && weight && slot_id && slot_p && slot_z && state && loss && lse, "ts_distill_fwd: null pointer");
  TS_CHECK_ARG(dim % 8 == 0 && ld_hidden % 8 == 0 && ld_weight % 8 == 0 && ld_hidden >= dim && ld_weight >= dim &&
                   ok16(hidden) && ok16(weight),
               "ts_distill_fwd: hidden/weight rows must be 16-byte aligned with dim %% 8 == 0");
  TS_CHECK_ARG(255 * ld_hidden < (1ll << 30) && 255 * ld_weight < (1ll << 30),
               "ts_distill_fwd: leading dimensions too large for 32-bit tile offsets");
  TS_CHECK_ARG(workspace && workspace_bytes >= ts_distill_fwd_workspace(rows, vocab),
               "ts_distill_fwd: workspace of %lld bytes, need %lld", (long long)workspace_bytes,
               (long long)ts_distill_fwd_workspace(rows, vocab));
  StatsArgs a;
  a.h = (const ts::bf16*)hidden;
  a.ldh = ld_hidden;
  a.w = (const ts::bf16*)weight;
  a.ldw = ld_weight;
  a.rows = (int)rows;
  a.dim = (int)dim;
  a.vocab = (int)vocab;
  a.n_vtiles = (int)((vocab + TM - 1) / TM);
  const int width = logits_tile(rows, a.n_vtiles, ld_hidden);
  a.n_ttiles = (int)((rows + width - 1) / width);
  a.unit = (float)(1.4426950408889634 / temperature);
  a.part_m = (float*)workspace;
  a.part_s = a.part_m + (int64_t)a.n_vtiles * rows;
  TS_CHECK_ARG((int64_t)a.n_ttiles * a.n_vtiles < (1ll << 31), "ts_distill_fwd: grid too large");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("distill.stats_kernel", s);
    TS_LAUNCH_TOKENS(dtype, width, stats_kernel, dim3((unsigned)(a.n_ttiles * a.n_vtiles)), dim3(kGemmThreads), 0, s, a);
  }
  int st = ts::check_launch("ts_distill_fwd (tiles)");
  if (st != TS_OK) return st;
  st = ts_distill_scores(hidden, ld_hidden, weight, ld_weight, slot_id, pitch, rows, top, dim, slot_z, dtype, stream);
  if (st != TS_OK) return st;
  {
    ts::TimedLaunch timed_("distill.loss_kernel", s);
    hipLaunchKernelGGL((loss_kernel<float, true>), dim3((unsigned)((rows + kLossTokens - 1) / kLossTokens)),
                       dim3(64 * kLossTokens), 0, s, a.part_m, a.part_s, a.n_vtiles, (int)rows, a.unit, slot_id, slot_p,
                       slot_z, (int)pitch, (int)top, state, (float)(1. / temperature), lse, loss);
  }
  return ts::check_launch("ts_distill_fwd (loss)");
}

int ts_distill_loss(const int32_t* slot_id, const void* slot_p, const void* slot_z, int64_t pitch, int64_t top,
                    const int32_t* state, const void* lse, int64_t rows, void* loss, int dtype, void* stream) {
  TS_CHECK_ARG(dtype == TS_F32 || dtype == TS_F64, "ts_distill_loss: dtype %d (fp32 or fp64)", dtype);
  TS_CHECK_ARG(rows >= 0 && rows < (1 << 30) && top > 0 && top <= pitch && pitch <= kMaxTop,
               "ts_distill_loss: bad shape");
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(slot_id && slot_p && slot_z && state && lse && loss, "ts_distill_loss: null pointer");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("distill.loss_kernel", s);
    const dim3 grid((unsigned)((rows + kLossTokens - 1) / kLossTokens)), block(64 * kLossTokens);
    if (dtype == TS_F64)
      hipLaunchKernelGGL((loss_kernel<double, false>), grid, block, 0, s, (const float*)nullptr, (const float*)nullptr,
                         0, (int)rows, 0.f, slot_id, (const double*)slot_p, (const double*)slot_z, (int)pitch, (int)top,
                         state, 1., (double*)lse, (double*)loss);
    else
      hipLaunchKernelGGL((loss_kernel<float, false>), grid, block, 0, s, (const float*)nullptr, (const float*)nullptr,
                         0, (int)rows, 0.f, slot_id, (const float*)slot_p, (const float*)slot_z, (int)pitch, (int)top,
                         state, 1.f, (float*)lse, (float*)loss);
  }
  return ts::check_launch("ts_distill_loss");
}

int ts_distill_slots(const int32_t* slot_id, const void* slot_p, const void* slot_z, int64_t pitch, int64_t top,
                     const void* lse, const void* grad, int64_t rows, double logit_scale, double grad_scale,
                     void* dlogits, int64_t ld_dlogits, int dtype, void* stream);

int ts_distill_dlogits(const void* hidden, int64_t ld_hidden, const void* weight, int64_t ld_weight, int64_t rows,
                       int64_t dim, int64_t vocab, double temperature, const int32_t* slot_id, const float* slot_p,
                       const float* slot_z, int64_t pitch, int64_t top, const int32_t* state, const float* lse,
                       const float* grad, void* dlogits, int64_t ld_dlogits, int dtype, void* stream) {
  TS_CHECK_ARG(dtype == TS_BF16 || dtype == TS_F16, "ts_distill_dlogits: dtype %d (bf16 or fp16)", dtype);
  TS_CHECK_ARG(rows >= 0 && dim > 0 && vocab > 0 && rows < (1 << 30) && vocab < (1 << 30) && dim < (1 << 20) &&
                   top > 0 && top <= pitch && pitch <= kMaxTop,
               "ts_distill_dlogits: bad shape");
  TS_CHECK_ARG(temperature > 0 && temperature < __builtin_huge_val(), "ts_distill_dlogits: temperature %g",
               temperature);
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(hidden && weight && slot_id && slot_p && slot_z && state && lse && grad && dlogits,
               "ts_distill_dlogits: null pointer");
  TS_CHECK_ARG(dim % 8 == 0 && ld_hidden % 8 == 0 && ld_weight % 8 == 0 && ld_hidden >= dim && ld_weight >= dim &&
                   ok16(hidden) && ok16(weight) && ok16(dlogits) && ld_dlogits % 8 == 0 &&
                   ld_dlogits >= (vocab + 7) / 8 * 8,
               "ts_distill_dlogits: alignment or leading dimensions");
  TS_CHECK_ARG(255 * ld_hidden < (1ll << 30) && 255 * ld_weight < (1ll << 30),
               "ts_distill_dlogits: leading dimensions too large for 32-bit tile offsets");
  DlArgs a;
  a.h = (const ts::bf16*)hidden;
  a.ldh = ld_hidden;
  a.w = (const ts::bf16*)weight;
  a.ldw = ld_weight;
  a.lse = lse;
  a.g = grad;
  a.state = state;
  a.rows = (int)rows;
  a.dim = (int)dim;
  a.vocab = (int)vocab;
  a.vocab_pad = (int)((vocab + 7) / 8 * 8);
  a.n_vtiles = (int)((vocab + TM - 1) / TM);
  const int width = logits_tile(rows, a.n_vtiles, ld_hidden);
  a.n_ttiles = (int)((rows + width - 1) / width);
  a.unit = (float)(1.4426950408889634 / temperature);
  a.inv_t = (float)(1. / temperature);
  a.dl = (ts::bf16*)dlogits;
  a.ldl = ld_dlogits;
  TS_CHECK_ARG((int64_t)a.n_ttiles * a.n_vtiles < (1ll << 31), "ts_distill_dlogits: grid too large");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("distill.dlogits_kernel", s);
    TS_LAUNCH_TOKENS(dtype, width, dlogits_kernel, dim3((unsigned)(a.n_ttiles * a.n_vtiles)), dim3(kGemmThreads), 0, s, a);
  }
  const int st = ts::check_launch("ts_distill_dlogits");
  if (st != TS_OK) return st;
  return ts_distill_slots(slot_id, slot_p, slot_z, pitch, top, lse, grad, rows, 1. / temperature, 1. / temperature,
                          dlogits, ld_dlogits, dtype, stream);
}

int ts_distill_slots(const int32_t* slot_id, const void* slot_p, const void* slot_z, int64_t pitch, int64_t top,
                     const void* lse, const void* grad, int64_t rows, double logit_scale, double grad_scale,
                     void* dlogits, int64_t ld_dlogits, int dtype, void* stream) {
  TS_CHECK_ARG(known(dtype), "ts_distill_slots: dtype %d", dtype);
  TS_CHECK_ARG(rows >= 0 && rows < (1 << 30) && top > 0 && top <= pitch && pitch <= kMaxTop && ld_dlogits > 0,
               "ts_distill_slots: bad shape");
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(slot_id && slot_p && slot_z && lse && grad && dlogits, "ts_distill_slots: null pointer");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("distill.slots_kernel", s);
    const dim3 grid((unsigned)((rows * pitch + 255) / 256));
#define TS_SLOTS(T, C)                                                                                              \
  hipLaunchKernelGGL((slots_kernel<T, C>), grid, dim3(256), 0, s, slot_id, (const C*)slot_p, (const C*)slot_z,       \
                     (int)pitch, (int)top, rows, (const C*)lse, (const C*)grad, (C)logit_scale, (C)grad_scale,       \
                     (T*)dlogits, ld_dlogits)
    if (dtype == TS_BF16) TS_SLOTS(ts::bf16, float);
    else if (dtype == TS_F16) TS_SLOTS(ts::f16, float);
    else if (dtype == TS_F32) TS_SLOTS(float, float);
    else TS_SLOTS(double, double);
#undef TS_SLOTS
  }
  return ts::check_launch("ts_distill_slots");
}

int ts_distill_rows(const void* hidden, int64_t ld_hidden, const int32_t* state, int64_t rows, int64_t dim,
                    double scale, void* out, int64_t ld_out, int dtype, void* stream) {
  TS_CHECK_ARG(known(dtype), "ts_distill_rows: dtype %d", dtype);
  TS_CHECK_ARG(rows >= 0 && rows < (1 << 30) && dim > 0 && dim < (1 << 20) && ld_hidden >= dim && ld_out >= dim,
               "ts_distill_rows: bad shape");
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(hidden && state && out && hidden != out, "ts_distill_rows: null or aliased pointer");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("distill.rows_kernel", s);
#define TS_ROWS(T, C)                                                                                             \
  hipLaunchKernelGGL((rows_kernel<T, C>), dim3((unsigned)rows), dim3(256), 0, s, (const T*)hidden, ld_hidden, state, \
                     rows, (int)dim, (C)scale, (T*)out, ld_out)
    if (dtype == TS_BF16) TS_ROWS(ts::bf16, float);
    else if (dtype == TS_F16) TS_ROWS(ts::f16, float);
    else if (dtype == TS_F32) TS_ROWS(float, float);
    else TS_ROWS(double, double);
#undef TS_ROWS
  }
  return ts::check_launch("ts_distill_rows");
}

}  // extern "C"
