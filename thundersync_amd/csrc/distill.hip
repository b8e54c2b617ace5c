// Distillation from a teacher's top logits through the head, for gfx950: the per-row
// divergence of the student's softmax over the whole vocabulary from the teacher's over
// its K returned tokens, and its gradient, without a [N, V] block of logits.
//
//   z[n, v] = h[n] . W[v],  q[n] = softmax_v(z[n] / T),  p[n] = softmax over the row's
//   present slots of teacher[n] / T, the slots of one token added together
//   loss[n] = sum_k p_k (log p_k - log q_k),  dz[n, v] = g[n] / T (q_v - p_v)
//
// teacher_kernel turns each row's slots into (token, p).  16-bit types: stats_kernel reduces
// the logits of a 256-row vocabulary tile to (reference, sum exp) per token in its MFMA epilogue
// and, where the block is wanted, stores the tile's exponentials in the element type;
// scores_kernel takes the logits at the slots' tokens as dot products; loss_kernel merges the
// tiles and sums the slots.  One pass over 2 bytes an entry then stands in place of a second
// product of 2 D flops an entry.  Frozen head: softmax_kernel shifts the exponentials by whole
// octaves to one reference a row (no second rounding) and clears the slots' tokens, and
// slots_kernel adds these to the block's product with W in fp32.  Trainable head, whose block
// holds the upstream gradient: finish_kernel scales them to q and writes the slots' entries
// from their fp32 logits; where the block would outgrow its bound, dlogits_kernel forms it from
// the logits again.  fp32 and fp64: the logits of a block of rows by the exact product, then
// one work-group a row.  The vector-Jacobian products with W and h are the fused logprob's.
// Bound by the products (the fused logprob's GEMM core).
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
constexpr int kRowThreads = 512;  // of the kernels that give a row a work-group, at most
constexpr int64_t kMaxRows = (1ll << 32) / kRowThreads;  // a launch of 2^32 threads along an axis wraps
constexpr int kRowWaves = 4;    // rows per work-group of the per-row kernels
constexpr int kDead = 0, kLive = 1, kBadId = 2;  // row states
// octaves of a frozen head's stored softmax above 1.  fp16's largest number leaves 5 more, for logits over T of up
// to 1e8: in fp32 they step by 8 octaves and lie up to 4 above their tile's reference
constexpr int kHeadroom = 10;

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
// them, the others become absent; K <= 1024 comparisons a slot, from LDS.  Latency: 10 us at
// 2048 rows of 64 slots, 20 us at 1999 of 100, beside milliseconds of products.
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
// forward: per (vocabulary tile, token) reference and sum exp of z / T.  The reference is the
// tile's maximum in octaves (of z log2(e) / T), rounded up to a whole one: exponentials of two
// tiles differ by a power of two, which a 16-bit value is scaled by without another rounding.
//
// Few rows are bound by the weight's one read (48 rows, D 4096, V 151936: 286 us, 4.4 TB/s),
// many by MFMA at the power-limited clock: 2048 rows take 2.23 ms with the exponentials stored,
// 1144 TFLOP/s, MFMA 65 % busy.  A wide tile's epilogue (an exponential an entry, the tile
// staged through the ring's LDS) overlaps nothing, which is the distance to the 1373 TFLOP/s
// that grad_hidden reaches at the same sizes.
// ---------------------------------------------------------------------------
// (reference r, sum 2^(z unit - r)) of two disjoint sets of logits, either of which may be
// empty (r = -inf, sum 0); unit = log2(e) / T.  A set that holds a NaN has a NaN sum.
__device__ __forceinline__ void merge(float& m, float& s, float mo, float so) {
  if (mo == neg_inf() || m == neg_inf()) {
    m = fmaxf(m, mo);
    s += so;
    return;
  }
  const float mn = fmaxf(m, mo);
  s = fast_exp2(m - mn) * s + fast_exp2(mo - mn) * so;
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
  float* part_m;   // [n_vtiles][rows]: references
  float* part_s;
  bf16* exps;      // STORE: [rows][lde], 2^(z unit - the tile's reference) in E (pad columns 0)
  int64_t lde;
  int vocab_pad;
};

template <class S> constexpr int kPasses = S::BN > TN ? S::WN : 1;  // halves of a Wide tile take turns in the staging

// coalesced store of the staged [PT tokens][TM vocabulary rows] of one pass
template <class S, class Quarter>
__device__ __forceinline__ void store_staged(Quarter&& quarter, bf16* out, int64_t ld, int n0, int rows, int v0,
                                             int vocab_pad, int pass) {
  constexpr int PT = S::BN / kPasses<S>;
  const int vmax = min(TM, vocab_pad - v0);
#pragma unroll 4
  for (int it = 0; it < (PT * TM / 8) / kGemmThreads; ++it) {
    const int c = it * kGemmThreads + threadIdx.x;
    const int row = c / (TM / 8), chunk = (c % (TM / 8)) * 8;
    const int n = n0 + pass * PT + row;
    if (n < rows && chunk < vmax)
      *reinterpret_cast<u32x4*>(out + (int64_t)n * ld + v0 + chunk) =
          *reinterpret_cast<const u32x4*>(quarter(row >> 6) + (row & 63) * OPITCH + chunk);
  }
}

// The tile's maximum is exchanged between the waves before the exponentials are formed, so
// that all of a token's exponentials of the tile are relative to one number.  With STORE they
// are staged through the ring as 16-bit values: tokens 64 q .. 64 q + 63 in stage q.
template <typename E, class S, bool STORE>
__device__ __forceinline__ void stats_tile(const StatsArgs& p, bf16* s0, bf16* s1, bf16* s2, bf16* s3, float* xm,
                                           float* xs) {
  constexpr int MI = S::MI, NI = S::NI, PASSES = kPasses<S>;
  int vt, tt;
  grouped_tile(xcd_logical(blockIdx.x, p.n_ttiles * p.n_vtiles), p.n_vtiles, p.n_ttiles, vt, tt);
  const int v0 = vt * TM, n0 = tt * S::BN;
  f32x16 acc[MI][NI];
  gemm_tile<E, false, false, S>(acc, p.w + (int64_t)v0 * p.ldw, p.ldw, min(TM, p.vocab - v0),
                                p.h + (int64_t)n0 * p.ldh, p.ldh, min(S::BN, p.rows - n0), p.dim, s0, s1, s2, s3);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave % S::WM, wn = wave / S::WM;
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
    float m = neg_inf();
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int i = 0; i < 16; i += 2) m = fmaxf(m, fmaxf(acc[mi][ni][i], acc[mi][ni][i + 1]));
    mk[ni] = fmaxf(m, shfl_xor(m, 32));  // lane ^ 32 holds the column's other rows
    if (lane < 32) xm[wm * S::BN + b_row<S>(ni, lane, wn)] = mk[ni];
  }
  __syncthreads();
#pragma unroll
  for (int ni = 0; ni < NI; ++ni)
#pragma unroll
    for (int w = 0; w < S::WM; ++w) mk[ni] = fmaxf(mk[ni], xm[w * S::BN + b_row<S>(ni, lane, wn)]);
#pragma unroll
  for (int ni = 0; ni < NI; ++ni) mk[ni] = ceilf(mk[ni] * p.unit);
  auto quarter = [&](int q) -> bf16* { return q == 0 ? s0 : q == 1 ? s1 : q == 2 ? s2 : s3; };
  auto values = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
      float sum = 0.f;
      // nothing, or nothing but -inf and NaN, which a maximum does not show
      const bool none = mk[ni] == neg_inf();
      const int col = b_row<S>(ni, lane, PASSES > 1 ? 0 : wn);  // token within the pass
      bf16* out = quarter(col >> 6) + (col & 63) * OPITCH;
#pragma unroll
      for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          float e[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = acc[mi][ni][4 * i4 + j];
            e[j] = none ? (x == neg_inf() ? 0.f : __builtin_nanf("")) : fast_exp2(fmaf(x, p.unit, -mk[ni]));
            sum += e[j];
          }
          if (STORE)
            *reinterpret_cast<u32x2*>(out + a_row<S>(mi, 4 * i4, lane, wm)) =
                u32x2{pack2<E>(e[0], e[1]), pack2<E>(e[2], e[3])};
        }
      sk[ni] = sum;
      if (STORE && PASSES > 1) __builtin_amdgcn_sched_barrier(0);
    }
  };
  if constexpr (!STORE) {
    values();
  } else if constexpr (PASSES == 1) {
    values();
    __syncthreads();
    store_staged<S>(quarter, p.exps, p.lde, n0, p.rows, v0, p.vocab_pad, 0);
  } else {
    static_assert(PASSES == 2, "two halves");
    if (wn == 0) values();
    __syncthreads();
    store_staged<S>(quarter, p.exps, p.lde, n0, p.rows, v0, p.vocab_pad, 0);
    __syncthreads();
    if (wn == 1) values();
    __syncthreads();
    store_staged<S>(quarter, p.exps, p.lde, n0, p.rows, v0, p.vocab_pad, 1);
  }
#pragma unroll
  for (int ni = 0; ni < NI; ++ni) {
    const int col = b_row<S>(ni, lane, wn);
    const float so = shfl_xor(sk[ni], 32);
    sk[ni] += so;
    if (wm > 0 && lane < 32) xs[(wm - 1) * S::BN + col] = sk[ni];
  }
  __syncthreads();
#pragma unroll
  for (int ni = 0; ni < NI; ++ni) {
    const int col = b_row<S>(ni, lane, wn), n = n0 + col;
    if (wm == 0 && lane < 32 && n < p.rows) {
#pragma unroll
      for (int w = 0; w < S::WM - 1; ++w) sk[ni] += xs[w * S::BN + col];
      p.part_m[(int64_t)vt * p.rows + n] = mk[ni];
      p.part_s[(int64_t)vt * p.rows + n] = sk[ni];
    }
  }
}

template <typename E, class S>
__global__ __launch_bounds__(kGemmThreads, 1) void stats_kernel(StatsArgs p) {
  GEMM_RING_OF(S)
  float* xm = reinterpret_cast<float*>(s0);
  stats_tile<E, S, false>(p, s0, s1, s2, s3, xm, xm + S::WM * S::BN);
}

template <typename E, class S>
__global__ __launch_bounds__(kGemmThreads, 1) void stats_store_kernel(StatsArgs p) {
  GEMM_RING_OF(S)
  __shared__ float xm[S::WM * S::BN], xs[S::WM * S::BN];  // the ring holds the staged values meanwhile
  stats_tile<E, S, true>(p, s0, s1, s2, s3, xm, xs);
}

// ---------------------------------------------------------------------------
// the logits at the slots: z[n, k] = h[n] . W[slot_id[n, k]], a wave per slot.  Bound by the
// gathered rows of W: 2048 x 64 slots of 8 KB, 1.07 GB, in 150 us.  (Taken from the product's
// epilogue instead they would cost no read, and every tile a search of its tokens' slots.)
// ---------------------------------------------------------------------------
template <typename E>
__global__ __launch_bounds__(256) void scores_kernel(const bf16* __restrict__ h, int64_t ldh,
                                                     const bf16* __restrict__ w, int64_t ldw,
                                                     const int32_t* __restrict__ slot_id, int pitch, int top, int dim,
                                                     float* __restrict__ z) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n = blockIdx.x;
  const E* hr = reinterpret_cast<const E*>(h + n * ldh);
  for (int k = 4 * blockIdx.y + wave; k < top; k += 4 * gridDim.y) {
    const int id = slot_id[n * pitch + k];
    if (id < 0) continue;
    const E* wr = reinterpret_cast<const E*>(w + (int64_t)id * ldw);
    float acc = 0.f;
    for (int d = 8 * lane; d < dim; d += 512) {
      float a[8], b[8];
      load8(hr + d, a);
      load8(wr + d, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc = fmaf(a[i], b[i], acc);
    }
    acc = wave_sum(acc);
    if (lane == 0) z[n * pitch + k] = acc;
  }
}

// sum_k p_k (log p_k - (z_k / T - lse)) over a wave's slots of one row
template <typename C>
__device__ __forceinline__ C slots_loss(const int32_t* slot_id, const C* slot_p, const C* slot_z, int top, C inv_t,
                                        C lse, int lane, int lanes) {
  C sum = (C)0;
  for (int k = lane; k < top; k += lanes) {
    if (slot_id[k] < 0) continue;
    const C p = slot_p[k];
    if (p == (C)0) continue;
    sum += p * (log(p) - (slot_z[k] * inv_t - lse));
  }
  return sum;
}
template <typename C> __device__ __forceinline__ C row_loss(int state, C sum) {
  return state == kDead ? (C)0 : state == kBadId ? (C)__builtin_nan("") : sum;
}

// ---------------------------------------------------------------------------
// lse of z / T from the tiles' statistics, and the loss.  A work-group of 16 waves owns 16
// tokens: its 64 slots of 16 lanes merge the tiles t = slot, slot + 64, ..., then wave w
// sums token w's teacher slots.  Latency: 11 us at 48 rows, 12 us at 2048.
// ---------------------------------------------------------------------------
constexpr int kLossTokens = 16;
__global__ __launch_bounds__(64 * kLossTokens) void loss_kernel(const float* __restrict__ pm,
                                                                const float* __restrict__ ps, int n_vtiles, int rows,
                                                                const int32_t* __restrict__ slot_id,
                                                                const float* __restrict__ slot_p,
                                                                const float* __restrict__ slot_z, int pitch, int top,
                                                                const int32_t* __restrict__ state, float inv_t,
                                                                float* __restrict__ lse, float* __restrict__ loss,
                                                                float2* __restrict__ row_scale) {
  __shared__ float sm[kLossTokens][kLossTokens], ss[kLossTokens][kLossTokens];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n0 = blockIdx.x * kLossTokens;
  {
    const int tok = lane & 15, slot = 4 * wave + (lane >> 4), n = n0 + tok;
    float M = neg_inf(), S = 0.f;
    if (n < rows) {
#pragma unroll 4
      for (int t = slot; t < n_vtiles; t += 64) {
        const int64_t o = (int64_t)t * rows + n;
        merge(M, S, pm[o], ps[o]);
      }
    }
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) {
      const float mo = shfl_xor(M, o), so = shfl_xor(S, o);
      merge(M, S, mo, so);
    }
    if (lane < 16) {
      sm[wave][tok] = M;
      ss[wave][tok] = S;
    }
    __syncthreads();
  }
  const int n = n0 + wave;
  if (n >= rows) return;
  float M = sm[0][wave], S = ss[0][wave];
#pragma unroll
  for (int v = 1; v < kLossTokens; ++v) merge(M, S, sm[v][wave], ss[v][wave]);
  const float l = M * kLn2 + logf(S);
  const int64_t o = (int64_t)n * pitch;
  const float sum = wave_sum(slots_loss(slot_id + o, slot_p + o, slot_z + o, top, inv_t, l, lane, 64));
  if (lane == 0) {
    lse[n] = l;
    loss[n] = row_loss(state[n], sum);
    if (row_scale) row_scale[n] = float2{M - kHeadroom, 1.f / (ldexpf(1.f, kHeadroom) * S)};
  }
}

// ---------------------------------------------------------------------------
// Frozen head, after the forward: the stored exponentials of a row to one reference, the
// softmax then being row_scale[1] times the block, and zero at the slots' tokens.  An entry
// keeps its one rounding: it is multiplied by a power of two, and kHeadroom octaves above 1
// leave fp16's smallest normal number 24 below the row's largest (unscaled, the softmax of
// 151936 equal logits is 6.6e-6 with four bits of it lost).  Bound as finish_kernel: 2048 x
// 151936 in bf16 in 211 us, 5.9 TB/s.
// ---------------------------------------------------------------------------
constexpr int kFinish = 2048;  // columns of one row a work-group: 256 threads of 8
template <typename T>
__global__ __launch_bounds__(256) void softmax_kernel(T* __restrict__ block, int64_t ld,
                                                      const float* __restrict__ tile_ref,
                                                      const float2* __restrict__ row_scale, int rows,
                                                      const int32_t* __restrict__ state,
                                                      const int32_t* __restrict__ slot_id, int pitch, int top,
                                                      int columns) {
  const int64_t n = blockIdx.x;
  const int c0 = blockIdx.y * kFinish, c = c0 + 8 * threadIdx.x;
  const bool dead = state[n] == kDead;
  if (c < columns) {  // a multiple of 8
    float x[8];
    load8(block + n * ld + c, x);
    // (a reference that is no number belongs to a row whose factor is none)
    const float f = ldexpf(1.f, (int)fmaxf(tile_ref[(int64_t)(c / TM) * rows + n] - row_scale[n].x, -200.f));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = dead ? 0.f : x[i] * f;
    store8(block + n * ld + c, x);
  }
  if (dead) return;
  __syncthreads();  // the slots' entries after the others'
  for (int k = threadIdx.x; k < top; k += 256) {
    const int id = slot_id[n * pitch + k];
    if (id >= c0 && id < c0 + kFinish) block[n * ld + id] = from_f<T>(0.f);
  }
}

// unit[n] = factor[n] unit[n] + sum_k (q_k - p_k) W[slot_id[n, k]], all in fp32: the slots are
// the gradient's largest terms, and rounded in the block they alone made the error 1.4 times that
// of the result's rounding.  A work-group takes 512 columns of one row, its waves every fourth
// slot each, added in wave order.  Bound by the gathered rows of W: 2048 x 64 slots of
// 8 KB, 1.07 GB, in 180 us.
template <typename E>
__global__ __launch_bounds__(256) void slots_kernel(float* __restrict__ unit, const float2* __restrict__ row_scale,
                                                    const E* __restrict__ w, int64_t ldw,
                                                    const int32_t* __restrict__ slot_id,
                                                    const float* __restrict__ slot_p,
                                                    const float* __restrict__ slot_z, int pitch, int top, int dim,
                                                    float inv_t, const float* __restrict__ lse) {
  __shared__ float part[3][8][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n = blockIdx.x, o = n * pitch;
  const int d = 512 * blockIdx.y + 8 * lane;
  const bool on = d < dim;  // a multiple of 8
  const float l = lse[n];
  float acc[8] = {};
#pragma unroll 4
  for (int k = wave; k < top; k += 4) {
    const int id = slot_id[o + k];
    if (id < 0) continue;
    const float c = expf(slot_z[o + k] * inv_t - l) - slot_p[o + k];
    float x[8];
    if (on) load8(w + (int64_t)id * ldw + d, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = on ? fmaf(c, x[i], acc[i]) : 0.f;
  }
  if (wave > 0)
#pragma unroll
    for (int i = 0; i < 8; ++i) part[wave - 1][i][lane] = acc[i];
  __syncthreads();
  if (wave > 0 || !on) return;
  const float f = row_scale[n].y;
  float* out = unit + n * dim + d;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int v = 0; v < 3; ++v) acc[i] += part[v][i][lane];
    out[i] = fmaf(out[i], f, acc[i]);
  }
}

// ---------------------------------------------------------------------------
// dlogits = grad / T (q - p) (grad null: q - p, without the 1 / T) from what the forward
// stored: a work-group takes kFinish columns of one row.  E: exponentials relative to their
// 256-column tile's reference (FROM_EXPS), scaled once per tile; C: logits.  Bound by the
// block's bytes, read and written once: 2048 x 151936 in bf16 in 211 us, 5.9 TB/s.
// ---------------------------------------------------------------------------
template <typename T, typename C, bool FROM_EXPS>
__global__ __launch_bounds__(256) void finish_kernel(const T* src, int64_t lds, const float* __restrict__ tile_ref,
                                                     int tile_rows, const C* __restrict__ lse,
                                                     const C* __restrict__ grad, const int32_t* __restrict__ state,
                                                     const int32_t* __restrict__ slot_id, const C* __restrict__ slot_p,
                                                     const C* __restrict__ slot_z, int pitch, int top, int columns,
                                                     C inv_t, T* dst, int64_t ldd) {
  const int64_t n = blockIdx.x;
  const int c0 = blockIdx.y * kFinish, c = c0 + 8 * threadIdx.x;
  const bool dead = state[n] == kDead;
  const C l = lse[n], coef = grad ? grad[n] * inv_t : (C)1;
  if constexpr (FROM_EXPS) {
    if (c < columns) {  // a multiple of 8
      float x[8];
      load8(src + n * lds + c, x);
      const float f = fast_exp2(fmaf(-l, kLog2e, tile_ref[(int64_t)(c / TM) * tile_rows + n])) * coef;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = dead ? 0.f : x[i] * f;
      store8(dst + n * ldd + c, x);
    }
  } else {
    for (int i = threadIdx.x; i < kFinish; i += 256) {
      if (c0 + i >= columns) break;
      const C q = exp(src[n * lds + c0 + i] * inv_t - l);
      dst[n * ldd + c0 + i] = dead ? (C)0 : q * coef;
    }
  }
  if (dead) return;
  __syncthreads();  // the slots' entries after the others', rounded once from their own logits
  for (int k = threadIdx.x; k < top; k += 256) {
    const int64_t o = n * pitch + k;
    const int id = slot_id[o];
    if (id < c0 || id >= c0 + kFinish) continue;
    const C d = (exp(slot_z[o] * inv_t - l) - slot_p[o]) * coef;
    if constexpr (std::is_same_v<T, C>) dst[n * ldd + id] = d;
    else dst[n * ldd + id] = from_f<T>((float)d);
  }
}

// ---------------------------------------------------------------------------
// fp32 / fp64: lse, the slots' logits and the loss from a row of logits, a work-group a row.
// 50 us at 600 x 32003 in fp32, beside 1.2 ms of the three products (0.4 ms each, 99 TFLOP/s
// of fp32 MFMA).
// ---------------------------------------------------------------------------
template <typename C>
__global__ __launch_bounds__(kRowThreads) void row_stats_kernel(const C* __restrict__ z, int64_t ldz, int vocab,
                                                                C inv_t, const int32_t* __restrict__ slot_id,
                                                                const C* __restrict__ slot_p, C* __restrict__ slot_z,
                                                                int pitch, int top, const int32_t* __restrict__ state,
                                                                C* __restrict__ lse, C* __restrict__ loss) {
  __shared__ C sm[kRowThreads / 64], ss[kRowThreads / 64];
  const int64_t n = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const C* row = z + n * ldz;
  // the maximum (a NaN of the row shows in the sum)
  C m = -(C)__builtin_huge_val();
  for (int v = threadIdx.x; v < vocab; v += kRowThreads) m = fmax(m, row[v]);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) m = fmax(m, __shfl_xor(m, o, kWave));
  if (lane == 0) sm[wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowThreads / 64; ++w) m = fmax(m, sm[w]);
  C s = (C)0;
  for (int v = threadIdx.x; v < vocab; v += kRowThreads) s += exp((row[v] - m) * inv_t);
  s = wave_sum_of(s);
  if (lane == 0) ss[wave] = s;
  __syncthreads();
  s = ss[0];
#pragma unroll
  for (int w = 1; w < kRowThreads / 64; ++w) s += ss[w];
  const C l = m * inv_t + log(s);
  if (wave != 0) return;
  const int64_t o = n * pitch;
  for (int k = lane; k < top; k += 64)
    if (slot_id[o + k] >= 0) slot_z[o + k] = row[slot_id[o + k]];
  const C sum = wave_sum_of(slots_loss(slot_id + o, slot_p + o, slot_z + o, top, inv_t, l, lane, 64));
  if (lane == 0) {
    lse[n] = l;
    loss[n] = row_loss(state[n], sum);
  }
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
  constexpr int PASSES = kPasses<S>;
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
  auto store = [&](int pass) __attribute__((always_inline)) {
    store_staged<S>(quarter, p.dl, p.ldl, n0, p.rows, v0, p.vocab_pad, pass);
  };
  if constexpr (PASSES == 1) {
    values();
    __syncthreads();
    store(0);
  } else {
    static_assert(PASSES == 2, "two halves");
    if (wn == 0) values();
    __syncthreads();
    store(0);
    __syncthreads();
    if (wn == 1) values();
    __syncthreads();
    store(1);
  }
}

// dl[n, slot_id] = grad / T (q - p) with q = exp(z / T - lse), rounded once
template <typename E>
__global__ __launch_bounds__(256) void dlogits_slots_kernel(const int32_t* __restrict__ slot_id,
                                                            const float* __restrict__ slot_p,
                                                            const float* __restrict__ slot_z, int pitch, int top,
                                                            int64_t rows, const float* __restrict__ lse,
                                                            const float* __restrict__ g, float inv_t,
                                                            E* __restrict__ dl, int64_t ldl) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t n = i / pitch;
  const int k = (int)(i - n * pitch);
  if (n >= rows || k >= top) return;
  const int id = slot_id[i];
  if (id >= 0) dl[n * ldl + id] = from_f<E>((expf(slot_z[i] * inv_t - lse[n]) - slot_p[i]) * (g[n] * inv_t));
}

// out[n] = h[n], zeros where the row has no teacher
template <typename T>
__global__ __launch_bounds__(256) void rows_kernel(const T* __restrict__ h, int64_t ldh,
                                                   const int32_t* __restrict__ state, int dim, T* __restrict__ out) {
  const int64_t n = blockIdx.x;
  const bool dead = state[n] == kDead;
  for (int d = threadIdx.x; d < dim; d += 256) out[n * dim + d] = dead ? (T)0.f : h[n * ldh + d];
}

// out[n] = grad[n] / T unit[n], zeros where the row has no teacher, rounded once
template <typename T, typename C>
__global__ __launch_bounds__(256) void scale_kernel(const C* __restrict__ unit, const C* __restrict__ grad,
                                                    const int32_t* __restrict__ state, int dim, C inv_t,
                                                    T* __restrict__ out) {
  const int64_t n = blockIdx.x;
  const bool dead = state[n] == kDead;
  const C f = grad[n] * inv_t;
  for (int d = threadIdx.x; d < dim; d += 256) {
    const C x = dead ? (C)0 : unit[n * dim + d] * f;
    if constexpr (std::is_same_v<T, C>) out[n * dim + d] = x;
    else out[n * dim + d] = from_f<T>((float)x);
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
  TS_CHECK_ARG(rows >= 0 && rows < kMaxRows && top > 0 && top <= kMaxTop && vocab > 0 && vocab < (1 << 30) &&
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

int ts_distill_fwd(const void* hidden, int64_t ld_hidden, const void* weight, int64_t ld_weight, int64_t rows,
                   int64_t dim, int64_t vocab, double temperature, const int32_t* slot_id, const float* slot_p,
                   float* slot_z, int64_t pitch, int64_t top, const int32_t* state, float* loss, float* lse,
                   void* exps, int64_t ld_exps, float* row_scale, void* workspace, int64_t workspace_bytes, int dtype,
                   void* stream) {
  TS_CHECK_ARG(dtype == TS_BF16 || dtype == TS_F16, "ts_distill_fwd: dtype %d (bf16 or fp16)", dtype);
  TS_CHECK_ARG(rows >= 0 && dim > 0 && vocab > 0 && rows < kMaxRows && vocab < (1 << 30) && dim < (1 << 20) &&
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
  TS_CHECK_ARG(!exps || (ok16(exps) && ld_exps % 8 == 0 && ld_exps >= (vocab + 7) / 8 * 8),
               "ts_distill_fwd: exps' alignment or leading dimension");
  TS_CHECK_ARG(((uintptr_t)row_scale & 7) == 0, "ts_distill_fwd: row_scale must be 8-byte aligned");
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
  a.exps = (ts::bf16*)exps;
  a.lde = ld_exps;
  a.vocab_pad = (int)((vocab + 7) / 8 * 8);
  TS_CHECK_ARG((int64_t)a.n_ttiles * a.n_vtiles < kMaxGrid, "ts_distill_fwd: grid too large");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("distill.stats_kernel", s);
    const dim3 grid((unsigned)(a.n_ttiles * a.n_vtiles));
    if (exps) TS_LAUNCH_TOKENS(dtype, width, stats_store_kernel, grid, dim3(kGemmThreads), 0, s, a);
    else TS_LAUNCH_TOKENS(dtype, width, stats_kernel, grid, dim3(kGemmThreads), 0, s, a);
  }
  int st = ts::check_launch("ts_distill_fwd (tiles)");
  if (st != TS_OK) return st;
  {
    ts::TimedLaunch timed_("distill.scores_kernel", s);
    TS_LAUNCH_E(dtype, scores_kernel, dim3((unsigned)rows, (unsigned)std::min<int64_t>((top + 3) / 4, 8)), dim3(256), 0,
                s, a.h, ld_hidden, a.w, ld_weight, slot_id, (int)pitch, (int)top, (int)dim, slot_z);
  }
  {
    ts::TimedLaunch timed_("distill.loss_kernel", s);
    hipLaunchKernelGGL(loss_kernel, dim3((unsigned)((rows + kLossTokens - 1) / kLossTokens)), dim3(64 * kLossTokens),
                       0, s, a.part_m, a.part_s, a.n_vtiles, (int)rows, slot_id, slot_p, slot_z, (int)pitch, (int)top,
                       state, (float)(1. / temperature), lse, loss, (float2*)row_scale);
  }
  return ts::check_launch("ts_distill_fwd (loss)");
}

int ts_distill_fwd_exact(const void* logits, int64_t ld_logits, int64_t rows, int64_t vocab, double temperature,
                         const int32_t* slot_id, const void* slot_p, void* slot_z, int64_t pitch, int64_t top,
                         const int32_t* state, void* loss, void* lse, int dtype, void* stream) {
  TS_CHECK_ARG(dtype == TS_F32 || dtype == TS_F64, "ts_distill_fwd_exact: dtype %d (fp32 or fp64)", dtype);
  TS_CHECK_ARG(rows >= 0 && rows < kMaxRows && vocab > 0 && vocab < (1 << 30) && ld_logits >= vocab && top > 0 &&
                   top <= pitch && pitch <= kMaxTop,
               "ts_distill_fwd_exact: bad shape");
  TS_CHECK_ARG(temperature > 0 && temperature < __builtin_huge_val(), "ts_distill_fwd_exact: temperature %g",
               temperature);
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(logits && slot_id && slot_p && slot_z && state && loss && lse, "ts_distill_fwd_exact: null pointer");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("distill.row_stats_kernel", s);
    const dim3 grid((unsigned)rows), block(kRowThreads);
    if (dtype == TS_F64)
      hipLaunchKernelGGL(row_stats_kernel<double>, grid, block, 0, s, (const double*)logits, ld_logits, (int)vocab,
                         1. / temperature, slot_id, (const double*)slot_p, (double*)slot_z, (int)pitch, (int)top, state,
                         (double*)lse, (double*)loss);
    else
      hipLaunchKernelGGL(row_stats_kernel<float>, grid, block, 0, s, (const float*)logits, ld_logits, (int)vocab,
                         (float)(1. / temperature), slot_id, (const float*)slot_p, (float*)slot_z, (int)pitch, (int)top,
                         state, (float*)lse, (float*)loss);
  }
  return ts::check_launch("ts_distill_fwd_exact");
}

int ts_distill_softmax(void* block, int64_t ld_block, const float* tile_ref, const float* row_scale, int64_t rows,
                       int64_t vocab, const int32_t* slot_id, int64_t pitch, int64_t top, const int32_t* state,
                       int dtype, void* stream) {
  TS_CHECK_ARG(dtype == TS_BF16 || dtype == TS_F16, "ts_distill_softmax: dtype %d (bf16 or fp16)", dtype);
  const int64_t columns = (vocab + 7) / 8 * 8;
  TS_CHECK_ARG(rows >= 0 && rows < kMaxRows && vocab > 0 && vocab < 65535ll * kFinish && top > 0 && top <= pitch &&
                   pitch <= kMaxTop && ld_block >= columns && ld_block % 8 == 0,
               "ts_distill_softmax: bad shape");
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(block && tile_ref && row_scale && slot_id && state, "ts_distill_softmax: null pointer");
  TS_CHECK_ARG(ok16(block) && ((uintptr_t)row_scale & 7) == 0, "ts_distill_softmax: alignment");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("distill.softmax_kernel", s);
    const dim3 grid((unsigned)rows, (unsigned)((columns + kFinish - 1) / kFinish));
    if (dtype == TS_F16)
      hipLaunchKernelGGL(softmax_kernel<ts::f16>, grid, dim3(256), 0, s, (ts::f16*)block, ld_block, tile_ref,
                         (const float2*)row_scale, (int)rows, state, slot_id, (int)pitch, (int)top, (int)columns);
    else
      hipLaunchKernelGGL(softmax_kernel<ts::bf16>, grid, dim3(256), 0, s, (ts::bf16*)block, ld_block, tile_ref,
                         (const float2*)row_scale, (int)rows, state, slot_id, (int)pitch, (int)top, (int)columns);
  }
  return ts::check_launch("ts_distill_softmax");
}

int ts_distill_slots(float* unit, const float* row_scale, const void* weight, int64_t ld_weight, int64_t rows,
                     int64_t dim, double temperature, const int32_t* slot_id, const float* slot_p, const float* slot_z,
                     int64_t pitch, int64_t top, const float* lse, int dtype, void* stream) {
  TS_CHECK_ARG(dtype == TS_BF16 || dtype == TS_F16, "ts_distill_slots: dtype %d (bf16 or fp16)", dtype);
  TS_CHECK_ARG(rows >= 0 && rows < kMaxRows && dim > 0 && dim < (1 << 20) && dim % 8 == 0 && ld_weight >= dim &&
                   ld_weight % 8 == 0 && top > 0 && top <= pitch && pitch <= kMaxTop,
               "ts_distill_slots: bad shape");
  TS_CHECK_ARG(temperature > 0 && temperature < __builtin_huge_val(), "ts_distill_slots: temperature %g", temperature);
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(unit && row_scale && weight && slot_id && slot_p && slot_z && lse, "ts_distill_slots: null pointer");
  TS_CHECK_ARG(ok16(weight) && ((uintptr_t)row_scale & 7) == 0, "ts_distill_slots: alignment");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("distill.slots_kernel", s);
    const dim3 grid((unsigned)rows, (unsigned)((dim + 511) / 512));
    if (dtype == TS_F16)
      hipLaunchKernelGGL(slots_kernel<ts::f16>, grid, dim3(256), 0, s, unit, (const float2*)row_scale,
                         (const ts::f16*)weight, ld_weight, slot_id, slot_p, slot_z, (int)pitch, (int)top, (int)dim,
                         (float)(1. / temperature), lse);
    else
      hipLaunchKernelGGL(slots_kernel<ts::bf16>, grid, dim3(256), 0, s, unit, (const float2*)row_scale,
                         (const ts::bf16*)weight, ld_weight, slot_id, slot_p, slot_z, (int)pitch, (int)top, (int)dim,
                         (float)(1. / temperature), lse);
  }
  return ts::check_launch("ts_distill_slots");
}

int ts_distill_finish(const void* stored, int64_t ld_stored, const float* tile_ref, int64_t rows, int64_t vocab,
                      double temperature, const int32_t* slot_id, const void* slot_p, const void* slot_z,
                      int64_t pitch, int64_t top, const int32_t* state, const void* lse, const void* grad,
                      void* dlogits, int64_t ld_dlogits, int dtype, void* stream) {
  TS_CHECK_ARG(known(dtype), "ts_distill_finish: dtype %d", dtype);
  const bool exact = dtype == TS_F32 || dtype == TS_F64;
  TS_CHECK_ARG(rows >= 0 && rows < kMaxRows && vocab > 0 && vocab < 65535ll * kFinish && top > 0 && top <= pitch &&
                   pitch <= kMaxTop && ld_stored >= vocab && ld_dlogits >= vocab,
               "ts_distill_finish: bad shape");
  TS_CHECK_ARG(temperature > 0 && temperature < __builtin_huge_val(), "ts_distill_finish: temperature %g", temperature);
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(stored && dlogits && slot_id && slot_p && slot_z && state && lse && (exact || tile_ref),
               "ts_distill_finish: null pointer");
  const int64_t columns = exact ? vocab : (vocab + 7) / 8 * 8;
  TS_CHECK_ARG(exact || (ok16(stored) && ok16(dlogits) && ld_stored % 8 == 0 && ld_dlogits % 8 == 0 &&
                         ld_stored >= columns && ld_dlogits >= columns),
               "ts_distill_finish: alignment or leading dimensions");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("distill.finish_kernel", s);
    const dim3 grid((unsigned)rows, (unsigned)((columns + kFinish - 1) / kFinish));
#define TS_FINISH(T, C, EXPS)                                                                                        \
  hipLaunchKernelGGL((finish_kernel<T, C, EXPS>), grid, dim3(256), 0, s, (const T*)stored, ld_stored, tile_ref,       \
                     (int)rows, (const C*)lse, (const C*)grad, state, slot_id, (const C*)slot_p, (const C*)slot_z,    \
                     (int)pitch, (int)top, (int)columns, (C)(1. / temperature), (T*)dlogits, ld_dlogits)
    if (dtype == TS_BF16) TS_FINISH(ts::bf16, float, true);
    else if (dtype == TS_F16) TS_FINISH(ts::f16, float, true);
    else if (dtype == TS_F32) TS_FINISH(float, float, false);
    else TS_FINISH(double, double, false);
#undef TS_FINISH
  }
  return ts::check_launch("ts_distill_finish");
}

int ts_distill_dlogits(const void* hidden, int64_t ld_hidden, const void* weight, int64_t ld_weight, int64_t rows,
                       int64_t dim, int64_t vocab, double temperature, const int32_t* slot_id, const float* slot_p,
                       const float* slot_z, int64_t pitch, int64_t top, const int32_t* state, const float* lse,
                       const float* grad, void* dlogits, int64_t ld_dlogits, int dtype, void* stream) {
  TS_CHECK_ARG(dtype == TS_BF16 || dtype == TS_F16, "ts_distill_dlogits: dtype %d (bf16 or fp16)", dtype);
  TS_CHECK_ARG(rows >= 0 && dim > 0 && vocab > 0 && rows < kMaxRows && vocab < (1 << 30) && dim < (1 << 20) &&
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
  TS_CHECK_ARG((int64_t)a.n_ttiles * a.n_vtiles < kMaxGrid, "ts_distill_dlogits: grid too large");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("distill.dlogits_kernel", s);
    TS_LAUNCH_TOKENS(dtype, width, dlogits_kernel, dim3((unsigned)(a.n_ttiles * a.n_vtiles)), dim3(kGemmThreads), 0, s, a);
  }
  const int st = ts::check_launch("ts_distill_dlogits");
  if (st != TS_OK) return st;
  {
    ts::TimedLaunch timed_("distill.dlogits_slots_kernel", s);
    const dim3 grid((unsigned)((rows * pitch + 255) / 256));
    const float inv_t = (float)(1. / temperature);
    if (dtype == TS_F16)
      hipLaunchKernelGGL(dlogits_slots_kernel<ts::f16>, grid, dim3(256), 0, s, slot_id, slot_p, slot_z, (int)pitch, (int)top,
                         rows, lse, grad, inv_t, (ts::f16*)dlogits, ld_dlogits);
    else
      hipLaunchKernelGGL(dlogits_slots_kernel<ts::bf16>, grid, dim3(256), 0, s, slot_id, slot_p, slot_z, (int)pitch, (int)top,
                         rows, lse, grad, inv_t, (ts::bf16*)dlogits, ld_dlogits);
  }
  return ts::check_launch("ts_distill_dlogits (slots)");
}

int ts_distill_rows(const void* hidden, int64_t ld_hidden, const int32_t* state, int64_t rows, int64_t dim, void* out,
                    int dtype, void* stream) {
  TS_CHECK_ARG(known(dtype), "ts_distill_rows: dtype %d", dtype);
  TS_CHECK_ARG(rows >= 0 && rows < kMaxRows && dim > 0 && dim < (1 << 20) && ld_hidden >= dim,
               "ts_distill_rows: bad shape");
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(hidden && state && out && hidden != out, "ts_distill_rows: null or aliased pointer");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("distill.rows_kernel", s);
#define TS_ROWS(T)                                                                                                   \
  hipLaunchKernelGGL(rows_kernel<T>, dim3((unsigned)rows), dim3(256), 0, s, (const T*)hidden, ld_hidden, state,       \
                     (int)dim, (T*)out)
    if (dtype == TS_BF16) TS_ROWS(ts::bf16);
    else if (dtype == TS_F16) TS_ROWS(ts::f16);
    else if (dtype == TS_F32) TS_ROWS(float);
    else TS_ROWS(double);
#undef TS_ROWS
  }
  return ts::check_launch("ts_distill_rows");
}

int ts_distill_scale(const void* unit, const void* grad, const int32_t* state, int64_t rows, int64_t dim,
                     double temperature, void* out, int dtype, void* stream) {
  TS_CHECK_ARG(known(dtype), "ts_distill_scale: dtype %d", dtype);
  TS_CHECK_ARG(rows >= 0 && rows < kMaxRows && dim > 0 && dim < (1 << 20), "ts_distill_scale: bad shape");
  TS_CHECK_ARG(temperature > 0 && temperature < __builtin_huge_val(), "ts_distill_scale: temperature %g", temperature);
  if (rows == 0) return TS_OK;
  TS_CHECK_ARG(unit && grad && state && out, "ts_distill_scale: null pointer");
  hipStream_t s = (hipStream_t)stream;
  {
    ts::TimedLaunch timed_("distill.scale_kernel", s);
#define TS_SCALE(T, C)                                                                                               \
  hipLaunchKernelGGL((scale_kernel<T, C>), dim3((unsigned)rows), dim3(256), 0, s, (const C*)unit, (const C*)grad,     \
                     state, (int)dim, (C)(1. / temperature), (T*)out)
    if (dtype == TS_BF16) TS_SCALE(ts::bf16, float);
    else if (dtype == TS_F16) TS_SCALE(ts::f16, float);
    else if (dtype == TS_F32) TS_SCALE(float, float);
    else TS_SCALE(double, double);
#undef TS_SCALE
  }
  return ts::check_launch("ts_distill_scale");
}

}  // extern "C"
