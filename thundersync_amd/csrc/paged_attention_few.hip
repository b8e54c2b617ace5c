// Attention over a paged cache for sequences with few query rows: one token each, or a few.
//
// A work-group takes one tile after another: up to 16 R query rows of one KV head (its tokens' heads of the group side by
// side, so that keys and values are read once for all of them) over its part of the keys.  Its four waves take 32-key steps in
// turn, each with a running reference point, sum and accumulators of its own, and join them at the end; a tile that is not
// all its own leaves partial rows for merge_kernel.
//
// A step of a wave:  S^T = K Q^T (16x16x32, keys as rows), so a lane holds 8 of the 32 scores of one query row, which
// are, rounded, already the operand of O^T += V^T P^T: lane (g, r) has keys 4 g + i of both halves of query row r.  V^T
// needs 8 keys of one element: a lane reads ROW / 16 elements of each of its 8 keys (a wave whole rows), and
// pairs of keys are interleaved by byte permutes; codes become 16-bit values, times their scale, two to an instruction.
// Nothing passes through LDS, and no wave waits for another before the end.
//
// Bound by HBM: a step's 32 ROW bytes of keys and as many of values against about 150 VALU instructions and 2 ROW / 8
// matrix ones.  256 sequences of 256 to 16384 keys, 32/8 heads of 128 in 8 bits, take 700 to 750 us, 5.9 TB/s; one of 125000
// 53, 4.8 TB/s; 64 of 256 to 4096 in 16 bits 102 to 124, 5.0 TB/s.  64 of 100 to 6000, one to five rows, 24/4 heads of 256:
// 103 us, 6.3 TB/s of what is read; wide rows have 16 a tile, so sequences of 17 to 32 query rows are read twice, and 4.1
// TB/s is what reading them once would be.
#include "paged_attention.h"

namespace ts {
namespace paged {

constexpr int kWaves = 4;

// N bytes of a lane, at a multiple of four from the descriptor's base and `more`, a constant.  Reads go through a
// descriptor of the 16 tokens: a lane's place in them is one register for all of a kernel, where a pointer is two more
// for each read.
template <int N> struct Words {
  uint32_t w[N / 4];
};
template <int N> __device__ __forceinline__ Words<N> load_words(rsrc_t r, uint32_t at, int more) {
  Words<N> y;
  if constexpr (N == 4) {
    y.w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, at, more, 0);
  } else if constexpr (N == 8) {
    const auto v = __builtin_amdgcn_raw_buffer_load_b64(r, at, more, 0);
    __builtin_memcpy(y.w, &v, 8);
  } else if constexpr (N == 12) {
    const auto v = __builtin_amdgcn_raw_buffer_load_b96(r, at, more, 0);
    __builtin_memcpy(y.w, &v, 12);
  } else {
    const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, at, more, 0);
    __builtin_memcpy(y.w, &v, 16);
    if constexpr (N > 16) {
      const Words<N - 16> z = load_words<N - 16>(r, at, more + 16);
#pragma unroll
      for (int i = 0; i < (N - 16) / 4; ++i) y.w[4 + i] = z.w[i];
    }
  }
  return y;
}

// A step's keys or values of one 16-token tile, as loaded.
template <bool WIDE, int ROW> struct Tile {
  static constexpr int kSize = WIDE ? 2 : 1;
  static constexpr int kLoads = ROW * kSize / 64;  // 16-byte reads of a key's row by its four lanes
  u32x4 k[kLoads];
  Words<ROW / 16 * kSize> v[4];
};

template <typename T, bool WIDE, int ROW, int R>
__global__ __launch_bounds__(64 * kWaves, (few_occupancy(WIDE, ROW, R))) void few_kernel(AttnArgs) {
  constexpr int NC = ROW / 32;  // k-steps of S
  constexpr int NB = ROW / 16;  // elements of a value that a lane reads, and tiles of O
  constexpr int kSize = WIDE ? 2 : 1;
  using Part = float[16 * R][ROW + 4];
  using Query = u32x4[NC][64];
  constexpr int kBytes = kWaves * sizeof(Part) > R * sizeof(Query) ? kWaves * sizeof(Part) : R * sizeof(Query);
  __shared__ __attribute__((aligned(16))) char s_space[kBytes];
  Part* const s_part = (Part*)s_space;     // at the end
  Query* const s_query = (Query*)s_space;  // until then
  __shared__ float s_stat[kWaves][16 * R][2];
  const int lane_id = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  __shared__ Cursor<0>::Kept s_at[2];
  Cursor<0> at{};
  AttnArgs a = arguments();
  int past = 0, turn = 0;
  if (wave == 0) {
    const bool some = at.begin(a, 16 * R, (int)blockIdx.x, lane_id, past);
    at.put(s_at[0], some, past);
  }
  __syncthreads();
  if (!at.take(s_at[0], &past)) {
    // rows before the first sequence and behind the last: 16 a work-group, zeros
    if (a.batch.offsets && past >= 0) {
      const int before = min(max(0, a.batch.offsets[0]), a.batch.tokens);
      const int behind = min(max(before, a.batch.offsets[a.batch.seqs]), a.batch.tokens);
      const int none = before + a.batch.tokens - behind, row_bytes = a.heads * a.head_dim * 2;
      for (int k = 16 * past; k < min(16 * past + 16, none); ++k) {
        const int t = k < before ? k : behind + k - before;
        for (int i = threadIdx.x; i < row_bytes / 16; i += 64 * kWaves)
          *(u32x4*)(a.out + (int64_t)t * row_bytes + 16 * i) = u32x4{0, 0, 0, 0};
      }
    }
    return;
  }
  for (;;) {
    a = arguments();
    int lane = lane_id;
    asm volatile("" : "+v"(lane));  // what follows from it is worked out again a tile, not held over the loop
    const int g = lane >> 4, r = lane & 15;
    const int first_row = at.tile * 16 * R;
    const int rows = at.seq.n * a.group;
    const int len = at.seq.len, base = len - at.seq.n;  // position of the first new token
    int begin, end;
    at.piece(a, begin, end);
    if (a.plan && threadIdx.x == 0 && at.head == 0 && at.tile == 0 && at.from == 0)
      a.plan[at.s] = Plan{at.end - at.left, at.blocks, at.per, 0};

    // Query rows as B operands: element 16 g + 8 (c & 1) of the 64 of c / 2 for codes, 32 c + 8 g in 16 bits, as the
    // keys' elements lie in a lane's reads; the last key that each row sees.  The operands are the same in
    // every wave and stay in LDS: their registers are worth more to loads in flight.
    int limit[R];
    u32x4 query[R][(NC + kWaves - 1) / kWaves];
#pragma unroll
    for (int t = 0; t < R; ++t) {
      const int row = first_row + 16 * t + r;
      const int token = row / a.group, head = at.head * a.group + row % a.group;
      const bool there = row < rows;
      limit[t] = there ? base + token : -1;
      const char* p = a.query + ((int64_t)(at.seq.row0 + token) * a.token_stride + (int64_t)head * a.head_stride) * 2;
#pragma unroll
      for (int k = 0; k < (NC + kWaves - 1) / kWaves; ++k) {
        const int c = wave + kWaves * k, d = WIDE ? 32 * c + 8 * g : 64 * (c / 2) + 16 * g + 8 * (c & 1);
        query[t][k] = u32x4{0, 0, 0, 0};
        if (there && d < a.head_dim) query[t][k] = *(const u32x4*)(p + 2 * d);
      }
    }
    const int low = max(-1, base + min(first_row / a.group, at.seq.n - 1));  // the least of the rows' limits

    f32x4 acc[R][NB];
    float m[R], l[R];
#pragma unroll
    for (int t = 0; t < R; ++t) {
      m[t] = neg_inf();
      l[t] = 0.f;
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    const int32_t* table = a.batch.table + (int64_t)at.s * a.batch.ld_table;
    const int page_mask = (1 << a.page_shift) - 1;
    auto page_at = [&](int pos) -> int {  // of a 16-token tile; wave-uniform
      const int nth = pos >> a.page_shift;
      if (pos >= end || nth >= a.batch.width) return -1;
      const int page = uniform_table(table)[nth];
      return page >= 0 && page < a.pages ? page : -1;
    };
    // The same without a branch, for positions before the end, in two parts: what is read and what it says.
    auto read_near = [&](int pos) -> int { return uniform_table(table)[min(pos >> a.page_shift, a.batch.width - 1)]; };
    auto page_near = [&](int pos, int page) -> int {
      return (pos >> a.page_shift) < a.batch.width && page >= 0 && page < a.pages ? page : -1;
    };
    // A page that is none is read as page 0, and its scores and values are not used.
    Tile<WIDE, ROW> tile[2];
    float ks0 = 1.f, ks1 = 1.f, vs0 = 1.f, vs1 = 1.f;  // of the step whose keys have been asked for
    int page0 = -1, page1 = -1;
    const uint32_t key_lane = (r * ROW + (WIDE ? 8 : 16) * g) * kSize;
    const uint32_t value_lane = (4 * g * ROW + NB * r) * kSize;
    auto line_of = [&](int pos) -> int64_t { return ((int64_t)at.head << a.page_shift) + (pos & page_mask); };
    auto load_tile_keys = [&](int pos, bool there, int page, u32x4 (&k)[Tile<WIDE, ROW>::kLoads], float& key_scale,
                              float& value_scale)
                              __attribute__((always_inline)) {
      const int id = max(page, 0);
      const rsrc_t p = make_rsrc(a.key + id * a.key_page_stride + line_of(pos) * (ROW * kSize),
                                 there ? 16 * ROW * kSize : 0);
#pragma unroll
      for (int i = 0; i < Tile<WIDE, ROW>::kLoads; ++i) {
        const Words<16> x = load_words<16>(p, key_lane, 64 * i);
        k[i] = u32x4{x.w[0], x.w[1], x.w[2], x.w[3]};
      }
      if constexpr (!WIDE) {
        const int64_t scale = (((int64_t)id * a.kv_heads << a.page_shift) + line_of(pos)) >> 4;
        key_scale = uniform_table(a.key_scale)[scale];
        value_scale = uniform_table(a.value_scale)[scale];
      }
    };
    // of the pages that page0 and page1 say; a step that is not there reads nothing
    auto load_keys = [&](int pos, bool there) __attribute__((always_inline)) {
      load_tile_keys(pos, there, page0, tile[0].k, ks0, vs0);
      load_tile_keys(pos + 16, there, page1, tile[1].k, ks1, vs1);
    };
    auto load_values = [&](int pos, bool there) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const rsrc_t p = make_rsrc(a.value + max(h ? page1 : page0, 0) * a.value_page_stride +
                                       line_of(pos + 16 * h) * (ROW * kSize), there ? 16 * ROW * kSize : 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) tile[h].v[i] = load_words<NB * kSize>(p, value_lane, i * ROW * kSize);
      }
    };

    int pos = __builtin_amdgcn_readfirstlane(begin + 32 * wave);
    // Steps before `whole` are seen whole by every row.  Their reads run a step ahead, their page ids two, and
    // unconditionally, so that every wait counts exactly what was asked for since; past the last one the descriptors are
    // empty, and nothing is read.  256 sequences of 256 to 16384 keys: 812 us where the last reads were skipped.
    const int whole = min(end, low + 1) - 31;
    constexpr int kStride = 32 * kWaves;
    int ahead0 = -1, ahead1 = -1;
    if (pos < whole) {
      page0 = page_near(pos, read_near(pos));
      page1 = page_near(pos + 16, read_near(pos + 16));
      load_keys(pos, true);
      load_values(pos, true);
      ahead0 = read_near(pos + kStride);
      ahead1 = read_near(pos + kStride + 16);
    }
#pragma unroll
    for (int t = 0; t < R; ++t)
#pragma unroll
      for (int k = 0; k < (NC + kWaves - 1) / kWaves; ++k)
        if (wave + kWaves * k < NC) s_query[t][wave + kWaves * k][lane] = query[t][k];
    __syncthreads();
    // One step; `edge`: some row does not see some of its keys, or they are not there.
    auto step = [&](auto edge_) __attribute__((always_inline)) {
      constexpr bool edge = decltype(edge_)::value;
      if constexpr (edge) {  // few, and nothing is asked for ahead of them: the registers are worth more
        page0 = page_at(pos);
        page1 = page_at(pos + 16);
        load_keys(pos, true);
        load_values(pos, true);
      }
      asm volatile("" ::: "memory");  // the query's operands are read again, not held over the loop
      f32x4 sc[R][2];
      const bool ruined0 = page0 < 0 && pos < end, ruined1 = page1 < 0 && pos + 16 < end;
      // the scale of a half behind the end is whatever its place holds, and a code of 0 times a NaN is one
      const float vscale0 = vs0, vscale1 = edge && pos + 16 >= end ? 1.f : vs1;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int t = 0; t < R; ++t) sc[t][h] = f32x4{0.f, 0.f, 0.f, 0.f};
        const float key_scale = h ? ks1 : ks0;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          bf16x8 k;
          if constexpr (WIDE) {
            k = as_bf16x8(tile[h].k[c]);
          } else {
            const u32x4 x = tile[h].k[c / 2];
            const uint32_t lo = x[2 * (c & 1)], hi = x[2 * (c & 1) + 1];
            k = as_bf16x8(u32x4{widen2<T, false>(lo, key_scale), widen2<T, true>(lo, key_scale),
                                widen2<T, false>(hi, key_scale), widen2<T, true>(hi, key_scale)});
          }
#pragma unroll
          for (int t = 0; t < R; ++t) sc[t][h] = mma16<T>(k, as_bf16x8(s_query[t][c][lane]), sc[t][h]);
        }
#pragma unroll
        for (int t = 0; t < R; ++t) sc[t][h] *= a.scale;
      }
      const int next = pos + kStride;
      if constexpr (!edge) {
        page0 = page_near(next, ahead0);
        page1 = page_near(next + 16, ahead1);
        load_keys(next, next < whole);
        ahead0 = read_near(next + kStride);
        ahead1 = read_near(next + kStride + 16);
      }

      if (ruined0 | ruined1) {  // keys of a page that is none
#pragma unroll
        for (int t = 0; t < R; ++t) {
          if (ruined0) sc[t][0] = f32x4{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
          if (ruined1) sc[t][1] = f32x4{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
        }
      }
      bf16x8 p[R];
#pragma unroll
      for (int t = 0; t < R; ++t) {
        if constexpr (edge) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (pos + 16 * h + 4 * g + i > limit[t]) sc[t][h][i] = neg_inf();
        }
        float e[8], sum;
        auto exponentials = [&]() __attribute__((always_inline)) {
          const float ref = m[t] == neg_inf() ? 0.f : m[t];
          sum = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            e[j] = fast_exp2(sc[t][j >> 2][j & 3] - ref);
            sum += e[j];
          }
        };
        exponentials();
        // They stand unless a score passes the reference point by more than kSlack, which shows in the sum.
        if (__ballot((m[t] == neg_inf()) | (sum > kSlackSum<T>))) {
          float most = neg_inf();
#pragma unroll
          for (int j = 0; j < 8; ++j) most = fmaxf(most, sc[t][j >> 2][j & 3]);
          most = rows_max4(most);
          const bool move = most > m[t] + (kSlack + kLift<T>) || (m[t] == neg_inf() && most > m[t]);
          const float to = move ? most - kLift<T> : m[t], alpha = move ? fast_exp2(m[t] - to) : 1.f;
          m[t] = to;
          l[t] *= alpha;
#pragma unroll
          for (int b = 0; b < NB; ++b) acc[t][b] *= alpha;
          exponentials();
        }
        l[t] += sum;
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pack2<T>(e[2 * j], e[2 * j + 1]);
        p[t] = as_bf16x8(w);
      }

      // Values of keys behind the sequence are zeros.
      if constexpr (edge) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool there = pos + 16 * h + 4 * g + i < len;
#pragma unroll
            for (int w = 0; w < NB * kSize / 4; ++w) tile[h].v[i].w[w] = there ? tile[h].v[i].w[w] : 0u;
          }
      }
      auto value = [&](int b) -> u32x4 {  // element NB r + b of the lane's eight keys
        u32x4 f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if constexpr (WIDE) {
              const uint32_t x = tile[h].v[2 * k].w[b / 2], y = tile[h].v[2 * k + 1].w[b / 2];
              f[2 * h + k] = __builtin_amdgcn_perm(y, x, b & 1 ? 0x07060302u : 0x05040100u);
            } else {
              const uint32_t x = tile[h].v[2 * k].w[b / 4], y = tile[h].v[2 * k + 1].w[b / 4];
              const uint32_t z = __builtin_amdgcn_perm(y, x, b & 2 ? 0x07030602u : 0x05010400u);
              const float scale = h ? vscale1 : vscale0;
              f[2 * h + k] = b & 1 ? widen2<T, true>(z, scale) : widen2<T, false>(z, scale);
            }
          }
        return f;
      };
      if (!edge || at.seq.n == 1) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const bf16x8 v = as_bf16x8(value(b));
#pragma unroll
          for (int t = 0; t < R; ++t) acc[t][b] = mma16<T>(v, p[t], acc[t][b]);
        }
      } else {
        // Rows differ in what they see, and a weight of 0 does not take a NaN out: values that are not finite are left out of
        // the product, and a second one, of where they are with who sees them, ruins the elements of the rows that do.
        u32x4 seen[R];
#pragma unroll
        for (int t = 0; t < R; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = pos + 16 * (j >> 1) + 4 * g + 2 * (j & 1);
            seen[t][j] = (key <= limit[t] ? kOneOf<T> : 0u) | (key + 1 <= limit[t] ? kOneOf<T> << 16 : 0u);
          }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const u32x4 f = value(b);
          u32x4 fine, flag;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t x, y;
            split_finite<T>(f[j], x, y);
            fine[j] = x;
            flag[j] = y;
          }
#pragma unroll
          for (int t = 0; t < R; ++t) {
            acc[t][b] = mma16<T>(as_bf16x8(fine), p[t], acc[t][b]);
            const f32x4 n = mma16<T>(as_bf16x8(flag), as_bf16x8(seen[t]), f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (n[i] > 0.f) acc[t][b][i] = __builtin_nanf("");
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if constexpr (!edge) load_values(next, next < whole);
      pos = next;
    };
    while (pos < whole) step(std::false_type{});
    while (pos < end) step(std::true_type{});
    __syncthreads();  // the query's operands have been read

    a = arguments();
    // The waves' sums by one reference point: through LDS, and added there in the waves' order, a row in 16 threads.
#pragma unroll
    for (int t = 0; t < R; ++t) {
      l[t] = rows_sum4(l[t]);
      if (g == 0) {
        s_stat[wave][16 * t + r][0] = m[t];
        s_stat[wave][16 * t + r][1] = l[t];
      }
      if (first_row + 16 * t + r < rows)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int b = 0; b < NB; b += 4)
            *(f32x4*)&s_part[wave][16 * t + r][NB * (4 * g + i) + b] =
                f32x4{acc[t][b][i], acc[t][b + 1][i], acc[t][b + 2][i], acc[t][b + 3][i]};
    }
    __syncthreads();
    at.take(s_at[turn]);
    {
      const bool all = at.whole();
      const int slot = at.slot(a.kv_heads);
      const int first_row = at.tile * 16 * R, here = min(16 * R, at.seq.n * a.group - first_row);
      int tid = threadIdx.x;
      asm volatile("" : "+v"(tid));
      for (int in = tid >> 4; in < here; in += 4 * kWaves) {
        float most = neg_inf();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) most = fmaxf(most, s_stat[w][in][0]);
        const float by = most == neg_inf() ? 0.f : most;
        float f[kWaves], sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          f[w] = fast_exp2(s_stat[w][in][0] - by);
          sum = fmaf(s_stat[w][in][1], f[w], sum);
        }
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
        const int row = first_row + in, token = row / a.group, head = at.head * a.group + row % a.group;
        char* o = a.out + (((int64_t)(at.seq.row0 + token) * a.heads + head) * a.head_dim) * 2;
        const int64_t to = (int64_t)slot * (16 * R) + in;
        float* part = a.part[0] + to * ROW;
#pragma unroll
        for (int k = 0; k < ROW / 64; ++k) {
          const int d = 64 * k + 4 * (tid & 15);
          f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < kWaves; ++w) {
            const f32x4 y = *(const f32x4*)&s_part[w][in][d];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = fmaf(y[i], f[w], x[i]);
          }
          if (!all) *(f32x4*)(part + d) = x;
          else if (d < a.head_dim)
            *(u32x2*)(o + 2 * d) = u32x2{pack2<T>(x[0] * inv, x[1] * inv), pack2<T>(x[2] * inv, x[3] * inv)};
        }
        if (!all && (tid & 15) == 0) {
          a.stats[0][2 * to] = most;
          a.stats[0][2 * to + 1] = sum;
        }
      }
    }
    turn ^= 1;
    if (wave == 0) {
      const bool more = at.next(a, 16 * R, lane_id);
      at.put(s_at[turn], more, 0);
    }
    __syncthreads();  // the next tile is known, and its operands go where the sums were
    if (!at.take(s_at[turn])) return;
  }
}

template <typename T, bool WIDE, int ROW>
void launch_few_rows(const AttnArgs& a, const Sizes& z, hipStream_t s) {
  const dim3 grid((unsigned)(z.groups[0] + (a.batch.offsets ? (a.batch.tokens + 15) / 16 : 0))), block(64 * kWaves);
  ts::TimedLaunch timed_("paged.few_kernel", s);
  if (z.rows[0] == 16) hipLaunchKernelGGL((few_kernel<T, WIDE, ROW, 1>), grid, block, 0, s, a);
  else if constexpr (ROW <= 128) hipLaunchKernelGGL((few_kernel<T, WIDE, ROW, 2>), grid, block, 0, s, a);
}

template <typename T, bool WIDE>
void launch_few_t(const AttnArgs& a, const Sizes& z, int row, hipStream_t s) {
  switch (row) {
    case 64: launch_few_rows<T, WIDE, 64>(a, z, s); break;
    case 128: launch_few_rows<T, WIDE, 128>(a, z, s); break;
    case 192: launch_few_rows<T, WIDE, 192>(a, z, s); break;
    default: launch_few_rows<T, WIDE, 256>(a, z, s);
  }
}

void launch_few(const AttnArgs& a, const Sizes& z, int dtype, bool wide, int row, hipStream_t s) {
  if (dtype == kF16) wide ? launch_few_t<f16, true>(a, z, row, s) : launch_few_t<f16, false>(a, z, row, s);
  else wide ? launch_few_t<bf16, true>(a, z, row, s) : launch_few_t<bf16, false>(a, z, row, s);
}

}  // namespace paged
}  // namespace ts
