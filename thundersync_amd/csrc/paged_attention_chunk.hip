// Attention over a paged cache for sequences with many query rows: chunks of a prompt.
//
// A work-group takes one tile after another: 128 query rows of one KV head (its tokens' heads of the group side by side, 16
// NQB rows a wave) over its part of the keys that they see.  Tiles of 32 keys and values go through registers, where
// codes become 16-bit values times their scale, once for all waves, into double-buffered swizzled LDS rows, one
// barrier a tile; the next tile's reads are under way while a tile is computed.  As in the forward of packed attention,
// S^T = K Q^T with Q^T in registers leaves 8 of a tile's 32 scores of a query row in a lane, which are, rounded, the
// operand of O^T += V^T P^T, and V^T comes from transposed LDS reads; the reference point of a row moves only
// when a score passes it by 8 (log2 units).  Only tiles at a wave's diagonal are masked.
//
// Bound by the conversion, LDS reads and barrier of every 32 keys beside the products, which keep the matrix cores 30 % busy:
// four sequences' chunks of 512 tokens after 4757 to 14925 keys, 32/8 heads of 128, take 427 us in 8 bits, 770 TFLOP/s, and
// 397 in 16, 830.  Page ids a tile ahead and reads without a branch: 370 us over three batches, 375 without.  Tiles are dealt
// as if they saw all keys of their sequence, so whole prompts are slower: one of 8192 tokens 490 TFLOP/s.
#include "attention_impl.h"
#include "paged_attention.h"

namespace ts {
namespace paged {

using attn::kRowOffsets;
using attn::ld16;
using attn::ro_of;
using attn::row_swizzle;
using attn::st16;
using attn::swizzled_offsets;
using attn::to_of;
using attn::tr_read;

constexpr int kTileRows = 128, kKeys = 32;

template <int ROW> constexpr int kBlocks = ROW <= 192 ? 2 : 1;  // 16-row query blocks a wave
template <int ROW> constexpr int kChunkWaves = kTileRows / 16 / kBlocks<ROW>;

template <typename T, bool WIDE, int ROW>
__global__ __launch_bounds__(64 * kChunkWaves<ROW>, (chunk_occupancy(ROW))) void chunk_kernel(AttnArgs) {
  constexpr int NQB = kBlocks<ROW>, kWaves = kChunkWaves<ROW>, kThreads = 64 * kWaves;
  constexpr int NC = ROW / 32, NB = ROW / 16;
  constexpr int kSize = WIDE ? 2 : 1;
  constexpr int kChunks = kKeys * ROW / 8 / kThreads;  // eight elements each, of a thread and tile
  __shared__ __attribute__((aligned(16))) bf16 s_k[2][kKeys * ROW];
  __shared__ __attribute__((aligned(16))) bf16 s_v[2][kKeys * ROW];
  const int lane_id = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  __shared__ Cursor<1>::Kept s_cur[2];
  Cursor<1> cur{};
  AttnArgs a = arguments();
  int turn_of = 0;
  if (wave == 0) {
    int past;
    const bool some = cur.begin(a, kTileRows, (int)blockIdx.x, lane_id, past);
    cur.put(s_cur[0], some, 0);
  }
  __syncthreads();
  if (!cur.take(s_cur[0])) return;
  for (;;) {
    a = arguments();
    int lane = lane_id;
    asm volatile("" : "+v"(lane));  // what follows from it is worked out again a tile, not held over the loop
    const int g = lane >> 4, r = lane & 15;
    const int first_row = cur.tile * kTileRows, rows = cur.seq.n * a.group, len = cur.seq.len, base = len - cur.seq.n;
    int begin, end;
    cur.piece(a, begin, end);
    if (a.plan && threadIdx.x == 0 && cur.head == 0 && cur.tile == 0 && cur.from == 0)
      a.plan[cur.s] = Plan{cur.end - cur.left, cur.blocks, cur.per, 1};

    const int wave_row = first_row + 16 * NQB * wave;
    bf16x8 q[NQB][NC];
    int limit[NQB];
#pragma unroll
    for (int t = 0; t < NQB; ++t) {
      const int row = wave_row + 16 * t + r;
      const int token = row / a.group, head = cur.head * a.group + row % a.group;
      const bool there = row < rows;
      limit[t] = there ? base + token : -1;
      const char* p = a.query + ((int64_t)(cur.seq.row0 + token) * a.token_stride + (int64_t)head * a.head_stride) * 2;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        u32x4 v = u32x4{0, 0, 0, 0};
        if (there && 32 * c + 8 * g < a.head_dim) v = *(const u32x4*)(p + 2 * (32 * c + 8 * g));
        q[t][c] = as_bf16x8(v);
      }
    }
    // the greatest of the limits of the wave's rows, and of all
    const int high = wave_row < rows ? base + min((wave_row + 16 * NQB - 1) / a.group, cur.seq.n - 1) : -1;
    const int stop = min(end, base + min((first_row + kTileRows - 1) / a.group, cur.seq.n - 1) + 1);

    f32x4 acc[NB][NQB];
    float m[NQB], l[NQB];
#pragma unroll
    for (int t = 0; t < NQB; ++t) {
      m[t] = neg_inf();
      l[t] = 0.f;
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    int ro[kRowOffsets<ROW>], to[2 * kRowOffsets<ROW>];
    swizzled_offsets<ROW>(lane, ro, to);

    const int32_t* table = a.batch.table + (int64_t)cur.s * a.batch.ld_table;
    const int page_mask = (1 << a.page_shift) - 1;
    // What the table says of a 16-token tile, and the page that it is: its own key's row of the table, or its last.
    auto read_near = [&](int pos) -> int { return uniform_table(table)[max(0, min(pos >> a.page_shift, a.batch.width - 1))]; };
    auto page_near = [&](int pos, int id) -> int {
      return pos < end && (pos >> a.page_shift) < a.batch.width && id >= 0 && id < a.pages ? id : -1;
    };
    using Raw = std::conditional_t<WIDE, u32x4, u32x2>;
    Raw rk[kChunks], rv[kChunks];
    float ks[kChunks], vs[kChunks];
    int page[2], ahead[2] = {read_near(begin), read_near(begin + 16)};  // of the tile loaded, and of the next
    // chunk i = 64 (wave + kWaves u) + lane of a tile: eight elements of row i / (ROW / 8); a wave's 64 lie in one half
    auto load = [&](int pos) {
      page[0] = page_near(pos, ahead[0]);
      page[1] = page_near(pos + 16, ahead[1]);
#pragma unroll
      for (int u = 0; u < kChunks; ++u) {
        const int i = 64 * (wave + kWaves * u) + lane, row = i / (ROW / 8), c = i % (ROW / 8);
        const bool second = 64 * (wave + kWaves * u) / (ROW / 8) >= 16;
        const int id = second ? max(page[1], 0) : max(page[0], 0);
        const int64_t line = ((int64_t)cur.head << a.page_shift) + ((pos + (second ? 16 : 0)) & page_mask);
        // rows behind the sequence, and of a page that is none, are past the descriptors' ends, and read as zeros
        const int there = (second ? page[1] : page[0]) < 0 ? 0 : min(16, len - (pos + (second ? 16 : 0)));
        const uint32_t bytes = there * ROW * kSize, at = ((row & 15) * ROW + 8 * c) * kSize;
        const rsrc_t k = make_rsrc(a.key + id * a.key_page_stride + line * (ROW * kSize), bytes);
        const rsrc_t v = make_rsrc(a.value + id * a.value_page_stride + line * (ROW * kSize), bytes);
        if constexpr (WIDE) {
          rk[u] = __builtin_amdgcn_raw_buffer_load_b128(k, at, 0, 0);
          rv[u] = __builtin_amdgcn_raw_buffer_load_b128(v, at, 0, 0);
        } else {
          rk[u] = __builtin_amdgcn_raw_buffer_load_b64(k, at, 0, 0);
          rv[u] = __builtin_amdgcn_raw_buffer_load_b64(v, at, 0, 0);
        }
        if constexpr (!WIDE) {
          const int64_t scale = (((int64_t)id * a.kv_heads << a.page_shift) + line) >> 4;
          ks[u] = uniform_table(a.key_scale)[scale];
          vs[u] = uniform_table(a.value_scale)[scale];
        }
      }
      ahead[0] = read_near(pos + kKeys);
      ahead[1] = read_near(pos + kKeys + 16);
    };
    auto store = [&](bf16* k, bf16* v) {
#pragma unroll
      for (int u = 0; u < kChunks; ++u) {
        const int i = 64 * (wave + kWaves * u) + lane, row = i / (ROW / 8), c = i % (ROW / 8);
        const int at = row * ROW + ((c ^ row_swizzle<ROW>(row & 15)) << 3);
        if constexpr (WIDE) {
          st16(k + at, rk[u]);
          st16(v + at, rv[u]);
        } else {
          st16(k + at, u32x4{widen2<T, false>(rk[u][0], ks[u]), widen2<T, true>(rk[u][0], ks[u]),
                             widen2<T, false>(rk[u][1], ks[u]), widen2<T, true>(rk[u][1], ks[u])});
          st16(v + at, u32x4{widen2<T, false>(rv[u][0], vs[u]), widen2<T, true>(rv[u][0], vs[u]),
                             widen2<T, false>(rv[u][1], vs[u]), widen2<T, true>(rv[u][1], vs[u])});
        }
      }
    };

    auto compute = [&](auto masked_, int pos, const bf16* tk, const bf16* tv, int page0, int page1) __attribute__((always_inline)) {
      constexpr bool masked = decltype(masked_)::value;
      f32x4 sc[2][NQB];
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int t = 0; t < NQB; ++t) sc[h][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const bf16x8 k = as_bf16x8(ld16(tk + ro_of<ROW>(ro, c) + 16 * h * ROW));
#pragma unroll
          for (int t = 0; t < NQB; ++t) sc[h][t] = mma16<T>(k, q[t][c], sc[h][t]);
        }
      }
      // key reads three steps ahead of their products
      __builtin_amdgcn_sched_group_barrier(0x100, 3, 1);
#pragma unroll
      for (int st = 0; st < 2 * NC; ++st) {
        __builtin_amdgcn_sched_group_barrier(0x008, NQB, 1);
        if (st + 3 < 2 * NC) __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
      }
      __builtin_amdgcn_s_setprio(0);
      const float c = masked ? 1.f : a.scale;
      if constexpr (masked) {  // to log2 units before -inf, which a scale of 0 or less would not leave as it is
#pragma unroll
        for (int t = 0; t < NQB; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) sc[h][t] *= a.scale;
      }
      if (page0 < 0 || page1 < 0) {  // keys of a page that is none
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if ((h ? page1 : page0) < 0 && pos + 16 * h < end)
#pragma unroll
            for (int t = 0; t < NQB; ++t) sc[h][t] = f32x4{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
      }
      if constexpr (masked) {
#pragma unroll
        for (int t = 0; t < NQB; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (pos + 16 * h + 4 * g + i > limit[t]) sc[h][t][i] = neg_inf();
      }
      bf16x8 p[NQB];
#pragma unroll
      for (int t = 0; t < NQB; ++t) {
        float e[8], sum;
        auto exponentials = [&]() __attribute__((always_inline)) {
          const float ref = m[t] == neg_inf() ? 0.f : m[t];
          sum = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            e[j] = fast_exp2(fmaf(sc[j >> 2][t][j & 3], c, -ref));
            sum += e[j];
          }
        };
        exponentials();
        if (__ballot((m[t] == neg_inf()) | (sum > kSlackSum<T>))) {
          float most = neg_inf();
#pragma unroll
          for (int j = 0; j < 8; ++j) most = fmaxf(most, sc[j >> 2][t][j & 3] * c);
          most = rows_max4(most);
          const bool move = most > m[t] + (kSlack + kLift<T>) || (m[t] == neg_inf() && most > m[t]);
          const float to = move ? most - kLift<T> : m[t], alpha = move ? fast_exp2(m[t] - to) : 1.f;
          m[t] = to;
          l[t] *= alpha;
#pragma unroll
          for (int b = 0; b < NB; ++b) acc[b][t] *= alpha;
          exponentials();
        }
        l[t] += sum;
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pack2<T>(e[2 * j], e[2 * j + 1]);
        p[t] = as_bf16x8(w);
      }
      __builtin_amdgcn_s_setprio(1);
      if constexpr (!masked) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const u32x2 a0 = tr_read(tv + to_of<ROW>(to, b)), a1 = tr_read(tv + to_of<ROW>(to, b) + 16 * ROW);
          const bf16x8 v = as_bf16x8(u32x4{a0[0], a0[1], a1[0], a1[1]});
#pragma unroll
          for (int t = 0; t < NQB; ++t) acc[b][t] = mma16<T>(v, p[t], acc[b][t]);
        }
        // value reads four blocks ahead
        __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          __builtin_amdgcn_sched_group_barrier(0x008, NQB, 0);
          if (b + 4 < NB) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      } else {
        // A weight of 0 does not take a NaN out: values that are not finite are left out of the product, and a second one, of
        // where they are with who sees them, ruins the elements of the rows that do.
        u32x4 seen[NQB];
#pragma unroll
        for (int t = 0; t < NQB; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int at = pos + 16 * (j >> 1) + 4 * g + 2 * (j & 1);
            seen[t][j] = (at <= limit[t] ? kOneOf<T> : 0u) | (at + 1 <= limit[t] ? kOneOf<T> << 16 : 0u);
          }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const u32x2 a0 = tr_read(tv + to_of<ROW>(to, b)), a1 = tr_read(tv + to_of<ROW>(to, b) + 16 * ROW);
          const u32x4 f = u32x4{a0[0], a0[1], a1[0], a1[1]};
          u32x4 fine, flag;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t x, y;
            split_finite<T>(f[j], x, y);
            fine[j] = x;
            flag[j] = y;
          }
#pragma unroll
          for (int t = 0; t < NQB; ++t) {
            acc[b][t] = mma16<T>(as_bf16x8(fine), p[t], acc[b][t]);
            const f32x4 n = mma16<T>(as_bf16x8(flag), as_bf16x8(seen[t]), f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (n[i] > 0.f) acc[b][t][i] = __builtin_nanf("");
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    };

    // Tiles that every row sees whole, each asked for while the one before is computed.
    const int plain = min(stop, base + first_row / a.group + 1) - (kKeys - 1);  // such tiles begin before it
    int pos = begin;
    if (pos < plain) {
      load(pos);
      store(s_k[0], s_v[0]);
    }
    auto turn = [&](auto stage_) __attribute__((always_inline)) {
      constexpr int stage = decltype(stage_)::value;
      const int page0 = page[0], page1 = page[1], next = pos + kKeys;
      if (next < plain) load(next);
      __syncthreads();  // the tile is in, and the other stage has been read
      compute(std::false_type{}, pos, s_k[stage], s_v[stage], page0, page1);
      if (next < plain) store(s_k[stage ^ 1], s_v[stage ^ 1]);
      pos = next;
    };
    while (pos < plain) {
      turn(std::integral_constant<int, 0>{});
      if (pos >= plain) break;
      turn(std::integral_constant<int, 1>{});
    }
    // The few at the diagonal, one by one: the registers are worth more.
    for (; pos < stop; pos += kKeys) {
      load(pos);
      __syncthreads();
      store(s_k[0], s_v[0]);
      __syncthreads();
      if (pos <= high) compute(std::true_type{}, pos, s_k[0], s_v[0], page[0], page[1]);
    }

    a = arguments();
    cur.take(s_cur[turn_of]);
    const bool all = cur.whole();
    const int slot = cur.slot(a.kv_heads);
#pragma unroll
    for (int t = 0; t < NQB; ++t) {
      const float sum = rows_sum4(l[t]);
      const int row = wave_row + 16 * t + r;
      if (row >= rows) continue;
      if (!all) {
        const int64_t at = (int64_t)slot * kTileRows + row - first_row;
        float* o = a.part[1] + at * ROW + 4 * g;
#pragma unroll
        for (int b = 0; b < NB; ++b) *(f32x4*)(o + 16 * b) = acc[b][t];
        if (g == 0) {
          a.stats[1][2 * at] = m[t];
          a.stats[1][2 * at + 1] = sum;
        }
        continue;
      }
      const float inv = sum > 0.f ? 1.f / sum : 0.f;
      const int token = row / a.group, head = cur.head * a.group + row % a.group;
      char* o = a.out + (((int64_t)(cur.seq.row0 + token) * a.heads + head) * a.head_dim + 4 * g) * 2;
#pragma unroll
      for (int b = 0; b < NB; ++b)
        if (16 * b + 4 * g < a.head_dim) {
          const f32x4 v = acc[b][t] * inv;
          *(u32x2*)(o + 32 * b) = u32x2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
        }
    }
    turn_of ^= 1;
    if (wave == 0) {
      const bool more = cur.next(a, kTileRows, lane_id);
      cur.put(s_cur[turn_of], more, 0);
    }
    __syncthreads();  // the next tile is known, and the last keys have been read
    if (!cur.take(s_cur[turn_of])) return;
  }
}

template <typename T, bool WIDE, int ROW>
void launch_chunk_rows(const AttnArgs& a, const Sizes& z, hipStream_t s) {
  ts::TimedLaunch timed_("paged.chunk_kernel", s);
  hipLaunchKernelGGL((chunk_kernel<T, WIDE, ROW>), dim3((unsigned)z.groups[1]), dim3(64 * kChunkWaves<ROW>), 0, s, a);
}

template <typename T, bool WIDE>
void launch_chunk_t(const AttnArgs& a, const Sizes& z, int row, hipStream_t s) {
  switch (row) {
    case 64: launch_chunk_rows<T, WIDE, 64>(a, z, s); break;
    case 128: launch_chunk_rows<T, WIDE, 128>(a, z, s); break;
    case 192: launch_chunk_rows<T, WIDE, 192>(a, z, s); break;
    default: launch_chunk_rows<T, WIDE, 256>(a, z, s);
  }
}

void launch_chunks(const AttnArgs& a, const Sizes& z, int dtype, bool wide, int row, hipStream_t s) {
  if (dtype == kF16) wide ? launch_chunk_t<f16, true>(a, z, row, s) : launch_chunk_t<f16, false>(a, z, row, s);
  else wide ? launch_chunk_t<bf16, true>(a, z, row, s) : launch_chunk_t<bf16, false>(a, z, row, s);
}

}  // namespace paged
}  // namespace ts
