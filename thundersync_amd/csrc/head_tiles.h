// Tiles of the head's logits for the kernels that form them on the MFMA core: token rows per
// tile by the launch, and the staging of a tile's 16-bit results.
#pragma once

#include "common.h"
#include "gemm_core.h"

namespace ts {
namespace head {

using namespace ts::gemm;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
__device__ __forceinline__ float neg_inf() { return -__builtin_huge_valf(); }

inline bool ok16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Token rows per tile of a launch: the rows spread evenly over as few tiles as
// 256-token tiles take.  Rows past the end of a tile are MFMA work on zeros --
// cheap on a chip whose clock follows its power, so a narrower tile pays only
// where it is much narrower: 64 or 128 tokens (4096 x 151936: 25 rows forward 279
// -> 264, dlogits 307 -> 269, grad_hidden 201 -> 188 us, 128 rows 307 -> 288, 337 ->
// 295, 235 -> 223), and for grad_hidden, whose launch of few rows is one round that
// ends with its widest tiles, 192 for up to 160 (320 rows 463 -> 409; at 192 rows a
// tile 464 -> 478, and forward and dlogits gain nothing).
inline int token_tile(int64_t rows, bool up_to_192) {
  const int64_t tiles = (rows + TN - 1) / TN, each = (rows + tiles - 1) / tiles;
  return each <= 64 ? 64 : each <= 128 ? 128 : up_to_192 && each <= 160 ? 192 : 256;
}

// The 320-token tile (Wide) reads a weight tile once for rows that need two or
// more 256-token ones, in kWideCost / 256 of a 256-token tile's time (by its MFMAs
// 320 / 256; set to what the launches below take).  `stride`: the token
// operand's, for the 32-bit offsets of its rows within a tile.
constexpr int kWideTokens = Wide::BN;
constexpr int kWideCost = 352;
inline bool wide_fits(int64_t rows, int64_t stride) { return rows > TN && (kWideTokens - 1) * stride < (1ll << 30); }

// Forward and dlogits: 320 where the launch then takes less time in rounds of one
// work-group per CU: 1 tile for 2 at 257 .. 320 rows of 594 vocabulary tiles (3
// rounds for 5: 281 rows forward 488 -> 434 us, dlogits 500 -> 450), 2 for 3 at 600 (5
// for 7: 755 -> 698, 778 -> 723), but not at 384 (5 for 5: 520 -> 651) or 2048 (17 for
// 19: 2157 -> 2286).
inline int logits_tile(int64_t rows, int64_t vtiles, int64_t stride) {
  auto rounds = [&](int64_t w) { return ((rows + w - 1) / w * vtiles + 255) / 256; };
  if (wide_fits(rows, stride) && rounds(kWideTokens) * kWideCost < rounds(TN) * TN) return kWideTokens;
  return token_tile(rows, false);
}

constexpr int OPITCH = TM + 8;  // staging pitch (bf16) of [64 tokens][TM vocab] quarter tiles
static_assert(64 * OPITCH <= kRingElems, "a quarter of the dlogits tile fits one ring stage");

}  // namespace head
}  // namespace ts

// launch kernel<element, tile shape> by a DType code and token_tile's width
#define TS_LAUNCH_TOKENS(dtype, width, kernel, ...)                               \
  do {                                                                            \
    if ((width) == 64) TS_LAUNCH_E_T(dtype, kernel, Narrow<1>, __VA_ARGS__);      \
    else if ((width) == 128) TS_LAUNCH_E_T(dtype, kernel, Narrow<2>, __VA_ARGS__); \
    else if ((width) == ::ts::head::kWideTokens) TS_LAUNCH_E_T(dtype, kernel, Wide, __VA_ARGS__); \
    else TS_LAUNCH_E_T(dtype, kernel, Full, __VA_ARGS__);                         \
  } while (0)
