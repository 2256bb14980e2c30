// What the tile products of the microscaled operators (mx.h) share.
#pragma once
#include <type_traits>

#include "mx.h"

namespace shk {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

// Two values as bfloat16, by the conversion that scales (exact, and NaN under the scale 255): those
// of the low or high half of a word of four 8-bit codes, or of byte PART of a word of eight e2m1
// codes.
template <int F, int PART>
__device__ __forceinline__ uint32_t mx_values2(uint32_t w, float scale) {
  if constexpr (F == MX_E2M1)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, PART));
  else if constexpr (F == MX_E4M3)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, PART != 0));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, scale, PART != 0));
}
// The scale operand of a byte: the conversion reads its exponent, and NaN in an infinity's.
__device__ __forceinline__ float mx_scale_operand(uint32_t s) { return __uint_as_float(s << 23); }

// Workgroup -> tile: tiles in bands of four rows of tiles, and each of the eight XCDs (workgroups
// go to them in turn) a contiguous run of that order, so that an XCD's second-level cache serves
// few rows and columns of tiles.
__device__ __forceinline__ void mx_tile_of(int id, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int tiles = tiles_m * tiles_n, per = tiles / 8, extra = tiles % 8, xcd = id % 8;
  const int t = xcd * per + min(xcd, extra) + id / 8;
  const int band = t / (4 * tiles_n), first = 4 * band, rows = min(4, tiles_m - first);
  const int in_band = t - band * 4 * tiles_n;
  tm = first + in_band % rows;
  tn = in_band / rows;
}

// A product's tiles: how many of its rows of tiles of 256, the first ones, are taken (none, as many
// as fill whole rounds of the 256 CUs, or all); the rows behind them go to tiles of 128. The fewest
// rounds win, a tile of 256 counting `ratio` of 128.
inline int64_t mx_tiles(int64_t M, int64_t N, int64_t edge) {
  return M <= 0 ? 0 : ((M + edge - 1) / edge) * ((N + edge - 1) / edge);
}
inline int mx_large_rows(int64_t M, int64_t N, double ratio) {
  const int64_t all = (M + 255) / 256, row = mx_tiles(1, N, 256), filled = all * row / 256 * 256 / row;
  int64_t best = 0;
  double least = 1e300;
  for (int64_t m : {(int64_t)0, filled, all}) {
    const int64_t large = (m * row + 255) / 256, small = (mx_tiles(M - 256 * m, N, 128) + 255) / 256;
    const double t = ratio * (double)large + (double)small;
    if (t < least) least = t, best = m;
  }
  return (int)best;
}

}  // namespace
}  // namespace shk
