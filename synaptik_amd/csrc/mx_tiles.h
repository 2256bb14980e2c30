// What the tile products of the microscaled operators (mx.h) share.
#pragma once
#include <type_traits>

#include "mx.h"

namespace shk {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

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

}  // namespace
}  // namespace shk
