// Launches that stay within what a grid holds: its first dimension has fewer than 2^32 threads, and
// a launch beyond that is refused. Host code without HIP, so that it can be checked by itself.
#pragma once
#include <cstdint>

namespace shk {

constexpr int64_t LAUNCH_THREADS = (1ll << 32) - 1;  // of a grid's first dimension

// Packing of a microscaled product's operands (mx_gemm.hip): a unit is 32 k of 64 rows of A or of
// 256 columns of B, `blocks` of them for each 32 k. A product of little width and great depth has
// more units than a launch has workgroups (65 x 129 by 179 million: 2^32 threads), so the launch has
// at most PACK_GROUPS workgroups of PACK_THREADS, each taking every PACK_GROUPS-th unit.
constexpr int64_t PACK_GROUPS = 1 << 16, PACK_THREADS = 256;
inline int64_t mx_pack_blocks(int64_t M, int64_t N) { return (M + 63) / 64 + (N + 255) / 256; }
inline int64_t mx_pack_units(int64_t M, int64_t N, int64_t K) {
  return (K + 31) / 32 * mx_pack_blocks(M, N);
}
inline int64_t mx_pack_groups(int64_t units) { return units < PACK_GROUPS ? units : PACK_GROUPS; }

// Column sums have a workgroup of COLSUM_THREADS for every COLSUM_WIDTH columns at the least, which 2^30
// columns would take beyond a launch: wider ones go COLSUM_COLS at a time.
constexpr int64_t COLSUM_WIDTH = 64, COLSUM_THREADS = 256, COLSUM_COLS = 1ll << 29;
inline int64_t colsum_groups(int64_t cols) { return (cols + COLSUM_WIDTH - 1) / COLSUM_WIDTH; }

}  // namespace shk
