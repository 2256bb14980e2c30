// Sums over a wave's lanes by DPP: a step is two moves and an addition within the vector unit, where a
// shuffle goes through LDS and back twice for a binary64 value. The order is fixed.
#pragma once
#include "common.h"

namespace shk {

// v of the lane that CTRL names, 0 where it names none or the row of 16 lanes is not in MASK.
template <int CTRL, int MASK = 0xf>
__device__ __forceinline__ double dpp_get(double v) {
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, MASK, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, MASK, 0xf, true);
  return __hiloint2double(hi, lo);
}

// A value that is the same in every lane, in scalar registers.
__device__ __forceinline__ double wave_uniform(double v) {
  return __hiloint2double(__builtin_amdgcn_readfirstlane(__double2hiint(v)),
                          __builtin_amdgcn_readfirstlane(__double2loint(v)));
}

// The sum over all 64 lanes, the same in every lane. All lanes are active.
__device__ __forceinline__ double wave_total(double v) {
  v += dpp_get<0x111>(v);        // the lanes 1, 2, 4, 8 before within a row of 16
  v += dpp_get<0x112>(v);
  v += dpp_get<0x114>(v);
  v += dpp_get<0x118>(v);
  v += dpp_get<0x142, 0xa>(v);   // lane 15 of the row before, into rows 1 and 3
  v += dpp_get<0x143, 0xc>(v);   // lane 31, into rows 2 and 3
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), 63),
                          __builtin_amdgcn_readlane(__double2loint(v), 63));
}

// The sum over each group of L lanes (a power of two), the same in every lane of it. A group is
// active or not as a whole.
template <int L>
__device__ __forceinline__ double team_total(double v) {
  if constexpr (L == 64) return wave_total(v);
  if constexpr (L >= 2) v += dpp_get<0xb1>(v);    // the neighbour
  if constexpr (L >= 4) v += dpp_get<0x4e>(v);    // the other pair of four
  if constexpr (L >= 8) v += dpp_get<0x141>(v);   // the other four of eight, mirrored
  if constexpr (L >= 16) v += dpp_get<0x140>(v);  // the other eight of sixteen, mirrored
  if constexpr (L >= 32) v += __shfl_xor(v, 16, 64);
  return v;
}

}  // namespace shk
