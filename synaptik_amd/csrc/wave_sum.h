// Sums over a wave's lanes within the vector unit: by DPP within a row of 16 lanes, by row swaps
// between rows, where a shuffle goes through LDS and back twice for a binary64 value. Several sums are
// formed together: each of the first steps halves the values that a lane still adds up, so that four
// sums over 64 lanes take 7 additions instead of 24. The order is fixed.
#pragma once
#include <type_traits>

#include "common.h"

namespace shk {

// v of the lane that CTRL names for this one.
template <int CTRL>
__device__ __forceinline__ double dpp_get(double v) {
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xf, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xf, 0xf, true);
  return __hiloint2double(hi, lo);
}
constexpr int DPP_XOR1 = 0xb1, DPP_XOR2 = 0x4e;           // within four lanes
constexpr int DPP_ROR4 = 0x124, DPP_ROR8 = 0x128;         // around a row of 16
constexpr int DPP_MIRROR8 = 0x141, DPP_MIRROR16 = 0x140;  // eight and sixteen lanes reversed

// v plus that of the lane 16 (32) before or behind it. All lanes are active.
__device__ __forceinline__ double add_row(double v) {
  const auto lo = __builtin_amdgcn_permlane16_swap(__double2loint(v), __double2loint(v), false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(__double2hiint(v), __double2hiint(v), false, false);
  return __hiloint2double(hi[0], lo[0]) + __hiloint2double(hi[1], lo[1]);
}
__device__ __forceinline__ double add_half(double v) {
  const auto lo = __builtin_amdgcn_permlane32_swap(__double2loint(v), __double2loint(v), false, false);
  const auto hi = __builtin_amdgcn_permlane32_swap(__double2hiint(v), __double2hiint(v), false, false);
  return __hiloint2double(hi[0], lo[0]) + __hiloint2double(hi[1], lo[1]);
}

// The sum of v over the lanes whose numbers differ in the bits FROM .. TO - 1 (powers of two).
template <int FROM, int TO>
__device__ __forceinline__ double add_lanes(double v) {
  if constexpr (FROM <= 1 && TO > 1) v += dpp_get<DPP_XOR1>(v);
  if constexpr (FROM <= 2 && TO > 2) v += dpp_get<DPP_XOR2>(v);
  if constexpr (FROM <= 4 && TO > 4) {
    // (a rotation by four is the other quad where lanes eight apart are alike: afterwards, or here)
    if constexpr (TO > 8) v += dpp_get<DPP_ROR8>(v);
    v += dpp_get<DPP_ROR4>(v);
  } else if constexpr (FROM == 8 && TO > 8) {
    v += dpp_get<DPP_ROR8>(v);
  }
  if constexpr (FROM <= 16 && TO > 16) v = add_row(v);
  if constexpr (FROM <= 32 && TO > 32) v = add_half(v);
  return v;
}

// The value of lane k in every lane.
__device__ __forceinline__ double lane_value(double v, int k) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), k),
                          __builtin_amdgcn_readlane(__double2loint(v), k));
}

// Sums of K values (1, 2 or 4) over 64 lanes: lane l returns that of value l % K.
template <int K>
__device__ __forceinline__ double wave_sums(const double (&v)[K]) {
  const int lane = threadIdx.x & 63;
  if constexpr (K == 1) {
    return add_lanes<1, 64>(v[0]);
  } else if constexpr (K == 2) {
    const bool odd = lane & 1;
    const double keep = odd ? v[1] : v[0], give = odd ? v[0] : v[1];
    return add_lanes<2, 64>(keep + dpp_get<DPP_XOR1>(give));
  } else {
    static_assert(K == 4);
    const bool odd = lane & 1, high = lane & 2;
    double a = odd ? v[1] : v[0], b = odd ? v[3] : v[2];  // the values odd and odd + 2
    a += dpp_get<DPP_XOR1>(odd ? v[0] : v[1]);
    b += dpp_get<DPP_XOR1>(odd ? v[2] : v[3]);
    const double keep = high ? b : a, give = high ? a : b;
    return add_lanes<4, 64>(keep + dpp_get<DPP_XOR2>(give));
  }
}

// The largest value over 64 lanes, the same in every lane; NaN counts as absent. All lanes are active.
__device__ __forceinline__ float wave_largest(float v) {
  const auto other = [&](auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  v = fmaxf(v, other(std::integral_constant<int, DPP_XOR1>()));
  v = fmaxf(v, other(std::integral_constant<int, DPP_XOR2>()));
  v = fmaxf(v, other(std::integral_constant<int, DPP_MIRROR8>()));
  v = fmaxf(v, other(std::integral_constant<int, DPP_MIRROR16>()));
  const auto row = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
  v = fmaxf(__int_as_float(row[0]), __int_as_float(row[1]));
  const auto half = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
  return fmaxf(__int_as_float(half[0]), __int_as_float(half[1]));
}

// Sums of K values over a workgroup of NT threads, the same in every thread; `lds`: K NT / 64 doubles,
// free again after the next barrier but one.
template <int NT, int K>
__device__ __forceinline__ void group_sums(double (&v)[K], double* lds) {
  constexpr int NW = NT / 64;
  double s = wave_sums<K>(v);
  if constexpr (NW > 1) {
    const int lane = threadIdx.x & 63;
    if (lane < K) lds[(threadIdx.x >> 6) * K + lane] = s;
    __syncthreads();
    s = add_lanes<K, NW * K>(lds[lane & (NW * K - 1)]);
  }
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = lane_value(s, k);
}

// Sums of K values over each group of L lanes (a power of two), the same in every lane of it. A group
// is active or not as a whole.
template <int L, int K>
__device__ __forceinline__ void team_sums(double (&v)[K]) {
  if constexpr (L == 64) {
    const double s = wave_sums<K>(v);
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = lane_value(s, k);
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if constexpr (L >= 2) v[k] += dpp_get<DPP_XOR1>(v[k]);
      if constexpr (L >= 4) v[k] += dpp_get<DPP_XOR2>(v[k]);
      if constexpr (L >= 8) v[k] += dpp_get<DPP_MIRROR8>(v[k]);
      if constexpr (L >= 16) v[k] += dpp_get<DPP_MIRROR16>(v[k]);
      if constexpr (L >= 32) v[k] += __shfl_xor(v[k], 16, 64);
    }
  }
}

}  // namespace shk
