// Four consecutive floats of a row that may start at any float and end inside a group: the
// hardware's 16-byte accesses take such addresses, and a group's floats behind the row's end are
// neither read nor written.
#pragma once
#include "common.h"

namespace shk {

// p[0 .. 3], of which the first `rest` belong to the row (none when rest <= 0); the others read as 0.
template <bool STREAM = false, typename N>
__device__ __forceinline__ float4 ld4(const float* p, N rest) {
  if (rest >= 4) {
    const float4u* q = reinterpret_cast<const float4u*>(p);
    const float4u t = STREAM ? __builtin_nontemporal_load(q) : *q;
    return make_float4(t[0], t[1], t[2], t[3]);
  }
  return make_float4(rest > 0 ? p[0] : 0.0f, rest > 1 ? p[1] : 0.0f, rest > 2 ? p[2] : 0.0f, 0.0f);
}
template <bool STREAM = false, typename N>
__device__ __forceinline__ void st4(float* p, N rest, const float4& v) {
  if (rest >= 4) {
    float4u* q = reinterpret_cast<float4u*>(p);
    const float4u t = {v.x, v.y, v.z, v.w};
    if (STREAM) __builtin_nontemporal_store(t, q);
    else *q = t;
    return;
  }
  if (rest > 0) p[0] = v.x;
  if (rest > 1) p[1] = v.y;
  if (rest > 2) p[2] = v.z;
}

// The same from a row's start and a group's offset in it, in bytes: one base register for a wave whose
// lanes read one row.
template <bool STREAM = false>
__device__ __forceinline__ float4 ld4_at(const float* row, uint32_t bytes, int rest) {
  return ld4<STREAM>(reinterpret_cast<const float*>(reinterpret_cast<const char*>(row) + bytes), rest);
}
template <bool STREAM = false>
__device__ __forceinline__ void st4_at(float* row, uint32_t bytes, int rest, const float4& v) {
  st4<STREAM>(reinterpret_cast<float*>(reinterpret_cast<char*>(row) + bytes), rest, v);
}

}  // namespace shk
