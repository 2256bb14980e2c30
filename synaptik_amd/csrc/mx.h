// Microscaled tensors: codes of 8 or 4 bits under one power of two for every 32 values of a row.
//
// A [R, C] tensor holds G = ceil(C / 128) groups of 128 values a row: 128 code bytes a group for
// the 8-bit formats (one a value), 64 for e2m1 (two values a byte, the even column in the low
// half), and four scale bytes a group, one for each block of 32 columns. Codes behind column C are
// zero. A scale byte s is the exponent of a power of two, 2^(s - 127) (255: NaN, the block's values
// are NaN); a code c of that block stands for value(c) * 2^(s - 127). Rows and groups follow each
// other without gaps, so group g of row r has the ordinal r G + g in both arrays. Whole groups keep
// every block and every row aligned to 64 bytes whatever C is, and give a matrix instruction that
// contracts 128 values its four scales in one 4-byte word.
//   e4m3 (0): 1 sign, 4 exponent, 3 mantissa bits, largest 448, no infinities, NaN 0x7f / 0xff
//   e5m2 (1): 1, 5, 2, largest 57344, infinities 0x7c / 0xfc, NaN above
//   e2m1 (2): 1, 2, 1, values 0, 0.5, 1, 1.5, 2, 3, 4, 6; neither infinities nor NaN
// Restoring and gradients take every scale as it is. The products take values that are zero or from
// 2^-126 to below 2^128 in magnitude exactly, which is all that encoding gives, and all that scales of
// 17 to 239 give in any format. Through bfloat16 a smaller one counts with an error below 2^-126 (the
// matrix cores read subnormal values as zeros) and a larger one as an infinity; the scaled 4-bit
// instructions take both as they are.
#pragma once
#include "common.h"

namespace shk {

constexpr int MX_GROUP = 128, MX_BLOCK = 32;

inline int64_t mx_groups(int64_t C) { return (C + MX_GROUP - 1) / MX_GROUP; }
constexpr int mx_group_bytes(int format) { return format == MX_E2M1 ? 64 : 128; }

// Encoding picks the smallest power of two under which the block's largest finite magnitude lies
// within the format, so that nothing saturates (but for values that would round to 2^128: they take
// the largest code below, MxFormat::LARGEST, so that a finite value stays finite), and never one
// below 2^MX_LEAST_EXPONENT: then every nonzero value a code stands for (at least 2^-16 times its
// scale) is a normal binary32 and bfloat16 number.
constexpr int MX_LEAST_EXPONENT = -110;

template <int F>
struct MxFormat;
template <>
struct MxFormat<MX_E4M3> {
  static constexpr int TOP = 8;                  // binade of the largest value
  static constexpr uint32_t MANTISSA = 0x600000;  // and its mantissa: 1.75 * 2^8
  static constexpr uint32_t LARGEST = 0x7f700000;  // 1.875 * 2^127: the format's last below 2^128
};
template <>
struct MxFormat<MX_E5M2> {
  static constexpr int TOP = 15;
  static constexpr uint32_t MANTISSA = 0x600000;
  static constexpr uint32_t LARGEST = 0x7f600000;
};
template <>
struct MxFormat<MX_E2M1> {
  static constexpr int TOP = 2;
  static constexpr uint32_t MANTISSA = 0x400000;  // 1.5 * 2^2
  static constexpr uint32_t LARGEST = 0x7f400000;
};

// The scale byte of a block whose largest finite magnitude has these bits.
template <int F>
__device__ __forceinline__ uint32_t mx_scale_of(uint32_t largest) {
  // the binade, one more when the mantissa is above that of the format's largest value
  const int e = (int)((largest + (0x7fffffu - MxFormat<F>::MANTISSA)) >> 23) - MxFormat<F>::TOP;
  return (uint32_t)max(e, MX_LEAST_EXPONENT + 127);
}

// 2^(s - 127) and its reciprocal (of scales that encoding gives: both are normal numbers).
__device__ __forceinline__ float mx_factor(uint32_t s) {
  return __uint_as_float(s == 0 ? 0x00400000u : s == 255u ? 0x7fc00000u : s << 23);
}
__device__ __forceinline__ float mx_reciprocal(uint32_t s) {
  return __uint_as_float((254u - s) << 23);
}

// The maximum over the eight lanes that hold a block's 32 values: two quad permutations, then the
// mirror image within eight lanes.
__device__ __forceinline__ uint32_t mx_block_largest(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, false));
  return v;
}

// Four values, already divided by their scale, as codes: a word of four bytes, or 16 bits of four
// halves for e2m1. Rounding is to nearest, ties to even, and nothing overflows (mx_scale_of). x
// holds the values before scaling: with KEEP a nonzero one never becomes a zero code; an infinity
// or a NaN of an 8-bit format becomes the format's (e4m3 has NaN alone).
template <int F, bool KEEP>
__device__ __forceinline__ uint32_t mx_codes4(const float (&x)[4], float reciprocal) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float limit = __uint_as_float(MxFormat<F>::LARGEST);
    y[i] = fminf(fmaxf(x[i], -limit), limit) * reciprocal;
  }
  if constexpr (F == MX_E2M1) {
    uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[0], y[1], 1.0f, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[2], y[3], 1.0f, 1);
    return c & 0xffffu;
  } else {
    int c;
    if constexpr (F == MX_E4M3) {
      c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      c = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true);
    } else {
      c = __builtin_amdgcn_cvt_pk_bf8_f32(y[0], y[1], 0, false);
      c = __builtin_amdgcn_cvt_pk_bf8_f32(y[2], y[3], c, true);
    }
    uint32_t w = (uint32_t)c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = 0xffu << (8 * i), b = __float_as_uint(x[i]);
      if (KEEP && (w & (0x7fu << (8 * i))) == 0 && (b << 1) != 0) w |= 1u << (8 * i);
      if ((b & 0x7f800000u) == 0x7f800000u) {
        const uint32_t v = (F == MX_E5M2 && (b & 0x7fffffu) == 0 ? 0x7cu : 0x7fu) | ((b >> 24) & 0x80u);
        w = (w & ~m) | (v << (8 * i));
      }
    }
    return w;
  }
}

// The values of four codes (a word, or the low 16 bits for e2m1) before their scale.
template <int F>
__device__ __forceinline__ void mx_values4(uint32_t w, float (&v)[4]) {
  typedef float floatx2 __attribute__((ext_vector_type(2)));
  floatx2 a, b;
  if constexpr (F == MX_E2M1) {
    a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
    b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
  } else if constexpr (F == MX_E4M3) {
    a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  } else {
    a = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, false);
    b = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, true);
  }
  v[0] = a[0];
  v[1] = a[1];
  v[2] = b[0];
  v[3] = b[1];
}

// The codes of the four columns 4 q .. 4 q + 3 of a row, as mx_values4 takes them. 32-bit code
// words of 8-bit formats, 16-bit ones of e2m1: aligned, since groups are.
template <int F>
__device__ __forceinline__ uint32_t mx_load4(const uint8_t* row, int64_t q) {
  if constexpr (F == MX_E2M1) return reinterpret_cast<const uint16_t*>(row)[q];
  else return reinterpret_cast<const uint32_t*>(row)[q];
}

// Calls f(integral_constant<int, format>).
template <typename Fn>
inline void mx_with_format(int format, Fn f) {
  switch (format) {
    case MX_E4M3: f(std::integral_constant<int, MX_E4M3>()); break;
    case MX_E5M2: f(std::integral_constant<int, MX_E5M2>()); break;
    default: f(std::integral_constant<int, MX_E2M1>()); break;
  }
}

}  // namespace shk
