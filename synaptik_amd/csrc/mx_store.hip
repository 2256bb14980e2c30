// Microscaled tensors (mx.h): encoding, restoring, and the cotangent of an activation from its
// 8-bit checkpoint.
#include <algorithm>
#include <type_traits>

#include "mx.h"

namespace shk {
namespace {

// Columns 4 q .. 4 q + 3 of a row of C floats (`rest` = C - 4 q of them at most; none when rest <= 0).
__device__ __forceinline__ void load4(const float* p, int rest, float (&v)[4]) {
  if (rest >= 4) {
    const float4u t = *reinterpret_cast<const float4u*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = t[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < rest ? p[i] : 0.0f;
  }
}
__device__ __forceinline__ void store4(float* p, int rest, const float (&v)[4]) {
  if (rest >= 4) {
    *reinterpret_cast<float4u*>(p) = float4u{v[0], v[1], v[2], v[3]};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < rest) p[i] = v[i];
  }
}

// One group of 128 values for 32 lanes, four values a lane, U groups a lane and round: a block is
// eight lanes, whose largest magnitude goes round by DPP. Memory bounds it: [8192, 4096] to e2m1 takes
// 25 us, 152 MB at 6.1 TB/s, and the way back 23 us, 6.6 TB/s; [500, 1021]
// 2.9 us, little more than a launch.
template <int F, bool KEEP, int U>
__global__ void __launch_bounds__(256) mx_encode(const float* __restrict__ x, int64_t ldx,
                                                 uint8_t* __restrict__ codes,
                                                 uint8_t* __restrict__ scales, int C, uint32_t G,
                                                 uint32_t total) {
  const int q = threadIdx.x & 31;
  for (uint64_t base = (uint64_t)blockIdx.x * (8 * U) + (threadIdx.x >> 5); base < total;
       base += (uint64_t)gridDim.x * (8 * U)) {
    float v[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t t = (uint32_t)min(base + 8 * u, (uint64_t)total - 1);
      const uint32_t r = t / G, c = (t - r * G) * MX_GROUP + 4 * q;
      load4(x + (int64_t)r * ldx + c, C - (int)c, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (base + 8 * u >= total) break;
      const uint64_t t = base + 8 * u;
      uint32_t largest = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t b = __float_as_uint(v[u][i]) & 0x7fffffffu;
        // (an infinity or NaN of an e2m1 block takes the block; elsewhere it has a code)
        largest = max(largest, F != MX_E2M1 && b >= 0x7f800000u ? 0u : b);
      }
      largest = mx_block_largest(largest);
      const bool lost = F == MX_E2M1 && largest >= 0x7f800000u;
      const uint32_t s = mx_scale_of<F>(largest);
      uint32_t w = mx_codes4<F, KEEP>(v[u], mx_reciprocal(s));
      if (F == MX_E2M1) reinterpret_cast<uint16_t*>(codes)[t * 32 + q] = lost ? 0 : (uint16_t)w;
      else reinterpret_cast<uint32_t*>(codes)[t * 32 + q] = w;
      if ((q & 7) == 0) scales[t * 4 + (q >> 3)] = lost ? 255 : (uint8_t)s;
    }
  }
}

template <int F, int U>
__global__ void __launch_bounds__(256) mx_decode(const uint8_t* __restrict__ codes,
                                                 const uint8_t* __restrict__ scales,
                                                 float* __restrict__ y, int64_t ldy, int C, uint32_t G,
                                                 uint32_t total) {
  const int q = threadIdx.x & 31;
  for (uint64_t base = (uint64_t)blockIdx.x * (8 * U) + (threadIdx.x >> 5); base < total;
       base += (uint64_t)gridDim.x * (8 * U)) {
    uint32_t w[U], s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t t = min(base + 8 * u, (uint64_t)total - 1);
      w[u] = mx_load4<F>(codes, t * 32 + q);
      s[u] = scales[t * 4 + (q >> 3)];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (base + 8 * u >= total) break;
      const uint32_t t = (uint32_t)(base + 8 * u);
      const uint32_t r = t / G, c = (t - r * G) * MX_GROUP + 4 * q;
      const float f = mx_factor(s[u]);
      float v[4];
      mx_values4<F>(w[u], v);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] *= f;
      store4(y + (int64_t)r * ldy + c, C - (int)c, v);
    }
  }
}

// dZ = act_grad(dY, Y) from Y's codes, and the column sums of this workgroup's rows in binary64:
// PARTIAL as row blockIdx.y of [gridDim.y, C], WHOLE (one row of workgroups) rounded into the
// result. A workgroup takes 4 Q columns and `rows` rows, Q lanes a row: 256 columns and four rows at
// once where its sums are partial, 32 columns (one line of memory) and 128 rows at once where they
// are whole. dy and dz may be the same memory.
constexpr int AG_UNROLL = 4;
enum Sums { NO_SUMS, PARTIAL, WHOLE };
template <int F, int ACT, int SUMS>
__global__ void __launch_bounds__(SUMS == WHOLE ? 1024 : 256)
    mx_act_grad(const float* dy, int64_t ldy, const uint8_t* __restrict__ codes,
                const uint8_t* __restrict__ scales, float* dz, int64_t ldz, void* __restrict__ sums,
                int64_t R, int C, int64_t G, int64_t rows) {
  constexpr int Q = SUMS == WHOLE ? 8 : 64, AT_ONCE = SUMS == WHOLE ? 128 : 4;
  const int quad = threadIdx.x % Q, w = threadIdx.x / Q;
  const int64_t c = (int64_t)blockIdx.x * (4 * Q) + 4 * quad;
  const int rest = (int)min((int64_t)4, C - c);
  const int64_t last = min(R, ((int64_t)blockIdx.y + 1) * rows);
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  if (rest > 0) {
    for (int64_t r0 = (int64_t)blockIdx.y * rows + w; r0 < last; r0 += AT_ONCE * AG_UNROLL) {
      float g[AG_UNROLL][4];
      uint32_t code[AG_UNROLL], s[AG_UNROLL];
#pragma unroll
      for (int u = 0; u < AG_UNROLL; ++u) {
        const int64_t r = min(r0 + AT_ONCE * u, last - 1);
        load4(dy + r * ldy + c, rest, g[u]);
        code[u] = mx_load4<F>(codes, r * G * 32 + c / 4);
        s[u] = scales[r * G * 4 + c / 32];
      }
#pragma unroll
      for (int u = 0; u < AG_UNROLL; ++u) {
        const int64_t r = r0 + AT_ONCE * u;
        if (r >= last) break;
        const float f = mx_factor(s[u]);
        float y[4];
        mx_values4<F>(code[u], y);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          g[u][i] = act_grad(ACT, g[u][i], y[i] * f);
          if (SUMS != NO_SUMS) sum[i] += (double)g[u][i];
        }
        store4(dz + r * ldz + c, rest, g[u]);
      }
    }
  }
  if constexpr (SUMS != NO_SUMS) {
    // the rows of a wave, then the waves in order
    constexpr int WAVES = SUMS == WHOLE ? 16 : 4;
    __shared__ double wave_sums[WAVES][4 * Q];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int o = Q; o < 64; o *= 2) sum[i] += __shfl_xor(sum[i], o, 64);
    }
    if ((threadIdx.x & 63) < Q) {
#pragma unroll
      for (int i = 0; i < 4; ++i) wave_sums[threadIdx.x >> 6][4 * quad + i] = sum[i];
    }
    __syncthreads();
    const int64_t col = (int64_t)blockIdx.x * (4 * Q) + threadIdx.x;
    if (threadIdx.x < 4 * Q && col < C) {
      double v = wave_sums[0][threadIdx.x];
#pragma unroll
      for (int i = 1; i < WAVES; ++i) v += wave_sums[i][threadIdx.x];
      if (SUMS == WHOLE) static_cast<float*>(sums)[col] = (float)v;
      else static_cast<double*>(sums)[(int64_t)blockIdx.y * C + col] = v;
    }
  }
}

// Whether one workgroup takes all rows of its columns, whose sums then need no second launch (us, a
// run's 11 included: 500x4096 17.2 against 18.8, 1024x1000 18.5 against 19.5, 1024x4096 22.5 either
// way, but 2048x1000 28.0 against 22.4); a launch has fewer than 2^32 threads.
bool whole_sums(int64_t R, int64_t C) { return R <= 1024 && C <= 1 << 26; }

// Rows a workgroup takes otherwise: 16 (four a wave, all in flight at once) or as many as make 64
// slabs of rows, whose sums the second launch reads fastest (4096x1000 24.7 us, with 32 / 128 / 256
// slabs 27.2 / 25.8 / 30.7; 4096x4096 41.5, of which the first launch is 26 us for 151 MB, 5.8 TB/s, and
// 32 us, 4.7 TB/s, in a backward pass between other kernels), or 1024 workgroups where
// there are few columns and the slabs so many that their sums are folded in two launches (8192x200
// 20.5 against 26.0).
int64_t act_grad_rows(int64_t R, int64_t C) {
  const int64_t strips = (C + 255) / 256, slabs = R > 4096 && strips <= 2 ? 1024 / strips : 64;
  const int64_t rows = (R + slabs - 1) / slabs;
  return std::max<int64_t>(16, (rows + 15) / 16 * 16);
}

// Workgroups for `groups` groups of 128, eight a round and U rounds' loads in flight.
unsigned store_grid(int64_t groups, int u) {
  return (unsigned)std::min<int64_t>((groups + 8 * u - 1) / (8 * u), 1 << 20);
}
// Enough groups that every CU has work with four in flight a lane (e4m3, us a run with four and with
// one: encoding [256, 4096] 14.5 and 14.1, [1024, 4096] 16.4 and 16.2, [2048, 4096] 19.4 and 20.5,
// [8192, 4096] 37.6 and 39.2; restoring the last 37.3 and 37.5).
constexpr int64_t STORE_MANY = 4 * 8 * 1024;

}  // namespace

hipError_t launch_mx_encode(const float* x, int64_t ldx, uint8_t* codes, uint8_t* scales, int64_t R,
                            int64_t C, int format, int keep_nonzero, hipStream_t s) {
  const int64_t G = mx_groups(C), total = R * G;
  if (total <= 0) return hipSuccess;
  mx_with_format(format, [&](auto f) {
    constexpr int F = decltype(f)::value;
    auto go = [&](auto keep, auto u) {
      constexpr int U = decltype(u)::value;
      hipLaunchKernelGGL((mx_encode<F, decltype(keep)::value, U>), dim3(store_grid(total, U)),
                         dim3(256), 0, s, x, ldx, codes, scales, (int)C, (uint32_t)G,
                         (uint32_t)total);
    };
    auto by_size = [&](auto keep) {
      if (total >= STORE_MANY) go(keep, std::integral_constant<int, 4>());
      else go(keep, std::integral_constant<int, 1>());
    };
    if constexpr (F == MX_E2M1) by_size(std::false_type());  // (refused with keep_nonzero)
    else if (keep_nonzero) by_size(std::true_type());
    else by_size(std::false_type());
  });
  return hipGetLastError();
}

hipError_t launch_mx_decode(const uint8_t* codes, const uint8_t* scales, float* y, int64_t ldy,
                            int64_t R, int64_t C, int format, hipStream_t s) {
  const int64_t G = mx_groups(C), total = R * G;
  if (total <= 0) return hipSuccess;
  mx_with_format(format, [&](auto f) {
    constexpr int F = decltype(f)::value;
    auto go = [&](auto u) {
      constexpr int U = decltype(u)::value;
      hipLaunchKernelGGL((mx_decode<F, U>), dim3(store_grid(total, U)), dim3(256), 0, s, codes,
                         scales, y, ldy, (int)C, (uint32_t)G, (uint32_t)total);
    };
    if (total >= STORE_MANY) go(std::integral_constant<int, 4>());
    else go(std::integral_constant<int, 1>());
  });
  return hipGetLastError();
}

int64_t mx_act_grad_partial_doubles(int64_t R, int64_t C) {
  if (R <= 0 || C <= 0 || whole_sums(R, C)) return 0;
  const int64_t rows = act_grad_rows(R, C);
  return (R + rows - 1) / rows * C;
}

hipError_t launch_mx_act_grad(const float* dy, int64_t ldy, const uint8_t* codes,
                              const uint8_t* scales, float* dz, int64_t ldz, float* colsum, int64_t R,
                              int64_t C, int format, int act, double* partial, hipStream_t s) {
  if (C <= 0) return hipSuccess;
  const bool whole = colsum != nullptr && whole_sums(R, C);
  const int64_t G = mx_groups(C), rows = whole ? R : act_grad_rows(R, C);
  const int64_t slabs = whole ? 1 : (R + rows - 1) / rows;
  if (slabs > 0) {
    mx_with_format(format, [&](auto f) {
      constexpr int F = decltype(f)::value;
      auto go = [&](auto a) {
        constexpr int ACT = decltype(a)::value;
        auto with = [&](auto sums, void* to) {
          constexpr int SUMS = decltype(sums)::value, COLS = SUMS == WHOLE ? 32 : 256;
          const dim3 grid((unsigned)((C + COLS - 1) / COLS), (unsigned)slabs);
          hipLaunchKernelGGL((mx_act_grad<F, ACT, SUMS>), grid, dim3(SUMS == WHOLE ? 1024 : 256), 0, s, dy,
                             ldy, codes, scales, dz, ldz, to, R, (int)C, G, rows);
        };
        if (colsum == nullptr) with(std::integral_constant<int, NO_SUMS>(), nullptr);
        else if (whole) with(std::integral_constant<int, WHOLE>(), colsum);
        else with(std::integral_constant<int, PARTIAL>(), partial);
      };
      switch (act) {
        case ACT_RELU: go(std::integral_constant<int, ACT_RELU>()); break;
        case ACT_TANH: go(std::integral_constant<int, ACT_TANH>()); break;
        case ACT_SIGMOID: go(std::integral_constant<int, ACT_SIGMOID>()); break;
        default: go(std::integral_constant<int, ACT_NONE>()); break;
      }
    });
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (colsum == nullptr || whole) return hipSuccess;
  return launch_colsum_finish(partial, colsum, slabs, C, s);
}

}  // namespace shk
