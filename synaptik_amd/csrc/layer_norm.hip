// Layer norm over the last axis of X [R, C] and its backward pass.
//
//   mean = sum x / C, var = sum (x - mean)^2 / C, rstd = 1 / sqrt(var + eps)
//   y  = (x - mean) rstd gamma + beta                              (gamma, beta optional)
//   g  = dy gamma,  xh = (x - mean) rstd
//   dx = rstd (g - sum g / C - xh sum (g xh) / C)
//   dgamma = sum over rows of dy xh,  dbeta = sum over rows of dy
//
// Bound: memory. A row is read once and held in registers through its statistics, and the backward
// pass forms them again from the x that it reads anyway, so that nothing but x is kept between the
// two and a mean far from zero is not rounded to binary32 on the way. The mean and the sum of
// squares about it are binary64, as are all sums. dgamma and dbeta are summed beside dx: each
// workgroup takes every G-th group of rows, keeps its columns' sums in registers and writes one
// row of partial sums, which a second launch adds in a fixed order.
//
// All of a row's sums are formed at once, over d = x - x_0 instead of x - mean:
//   delta = sum d / C = mean - x_0,  var = sum d^2 / C - delta^2,
//   sum g (x - mean) = sum g d - delta sum g.
// As x_0 is a value of the row, delta^2 <= C var, so the difference loses at most log2 (C + 1) of the
// 53 bits of sums whose terms pass through some 30 roundings (a thread's values, then a tree): var
// is within 2^-33 of its value at 16384 columns, and exactly 0 for a constant row.
#include <algorithm>

#include "common.h"
#include "kernels.h"
#include "row4.h"
#include "wave_sum.h"

namespace shk {
namespace {

// A row in the registers of T threads, V groups of four floats each, T groups apart.
template <int T, int V>
struct Row {
  float4 v[V];
  // `rest`: the floats from this thread's first group to the row's end
  template <bool STREAM>
  __device__ __forceinline__ void load(const float* row, int t, int rest) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = ld4_at<STREAM>(row, 16u * t + 16u * T * i, rest - 4 * T * i);
  }
  __device__ __forceinline__ void load_or(const float* row, int t, int rest, float otherwise) {
    if (row != nullptr) return load<false>(row, t, rest);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = make_float4(otherwise, otherwise, otherwise, otherwise);
  }
};
#define LN_EACH(i, j, c, C)                                      \
  _Pragma("unroll") for (int i = 0; i < V; ++i)                  \
    _Pragma("unroll") for (int j = 0; j < 4; ++j)                \
      if (const int64_t c = 4 * (t + (int64_t)i * T) + j; c < (C))

__device__ __forceinline__ float& at(float4& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }
__device__ __forceinline__ float at(const float4& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }

// Sums of a row that T threads hold.
template <int NT, int T, int K>
__device__ __forceinline__ void row_sums(double (&v)[K], double* lds) {
  if constexpr (T < NT) team_sums<T, K>(v);
  else group_sums<NT, K>(v, lds);
}
// The mean of squares less the square of the mean, not below zero (NaN stays).
__device__ __forceinline__ double variance(double squares, double delta) {
  const double v = fma(-delta, delta, squares);
  return v < 0.0 ? 0.0 : v;
}

struct FwdArgs {
  const float* x;
  const float* gamma;
  const float* beta;
  float* y;
  int64_t R, C, ldx, ldy;
  double eps, inv_C;
};

// T threads a row: a part of a wave, or the whole workgroup. [16384, 4096], 537 MB, takes 107 us, 5.0 TB/s;
// one row of 4096 3.1 us, a launch.
template <int NT, int T, int V, bool STREAM>
__global__ void __launch_bounds__(NT) ln_fwd(FwdArgs a) {
  __shared__ double lds[2][2 * (NT / 64)];
  int turn = 0;
  const int t = threadIdx.x % T, rest = (int)a.C - 4 * t;
  Row<T, V> gm, bt;
  gm.load_or(a.gamma, t, rest, 1.0f);
  bt.load_or(a.beta, t, rest, 0.0f);
  for (int64_t r = (int64_t)blockIdx.x * (NT / T) + threadIdx.x / T; r < a.R; r += (int64_t)gridDim.x * (NT / T)) {
    const float* row = a.x + r * a.ldx;
    const float x0 = row[0];
    Row<T, V> x;
    x.template load<STREAM>(row, t, rest);
    double s[2] = {0.0, 0.0};
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double d = (double)(j < rest - 4 * T * i ? at(x.v[i], j) : x0) - (double)x0;
        s[0] += d;
        s[1] = fma(d, d, s[1]);
      }
    row_sums<NT, T>(s, lds[turn]);
    turn ^= 1;
    const double delta = s[0] * a.inv_C, rstd = 1.0 / sqrt(variance(s[1] * a.inv_C, delta) + a.eps);
    float* y = a.y + r * a.ldy;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        at(o, j) = fmaf((float)((((double)at(x.v[i], j) - (double)x0) - delta) * rstd), at(gm.v[i], j), at(bt.v[i], j));
      st4_at<STREAM>(y, 16u * t + 16u * T * i, rest - 4 * T * i, o);
    }
  }
}

// Rows too wide for registers: three readings by one workgroup.
constexpr int LN_WIDE = 1024;
__device__ __forceinline__ void wide_stats(const float* x, int64_t C, double eps, double (*lds)[LN_WIDE / 64],
                                           double& mean, double& rstd) {
  double s[1] = {0.0}, q[1] = {0.0};
  for (int64_t c = 4 * threadIdx.x; c < C; c += 4 * LN_WIDE) {
    const float4 v = ld4(x + c, C - c);
    s[0] += ((double)v.x + (double)v.y) + ((double)v.z + (double)v.w);
  }
  group_sums<LN_WIDE, 1>(s, lds[0]);
  mean = s[0] / (double)C;
  for (int64_t c = 4 * threadIdx.x; c < C; c += 4 * LN_WIDE) {
    const float4 v = ld4(x + c, C - c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double d = c + j < C ? (double)at(v, j) - mean : 0.0;
      q[0] = fma(d, d, q[0]);
    }
  }
  group_sums<LN_WIDE, 1>(q, lds[1]);
  rstd = 1.0 / sqrt(q[0] / (double)C + eps);
}
__global__ void __launch_bounds__(LN_WIDE) ln_fwd_wide(FwdArgs a) {
  __shared__ double lds[2][LN_WIDE / 64];
  for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
    const float* x = a.x + r * a.ldx;
    double mean, rstd;
    wide_stats(x, a.C, a.eps, lds, mean, rstd);
    float* y = a.y + r * a.ldy;
    for (int64_t c = 4 * threadIdx.x; c < a.C; c += 4 * LN_WIDE) {
      const float4 v = ld4(x + c, a.C - c);
      const float4 gm = a.gamma != nullptr ? ld4(a.gamma + c, a.C - c) : make_float4(1.f, 1.f, 1.f, 1.f);
      const float4 bt = a.beta != nullptr ? ld4(a.beta + c, a.C - c) : make_float4(0.f, 0.f, 0.f, 0.f);
      float4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        at(o, j) = fmaf((float)(((double)at(v, j) - mean) * rstd), at(gm, j), at(bt, j));
      st4(y + c, a.C - c, o);
    }
  }
}

struct BwdArgs {
  const float* dy;
  const float* x;
  const float* gamma;
  float* dx;
  double* part;   // [gridDim.x][2][C]: partial sums of dgamma and dbeta; null: neither is wanted
  double* stats;  // [R][2]: mean and rstd (wide rows)
  int64_t R, C, lddy, ldx, lddx;
  double eps, inv_C;
};

// Values that the compiler takes as new, so that it forms what depends on them again instead of
// holding it in registers.
template <int V>
__device__ __forceinline__ void forget(float4 (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) asm volatile("" : "+v"(v[i].x), "+v"(v[i].y), "+v"(v[i].z), "+v"(v[i].w));
}

// dy and dx may be the same memory: a thread writes the elements that it read. AHEAD: the next row is
// on its way while this one is summed.
template <int NT, int T, int V, bool AHEAD, bool STREAM>
__device__ __forceinline__ void ln_bwd_rows(const BwdArgs& a, double (*lds)[4 * (NT / 64)], double (*dbs)[NT],
                                            double (&dg)[V][4], double (&db)[V][4]) {
  const int t = threadIdx.x % T, rest = (int)a.C - 4 * t;
  Row<T, V> gm;
  if (AHEAD) gm.load_or(a.gamma, t, rest, 1.0f);
  // (up to 16384 columns leave no registers for them: they come from the caches twice a row, and the sums of
  // dbeta lie in LDS)
  auto gamma = [&](int i) {
    if (AHEAD) return gm.v[i];
    return a.gamma != nullptr ? ld4_at(a.gamma, 16u * t + 16u * T * i, rest - 4 * T * i)
                              : make_float4(1.f, 1.f, 1.f, 1.f);
  };
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      dg[i][j] = 0.0;
      if (AHEAD) db[i][j] = 0.0;
      else dbs[4 * i + j][threadIdx.x] = 0.0;
    }
  const int64_t step = (int64_t)gridDim.x * (NT / T);
  int64_t r = (int64_t)blockIdx.x * (NT / T) + threadIdx.x / T;
  Row<T, V> x, dy, nx, ndy;
  float x0, nx0 = 0.0f;
  auto fetch = [&](int64_t row) {
    nx0 = a.x[row * a.ldx];
    nx.template load<STREAM>(a.x + row * a.ldx, t, rest);
    ndy.template load<STREAM>(a.dy + row * a.lddy, t, rest);
  };
  if (AHEAD && r < a.R) fetch(r);
  for (int turn = 0; r < a.R; r += step, turn ^= 1) {
    if (!AHEAD) fetch(r);
    x = nx;
    dy = ndy;
    x0 = nx0;
    if (AHEAD && r + step < a.R) fetch(r + step);
    double s[4] = {0.0, 0.0, 0.0, 0.0};  // sums of d, d^2, g, g d
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float4 gi = gamma(i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double d = (double)(j < rest - 4 * T * i ? at(x.v[i], j) : x0) - (double)x0;
        const double g = (double)at(dy.v[i], j) * (double)at(gi, j);
        s[0] += d;
        s[1] = fma(d, d, s[1]);
        s[2] += g;
        s[3] = fma(g, d, s[3]);
      }
      if (!AHEAD) __builtin_amdgcn_sched_barrier(0);
    }
    row_sums<NT, T>(s, lds[turn]);
    const double delta = s[0] * a.inv_C, rstd = 1.0 / sqrt(variance(s[1] * a.inv_C, delta) + a.eps);
    // dx = rstd (g - c1 - (d - delta) c2)
    const double c1 = s[2] * a.inv_C, c2 = rstd * rstd * (fma(-delta, s[2], s[3]) * a.inv_C);
    const double slope = -rstd * c2, offset = rstd * fma(delta, c2, -c1), shift = -delta * rstd;
    forget(x.v);
    forget(dy.v);
    float* dx = a.dx + r * a.lddx;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float4 gi = gamma(i);
      float4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double d = (double)at(x.v[i], j) - (double)x0, v = (double)at(dy.v[i], j);
        at(o, j) = (float)fma(d, slope, fma(v * (double)at(gi, j), rstd, offset));
        dg[i][j] = fma(v, fma(d, rstd, shift), dg[i][j]);
        if (AHEAD) db[i][j] += v;
        else dbs[4 * i + j][threadIdx.x] += v;
      }
      st4_at<STREAM>(dx, 16u * t + 16u * T * i, rest - 4 * T * i, o);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// Four waves on each SIMD where a workgroup holds a row; a wave that holds one has up to 256 registers.
// [16384, 4096], 805 MB, takes 146 us, 5.5 TB/s; two rounds of sums a row (the mean first) took 156 us, and
// sums by shuffles 220. [3001, 1531], 55 MB, takes 20 us, of which some 8 pass before the first row is
// summed and after the last.
template <int NT, int T, int V, bool AHEAD, bool STREAM>
__global__ void __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(T == 64 ? 2 : 4))) ln_bwd(BwdArgs a) {
  __shared__ double lds[2][4 * (NT / 64)];
  const int t = threadIdx.x % T;
  double dg[V][4], db[V][4];
  if constexpr (AHEAD) {
    ln_bwd_rows<NT, T, V, AHEAD, STREAM>(a, lds, nullptr, dg, db);
  } else {
    __shared__ double dbs[4 * V][NT];
    ln_bwd_rows<NT, T, V, AHEAD, STREAM>(a, lds, dbs, dg, db);
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) db[i][j] = dbs[4 * i + j][threadIdx.x];
  }
  if (a.part == nullptr) return;
  double* out = a.part + (int64_t)blockIdx.x * 2 * a.C;
  if constexpr (T == NT) {
    LN_EACH(i, j, c, a.C) {
      out[c] = dg[i][j];
      out[a.C + c] = db[i][j];
    }
  } else {
    // the rows that a wave holds beside each other, then the four waves one after the other
    __shared__ double cols[2][4 * T * V];
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int o = 32; o >= T; o >>= 1) {
          dg[i][j] += __shfl_xor(dg[i][j], o, 64);
          db[i][j] += __shfl_xor(db[i][j], o, 64);
        }
    for (int w = 0; w < NT / 64; ++w) {
      if ((int)(threadIdx.x >> 6) == w && (threadIdx.x & 63) < T) {
        LN_EACH(i, j, c, a.C) {
          cols[0][c] = w == 0 ? dg[i][j] : cols[0][c] + dg[i][j];
          cols[1][c] = w == 0 ? db[i][j] : cols[1][c] + db[i][j];
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < (int)a.C; c += NT) {
      out[c] = cols[0][c];
      out[a.C + c] = cols[1][c];
    }
  }
}

__global__ void __launch_bounds__(LN_WIDE) ln_bwd_wide(BwdArgs a) {
  __shared__ double lds[5][LN_WIDE / 64];
  for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
    const float* x = a.x + r * a.ldx;
    const float* dy = a.dy + r * a.lddy;
    double mean, rstd;
    wide_stats(x, a.C, a.eps, lds, mean, rstd);
    double q[2] = {0.0, 0.0};
    for (int64_t c = 4 * threadIdx.x; c < a.C; c += 4 * LN_WIDE) {
      const float4 xv = ld4(x + c, a.C - c), v = ld4(dy + c, a.C - c);
      const float4 gm = a.gamma != nullptr ? ld4(a.gamma + c, a.C - c) : make_float4(1.f, 1.f, 1.f, 1.f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (c + j >= a.C) break;
        const double g = (double)at(v, j) * (double)at(gm, j);
        q[0] += g;
        q[1] = fma(g, (double)at(xv, j) - mean, q[1]);
      }
    }
    group_sums<LN_WIDE, 2>(q, lds[2]);
    const double c1 = q[0] * a.inv_C, c2 = rstd * rstd * (q[1] * a.inv_C);
    float* dx = a.dx + r * a.lddx;
    for (int64_t c = 4 * threadIdx.x; c < a.C; c += 4 * LN_WIDE) {
      const float4 xv = ld4(x + c, a.C - c), v = ld4(dy + c, a.C - c);
      const float4 gm = a.gamma != nullptr ? ld4(a.gamma + c, a.C - c) : make_float4(1.f, 1.f, 1.f, 1.f);
      float4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double g = (double)at(v, j) * (double)at(gm, j);
        at(o, j) = (float)(rstd * (fma(-((double)at(xv, j) - mean), c2, g) - c1));
      }
      st4(dx + c, a.C - c, o);
    }
  }
}

// Mean and rstd of every row.
__global__ void __launch_bounds__(LN_WIDE) ln_stats_wide(BwdArgs a) {
  __shared__ double lds[2][LN_WIDE / 64];
  for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
    double mean, rstd;
    wide_stats(a.x + r * a.ldx, a.C, a.eps, lds, mean, rstd);
    if (threadIdx.x == 0) {
      a.stats[2 * r] = mean;
      a.stats[2 * r + 1] = rstd;
    }
  }
}
// Partial column sums of wide rows from their statistics: 256 columns, every gridDim.y-th row.
__global__ void __launch_bounds__(256) ln_cols_wide(BwdArgs a) {
  for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < a.C; c += (int64_t)gridDim.x * 256) {
    double dg = 0.0, db = 0.0;
    for (int64_t r = blockIdx.y; r < a.R; r += gridDim.y) {
      const double v = (double)a.dy[r * a.lddy + c];
      dg = fma(v, ((double)a.x[r * a.ldx + c] - a.stats[2 * r]) * a.stats[2 * r + 1], dg);
      db += v;
    }
    double* out = a.part + (int64_t)blockIdx.y * 2 * a.C;
    out[c] = dg;
    out[a.C + c] = db;
  }
}

// Adds P rows of partial sums: 32 columns by 16 parts of the rows. 512 rows of 8192 take 5.9 us.
__global__ void __launch_bounds__(512) ln_finish(const double* __restrict__ part, int64_t P, int64_t C,
                                                 float* dgamma, float* dbeta) {
  __shared__ double sum[16][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  for (int64_t base = (int64_t)blockIdx.x * 32; base < 2 * C; base += (int64_t)gridDim.x * 32) {
    const int64_t c = base + x;
    double s = 0.0;
    if (c < 2 * C) {
#pragma unroll 4
      for (int64_t p = y; p < P; p += 16) s += part[p * 2 * C + c];
    }
    sum[y][x] = s;
    __syncthreads();
    if (y == 0 && c < 2 * C) {
      double all = sum[0][x];
      for (int i = 1; i < 16; ++i) all += sum[i][x];
      float* out = c < C ? dgamma : dbeta;
      if (out != nullptr) out[c < C ? c : c - C] = (float)all;
    }
    __syncthreads();
  }
}

constexpr int64_t LN_REGS = 16384;  // columns up to which a row is held in registers

// Rows that a workgroup of the backward pass takes at once, and the workgroups.
struct BwdShape {
  int64_t rows, groups;
};
BwdShape bwd_shape(int64_t R, int64_t C) {
  BwdShape b{};
  if (C > LN_REGS) {
    b.rows = 1;
    b.groups = std::min<int64_t>(R, 64);
  } else if (C > 1024) {
    b.rows = 1;
    // (a CU holds one workgroup of 1024 threads; each writes 16 C bytes of partial sums)
    b.groups = std::min<int64_t>(R, C > 4096 ? 256 : 512);
  } else {
    int64_t lanes = 2;
    while (lanes < 64 && 4 * lanes < C) lanes *= 2;
    b.rows = 256 / lanes;
    b.groups = std::min<int64_t>((R + b.rows - 1) / b.rows, 1024);
  }
  return b;
}

// Tensors beyond what the last-level cache holds go past it: the backward pass of [16384, 4096], 805
// MB, takes 161 us so, 174 us with plain writes and more with plain reads; [65536, 1000] 169 and 187
// us. That of [3001, 1531], 55 MB, takes 27 us so and 20 us through the caches.
bool streams(int64_t bytes) { return bytes > 256 << 20; }

template <int NT, int T, int V>
void launch_fwd(const FwdArgs& a, hipStream_t s) {
  const int64_t rows = NT / T;
  const unsigned g = (unsigned)std::min<int64_t>((a.R + rows - 1) / rows, 1 << 16);
  if (streams(8 * a.R * a.C)) hipLaunchKernelGGL((ln_fwd<NT, T, V, true>), dim3(g), dim3(NT), 0, s, a);
  else hipLaunchKernelGGL((ln_fwd<NT, T, V, false>), dim3(g), dim3(NT), 0, s, a);
}
template <int NT, int T, int V, bool AHEAD = true>
void launch_bwd(const BwdArgs& a, int64_t groups, hipStream_t s) {
  const dim3 g((unsigned)groups);
  if (streams(12 * a.R * a.C)) hipLaunchKernelGGL((ln_bwd<NT, T, V, AHEAD, true>), g, dim3(NT), 0, s, a);
  else hipLaunchKernelGGL((ln_bwd<NT, T, V, AHEAD, false>), g, dim3(NT), 0, s, a);
}

}  // namespace

hipError_t launch_layer_norm(const LayerNormParams& p, hipStream_t s) {
  if (p.R <= 0 || p.C <= 0) return hipSuccess;
  const FwdArgs a{p.x, p.gamma, p.beta, p.y, p.R, p.C, p.ldx, p.ldy, (double)p.eps, 1.0 / (double)p.C};
  // A wave or less a row up to 1024 columns ([65536, 1000] 106 us, a workgroup a row 142 us), then eight
  // columns a thread ([16384, 4096] 107 us, sixteen 111 us).
  if (p.C <= 8) launch_fwd<256, 2, 1>(a, s);
  else if (p.C <= 16) launch_fwd<256, 4, 1>(a, s);
  else if (p.C <= 32) launch_fwd<256, 8, 1>(a, s);
  else if (p.C <= 64) launch_fwd<256, 16, 1>(a, s);
  else if (p.C <= 128) launch_fwd<256, 32, 1>(a, s);
  else if (p.C <= 256) launch_fwd<256, 64, 1>(a, s);
  else if (p.C <= 512) launch_fwd<256, 64, 2>(a, s);
  else if (p.C <= 1024) launch_fwd<256, 64, 4>(a, s);
  else if (p.C <= 2048) launch_fwd<256, 256, 2>(a, s);
  else if (p.C <= 4096) launch_fwd<512, 512, 2>(a, s);
  else if (p.C <= 8192) launch_fwd<1024, 1024, 2>(a, s);
  else if (p.C <= LN_REGS) launch_fwd<1024, 1024, 4>(a, s);
  else
    hipLaunchKernelGGL(ln_fwd_wide, dim3((unsigned)std::min<int64_t>(p.R, 1 << 16)), dim3(LN_WIDE), 0, s, a);
  return hipGetLastError();
}

int64_t layer_norm_grad_scratch_bytes(int64_t R, int64_t C) {
  if (R <= 0 || C <= 0) return 0;
  return bwd_shape(R, C).groups * 16 * C + (C > LN_REGS ? 16 * R : 0);
}

hipError_t launch_layer_norm_grad(const LayerNormGradParams& p, double* scratch, hipStream_t s) {
  if (p.C <= 0) return hipSuccess;
  const bool sums = p.dgamma != nullptr || p.dbeta != nullptr;
  const BwdShape b = bwd_shape(p.R, p.C);
  BwdArgs a{p.dy, p.x, p.gamma, p.dx, sums ? scratch : nullptr, scratch + b.groups * 2 * p.C, p.R, p.C,
            p.lddy, p.ldx, p.lddx, (double)p.eps, 1.0 / (double)p.C};
  if (p.R > 0) {
    if (p.C <= 8) launch_bwd<256, 2, 1>(a, b.groups, s);
    else if (p.C <= 16) launch_bwd<256, 4, 1>(a, b.groups, s);
    else if (p.C <= 32) launch_bwd<256, 8, 1>(a, b.groups, s);
    else if (p.C <= 64) launch_bwd<256, 16, 1>(a, b.groups, s);
    else if (p.C <= 128) launch_bwd<256, 32, 1>(a, b.groups, s);
    else if (p.C <= 256) launch_bwd<256, 64, 1>(a, b.groups, s);
    else if (p.C <= 512) launch_bwd<256, 64, 2>(a, b.groups, s);
    else if (p.C <= 1024) launch_bwd<256, 64, 4>(a, b.groups, s);
    else if (p.C <= 2048) launch_bwd<256, 256, 2>(a, b.groups, s);
    else if (p.C <= 4096) launch_bwd<512, 512, 2>(a, b.groups, s);
    else if (p.C <= 8192) launch_bwd<1024, 1024, 2>(a, b.groups, s);
    else if (p.C <= LN_REGS) launch_bwd<1024, 1024, 4, false>(a, b.groups, s);
    else {
      const dim3 rows((unsigned)std::min<int64_t>(p.R, 1 << 16));
      if (sums) {
        // (before dx, which may take dy's place)
        hipLaunchKernelGGL(ln_stats_wide, rows, dim3(LN_WIDE), 0, s, a);
        hipLaunchKernelGGL(ln_cols_wide, dim3((unsigned)std::min<int64_t>((p.C + 255) / 256, 1 << 16), (unsigned)b.groups),
                           dim3(256), 0, s, a);
      }
      hipLaunchKernelGGL(ln_bwd_wide, rows, dim3(LN_WIDE), 0, s, a);
    }
  }
  if (sums)
    hipLaunchKernelGGL(ln_finish, dim3((unsigned)std::min<int64_t>((2 * p.C + 31) / 32, 1 << 20)), dim3(512), 0, s,
                       (const double*)scratch, p.R > 0 ? b.groups : 0, p.C, p.dgamma, p.dbeta);
  return hipGetLastError();
}

}  // namespace shk
