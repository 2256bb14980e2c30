// Gated linear recurrence along the second axis of [B, T, D], and its backward pass.
//
//   f = 1 / (1 + exp(-z)),  h_t = f_t h_{t-1} + (1 - f_t) u_t,  h_{-1} = h0 (zero without one)
//   G_t  = dh_t + f_{t+1} G_{t+1}, at the last position dh + dlast
//   du_t = (1 - f_t) G_t,  dz_t = G_t (h_{t-1} - u_t) f_t (1 - f_t),  dh0 = f_0 G_0
//
// Each of the B D channels is a chain of steps s -> f s + b (forward b = (1 - f) u; backward, from
// the last position on, b = f dh and s = f_t G_t), and a run of steps is again such a step: its
// product of f and its result from s = 0. So a workgroup takes 64 channels, one a lane, its NW waves
// take TS consecutive positions each, form their runs' steps, read each other's from LDS, and
// carry on from their own first state: one pass over the data, whose positions' gates stay in
// registers. Where there are too few channels for the CUs, the positions are cut into chunks: a
// launch forms the chunks' steps, a second carries the state through them, a third is the pass
// above from each chunk's first state.
//
// States and products are binary32, as the outputs are; a gate and its complement come from one
// binary64 exponential, so that 1 - f keeps its bits where f is near one. A sequence shorter than T
// holds its state behind its end (f = 1, b = 0): its last state, and the gradient that enters there,
// need no case of their own. Positions behind the end are not read; their outputs are zero.
#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace shk {
namespace {

// f = sigmoid(z) and k = 1 - f, each rounded once (fexp64.h).
__device__ __forceinline__ void gates(float z, float& f, float& k) {
  const ExpParts p = exp_parts(-(double)fminf(fabsf(z), 110.0f));
  const double e = fma(p.p, p.scale, p.scale);
  const float a = (float)quotient_12(1.0, 1.0 + e), b = (float)quotient_12(e, 1.0 + e);
  f = z != z ? z : z >= 0.0f ? a : b;
  k = z != z ? z : z >= 0.0f ? b : a;
}

enum Mode { WHOLE, STEPS, CHUNK };  // the one pass; a chunk's step alone; a chunk from its first state

struct ScanArgs {
  const float* z;
  const float* u;
  const float* h;       // backward: the forward pass' states
  const float* dh;      // backward
  const float* first;   // [B, D]: h0 forward, dlast backward; null: zero
  const float* h0;      // backward: the state before position 0; null: zero
  float* out[2];        // forward: h; backward: dz, du
  float* last;          // [B, D]: the state behind the last step; null: not wanted
  const void* lengths;  // [B]; null: all T
  uint32_t* status;
  float* step_f;        // [chunks][B D]: the chunks' steps, and their first states
  float* step_b;
  float* state;
  int64_t B, T, D, chunk, chunks;  // chunk: positions of one; chunks > 1: split
  int len64;
};

__device__ __forceinline__ int64_t scan_length(const ScanArgs& a, int64_t b, bool flag) {
  if (a.lengths == nullptr) return a.T;
  const int64_t n = a.len64 ? static_cast<const int64_t*>(a.lengths)[b]
                            : (int64_t) static_cast<const int32_t*>(a.lengths)[b];
  if (n < 0 || n > a.T) {
    if (flag) atomicOr(a.status, (uint32_t)DEV_INDEX_OUT_OF_BOUNDS);
    return n < 0 ? 0 : a.T;
  }
  return n;
}

// What a position reads: forward z, u; backward z, dh, u, h_{t-1} (a chunk's step: z and dh).
template <bool BACK>
struct Position {
  float z, u;
  float dh, hp;
};

template <bool BACK, int MODE, int NW, int CW, int TS>
__global__ void __launch_bounds__(64 * NW * CW) scan_kernel(ScanArgs a) {
  __shared__ float2 steps[2][NW * CW][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int tw = NW > 1 ? w : 0;
  const int64_t channels = a.B * a.D;
  const int64_t groups = (channels + 64 * CW - 1) / (64 * CW);
  for (int64_t unit = blockIdx.x; unit < groups * a.chunks; unit += gridDim.x) {
    const int64_t piece = unit / groups;  // in the order of the steps
    const int64_t n0 = (unit % groups) * (64 * CW) + (CW > 1 ? w * 64 : 0) + lane;
    const bool live = n0 < channels;
    const int64_t n = live ? n0 : channels - 1;
    const int64_t seq = n / a.D, base = seq * a.T * a.D + (n - seq * a.D);
    const int64_t len = scan_length(a, seq, live && piece == 0);
    // steps [lo, hi) of this piece; step p is position p forward, T - 1 - p backward
    const int64_t lo = piece * a.chunk, hi = min(a.T, lo + a.chunk);
    auto position = [&](int64_t p) { return BACK ? a.T - 1 - p : p; };

    auto load = [&](Position<BACK> (&q)[TS], int64_t p0) {
#pragma unroll
      for (int i = 0; i < TS; ++i) {
        const int64_t p = p0 + i, t = position(p);
        const bool in = p < hi && t < len && live;
        const int64_t at = base + t * a.D;
        q[i].z = in ? __builtin_nontemporal_load(a.z + at) : 0.0f;
        if (!BACK) {
          q[i].u = in ? __builtin_nontemporal_load(a.u + at) : 0.0f;
        } else {
          q[i].dh = in ? __builtin_nontemporal_load(a.dh + at) : 0.0f;
          if (MODE != STEPS) {
            q[i].u = in ? __builtin_nontemporal_load(a.u + at) : 0.0f;
            q[i].hp = !in ? 0.0f : t > 0 ? __builtin_nontemporal_load(a.h + at - a.D)
                                 : a.h0 != nullptr ? a.h0[n] : 0.0f;
          }
        }
      }
    };

    float state = 0.0f, all = 1.0f;
    if (MODE == WHOLE) state = a.first != nullptr ? a.first[n] : 0.0f;
    if (MODE == CHUNK) state = a.state[piece * channels + n];
    Position<BACK> next[TS];
    load(next, lo + tw * TS);
    int turn = 0;
    for (int64_t p0 = lo; p0 < hi; p0 += NW * TS, turn ^= 1) {
      float f[TS], k[TS], b[TS], v[TS], w2[TS];
#pragma unroll
      for (int i = 0; i < TS; ++i) {
        const int64_t p = p0 + tw * TS + i, t = position(p);
        if (p < hi) {
          gates(next[i].z, f[i], k[i]);
          if (!(t < len)) f[i] = 1.0f;
          if (BACK) {
            v[i] = next[i].dh;
            b[i] = f[i] * v[i];
            if (MODE != STEPS) w2[i] = (next[i].hp - next[i].u) * (f[i] * k[i]);
          } else {
            b[i] = t < len ? k[i] * next[i].u : 0.0f;
          }
        } else {
          f[i] = 1.0f;
          b[i] = k[i] = v[i] = w2[i] = 0.0f;
        }
      }
      if (p0 + NW * TS < hi) load(next, p0 + (NW + tw) * TS);
      float s = state;
      if (NW > 1 || MODE == STEPS) {
        float run_f = 1.0f, run_b = 0.0f;
#pragma unroll
        for (int i = 0; i < TS; ++i) {
          run_b = fmaf(f[i], run_b, b[i]);
          run_f *= f[i];
        }
        if (NW > 1) {
          steps[turn][w][lane] = make_float2(run_f, run_b);
          __syncthreads();
#pragma unroll
          for (int j = 0; j < NW; ++j) {
            const float2 g = steps[turn][j][lane];
            if (j == tw) s = state;
            state = fmaf(g.x, state, g.y);
            all *= g.x;
          }
        } else {
          state = fmaf(run_f, state, run_b);
          all *= run_f;
        }
      }
      if (MODE != STEPS) {
#pragma unroll
        for (int i = 0; i < TS; ++i) {
          const int64_t p = p0 + tw * TS + i, t = position(p);
          const bool in = p < hi && live, real = t < len;
          const int64_t at = base + t * a.D;
          if (BACK) {
            const float g = v[i] + s;
            if (in) {
              __builtin_nontemporal_store(real ? g * w2[i] : 0.0f, a.out[0] + at);
              __builtin_nontemporal_store(real ? g * k[i] : 0.0f, a.out[1] + at);
            }
            s = fmaf(f[i], s, b[i]);
          } else {
            s = fmaf(f[i], s, b[i]);
            if (in) __builtin_nontemporal_store(real ? s : 0.0f, a.out[0] + at);
          }
        }
        if (NW == 1) state = s;
      }
    }
    if (tw == 0 && live) {
      if (MODE == WHOLE && a.last != nullptr) a.last[n] = state;
      if (MODE == STEPS) {
        a.step_f[piece * channels + n] = all;
        a.step_b[piece * channels + n] = state;
      }
    }
    if (NW > 1) __syncthreads();  // the steps in LDS have been read
  }
}

// The state before each chunk, and behind the last.
__global__ void __launch_bounds__(64) scan_carry(ScanArgs a) {
  const int64_t channels = a.B * a.D;
  for (int64_t n = (int64_t)blockIdx.x * 64 + threadIdx.x; n < channels; n += (int64_t)gridDim.x * 64) {
    float state = a.first != nullptr ? a.first[n] : 0.0f;
#pragma unroll 8
    for (int64_t i = 0; i < a.chunks; ++i) {
      a.state[i * channels + n] = state;
      state = fmaf(a.step_f[i * channels + n], state, a.step_b[i * channels + n]);
    }
    if (a.last != nullptr) a.last[n] = state;
  }
}

// Positions of a chunk: all of them where the channels fill the CUs or there is little to split.
constexpr int64_t SCAN_GROUPS = 512, SCAN_LEAST = 512;
int64_t scan_chunk(int64_t B, int64_t T, int64_t D) {
  const int64_t groups = (B * D + 63) / 64;
  if (groups >= SCAN_GROUPS / 2 || T < 2 * SCAN_LEAST) return T;
  const int64_t chunks = std::min(T / SCAN_LEAST, (SCAN_GROUPS + groups - 1) / groups);
  return chunks <= 1 ? T : ((T + chunks - 1) / chunks + 255) / 256 * 256;
}

template <bool BACK>
hipError_t launch_scan(ScanArgs a, float* scratch, hipStream_t s) {
  const int64_t channels = a.B * a.D;
  auto blocks = [&](int64_t wide) {
    return dim3((unsigned)std::min<int64_t>((channels + wide - 1) / wide * a.chunks, 1 << 20));
  };
  constexpr int TS = BACK ? 8 : 16;
  a.chunk = std::max<int64_t>(1, scan_chunk(a.B, a.T, a.D));
  a.chunks = std::max<int64_t>(1, (a.T + a.chunk - 1) / a.chunk);
  if (a.chunks > 1) {
    a.step_f = scratch;
    a.step_b = scratch + a.chunks * channels;
    a.state = scratch + 2 * a.chunks * channels;
    hipLaunchKernelGGL((scan_kernel<BACK, STEPS, 16, 1, TS>), blocks(64), dim3(1024), 0, s, a);
    hipLaunchKernelGGL(scan_carry, dim3((unsigned)((channels + 63) / 64)), dim3(64), 0, s, a);
    hipLaunchKernelGGL((scan_kernel<BACK, CHUNK, 16, 1, TS>), blocks(64), dim3(1024), 0, s, a);
  } else if (a.T <= 8) {
    hipLaunchKernelGGL((scan_kernel<BACK, WHOLE, 1, 4, 4>), blocks(256), dim3(256), 0, s, a);
  } else if (a.T <= 4 * TS) {
    hipLaunchKernelGGL((scan_kernel<BACK, WHOLE, 4, 1, TS>), blocks(64), dim3(256), 0, s, a);
  } else {
    hipLaunchKernelGGL((scan_kernel<BACK, WHOLE, 16, 1, TS>), blocks(64), dim3(1024), 0, s, a);
  }
  return hipGetLastError();
}

}  // namespace

int64_t gated_scan_scratch_bytes(int64_t B, int64_t T, int64_t D) {
  if (B <= 0 || T <= 0 || D <= 0) return 0;
  const int64_t chunk = scan_chunk(B, T, D), chunks = (T + chunk - 1) / chunk;
  return chunks > 1 ? 12 * chunks * B * D : 0;
}

hipError_t launch_gated_scan(const GatedScanParams& p, float* scratch, uint32_t* status, hipStream_t s) {
  if (p.B <= 0 || p.D <= 0) return hipSuccess;
  ScanArgs a{};
  a.z = p.z;
  a.u = p.u;
  a.first = p.h0;
  a.out[0] = p.h;
  a.last = p.last;
  a.lengths = p.lengths;
  a.len64 = p.len64;
  a.status = status;
  a.B = p.B;
  a.T = p.T;
  a.D = p.D;
  return launch_scan<false>(a, scratch, s);
}

hipError_t launch_gated_scan_grad(const GatedScanGradParams& p, float* scratch, uint32_t* status, hipStream_t s) {
  if (p.B <= 0 || p.D <= 0) return hipSuccess;
  ScanArgs a{};
  a.z = p.z;
  a.u = p.u;
  a.h = p.h;
  a.dh = p.dh;
  a.first = p.dlast;
  a.h0 = p.h0;
  a.out[0] = p.dz;
  a.out[1] = p.du;
  a.last = p.dh0;
  a.lengths = p.lengths;
  a.len64 = p.len64;
  a.status = status;
  a.B = p.B;
  a.T = p.T;
  a.D = p.D;
  return launch_scan<true>(a, scratch, s);
}

}  // namespace shk
