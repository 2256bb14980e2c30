// Gated linear recurrence along the second axis of [B, T, D], and its backward pass.
//
//   f = 1 / (1 + exp(-z)),  h_t = f_t h_{t-1} + (1 - f_t) u_t,  h_{-1} = h0 (zero without one)
//   G_t  = dh_t + f_{t+1} G_{t+1}, at the last position dh + dlast
//   du_t = (1 - f_t) G_t,  dz_t = G_t (h_{t-1} - u_t) f_t (1 - f_t),  dh0 = f_0 G_0
//
// Each of the B D channels is a chain of steps s -> f s + b (forward b = (1 - f) u; backward, from
// the last position on, s -> f (s + dh) with s = f_t G_t), and a run of steps is again such a step: its
// product of f and its result from s = 0. So a workgroup takes 64 channels, one a lane, its NW waves
// take TS consecutive positions each, form their runs' steps, read each other's from LDS, and
// carry on from their own first state: one pass over the data, whose positions' gates stay in
// registers. Where there are too few channels for the CUs, the positions are cut into chunks: a
// launch forms the chunks' steps, a second joins those before each chunk and is the pass above from
// there.
//
// A gate and its complement come from one binary64 exponential, so that 1 - f keeps its bits where f is
// near one. Rounded to binary32, f and 1 - f no longer add up to one: f is off by up to 3e-8, which a
// memory of 1 / (1 - f) positions adds up. So a run's product of gates is binary64, and so is the state that
// is handed from run to run: binary32 is what happens within the TS positions of one run, each run's result
// from s = 0, and the outputs. With z from 6 to 12 and u constant, begun with the state u, h was off by up to
// 8e-5 of u after 2048 positions and 1.3e-3 after 65536 with binary32 throughout, and is off by 2e-7. That
// costs 0 to 5 % of the time. (A call of up to 8 positions has no runs to join and is binary64 throughout;
// from call to call states are the binary32 values in memory.)
//
// A sequence shorter than T holds its state behind its end (z = inf there: f = 1, 1 - f = 0): its last
// state, and the gradient that enters there, need no case of their own. Positions behind the end are not
// read; their outputs are zero.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "flag.h"
#include "kernels.h"

namespace shk {
namespace {

// f = 1 / (1 + e) and k = e / (1 + e) with e = exp(-z), in binary64, k rounded once to binary32. e is
// 2^n exp(r), z = -(n ln2 + r), |r| <= 0.3466 (Cody and Waite, as in fexp64.h), with the Taylor
// polynomial to r^9 / 9!: what it leaves out is 0.3466^10 / 10! = 7e-12 of e, a ten-thousandth of a
// unit in binary32's last place of either. The reciprocal's estimate takes one Newton step. A gate beyond
// |z| = 700 leaves nothing of any binary32 state, or all of it, either way. This takes 30 vector operations, the functions of
// fexp64.h, which serve an exactness that two further roundings make moot here, 45.
__device__ __forceinline__ void gates(float z, double& f, float& k) {
  const double x = -(double)clamp_f(z, -700.0f, 700.0f);
  const double kd = fma(x, 0x1.71547652b82fep+0, 0x1.8p52);  // n in the low half
  const double n = kd - 0x1.8p52;
  double r = fma(-n, 0x1.62e42fefa39efp-1, x);
  r = fma(-n, 0x1.abc9e3b39803fp-56, r);
  double q = 1.0 / 362880.0;
  q = fma(q, r, 1.0 / 40320.0);
  q = fma(q, r, 1.0 / 5040.0);
  q = fma(q, r, 1.0 / 720.0);
  q = fma(q, r, 1.0 / 120.0);
  q = fma(q, r, 1.0 / 24.0);
  q = fma(q, r, 1.0 / 6.0);
  q = fma(q, r, 0.5);
  q = fma(q, r, 1.0);
  q = fma(q, r, 1.0);
  // 2^n: n from -1010 to 1010, added to the exponent
  const uint32_t hi = (uint32_t)__double2hiint(q) + ((uint32_t)__double2loint(kd) << 20);
  const double e = __hiloint2double(z != z ? 0x7ff80000 : (int)hi, __double2loint(q)), d = 1.0 + e;
  double y = __builtin_amdgcn_rcp(d);
  y = fma(fma(-d, y, 1.0), y, y);
  f = y;
  k = (float)(e * y);
}

// What bounds it: memory, if the 37 to 54 vector operations a position and channel (30 of them the gate) run beside the
// loads. So a wave's next positions are on their way while it works on these, addresses are the wave's
// (a scalar base, a lane's offset), and nothing spills. [16, 4096, 1024] backward, 1.6 GB, takes 308 us in
// one pass, 5.2 TB/s (lanes' own 64-bit addresses and spills: 2030 us); [1, 65536, 512] forward, 403 MB,
// 51 us for the chunks' steps and 67 us for the pass, whose first reading the caches keep part of.
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
  FlagWord flag;
  double2* step;        // [chunks][B D]: the chunks' steps
  float* state;         // [B D]: a copy of the first states
  int64_t B, T, D, chunk, chunks;  // chunk: positions of one; chunks > 1: split
  int64_t waves, parts;  // groups of up to 64 channels: of all sequences, of one
  int pack, lanes;       // sequences a wave takes, lanes of each
  int len64;
};

__device__ __forceinline__ int64_t scan_length(const ScanArgs& a, int64_t b, bool flags) {
  if (a.lengths == nullptr) return a.T;
  const int64_t n = a.len64 ? static_cast<const int64_t*>(a.lengths)[b]
                            : (int64_t) static_cast<const int32_t*>(a.lengths)[b];
  if (n < 0 || n > a.T) {
    if (flags) flag_out_of_bounds(a.flag);
    return n < 0 ? 0 : a.T;
  }
  return n;
}

template <bool BACK, int MODE, int NW, int CW, int TS, bool STREAM = false>
__global__ void __launch_bounds__(64 * NW * CW) scan_kernel(ScanArgs a) {
  constexpr int READS = !BACK || MODE == STEPS ? 2 : 4;  // z and u; z and dh; z, dh, u and h_{t-1}
  static_assert(NW > 1 || MODE == WHOLE);
  using F = std::conditional_t<NW == 1, double, float>;  // within a run (a wave by itself has one run)
  __shared__ double2 steps[2][NW * CW][64];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tw = NW > 1 ? w : 0;
  const int64_t width = a.T * a.D;  // floats of a sequence
  const int64_t blocks = (a.waves + CW - 1) / CW;
  for (int64_t unit = blockIdx.x; unit < blocks * a.chunks; unit += gridDim.x) {
    // (the chunks' second reading begins with those that the first one read last)
    const int64_t piece = MODE == CHUNK ? a.chunks - 1 - unit / blocks : unit / blocks;
    const int64_t wave = (unit % blocks) * CW + (CW > 1 ? w : 0);
    // this wave's channels: 64 of one sequence, or those of `pack` short ones
    const int64_t first_seq = wave / a.parts * a.pack, part = wave % a.parts;
    const int sub = a.pack > 1 ? lane / a.lanes : 0, c = (int)part * 64 + (a.pack > 1 ? lane % a.lanes : lane);
    const bool live = wave < a.waves && sub < a.pack && c < a.D && first_seq + sub < a.B;
    const int64_t seq = live ? first_seq + sub : 0, n = seq * a.D + (live ? c : 0);
    const int64_t base = first_seq * width + part * 64;
    const uint32_t at = 4u * (uint32_t)(sub * width + (c - (int)part * 64));  // bytes from there
    const int len = (int)scan_length(a, seq, live && piece == 0);
    // steps [lo, hi) of this piece; step p is position p forward, T - 1 - p backward; this lane's
    // sequence has those of [from, to)
    const int T = (int)a.T, lo = (int)(piece * a.chunk), hi = (int)min(a.T, piece * a.chunk + a.chunk);
    const int from = BACK ? T - len : 0, to = BACK ? T : len;
    const int64_t dir = BACK ? -a.D : a.D;
    auto row = [&](const float* x, int p) { return x + base + (int64_t)(BACK ? T - 1 - p : p) * a.D; };
    auto get = [&](const float* x) {
      const float* p = reinterpret_cast<const float*>(reinterpret_cast<const char*>(x) + at);
      return STREAM && MODE == WHOLE ? __builtin_nontemporal_load(p) : *p;
    };
    auto put = [&](float* x, float v) {
      float* p = reinterpret_cast<float*>(reinterpret_cast<char*>(x) + at);
      if (STREAM) __builtin_nontemporal_store(v, p);
      else *p = v;
    };
    const float* const src[4] = {a.z, BACK ? a.dh : a.u, a.u, a.h};
    // steps p0 .. p0 + TS - 1 are positions of every lane's sequence in this piece
    auto whole = [&](int p0) { return p0 + TS <= hi && __all(!live || (from <= p0 && p0 + TS <= to)); };
    float next[READS][TS];
    auto load = [&](int p0) {
      if (whole(p0) && (READS < 4 || p0 + TS < T)) {  // (before position 0 there is h0)
        if (live) {
#pragma unroll
          for (int r = 0; r < READS; ++r) {
            const float* x = row(src[r], p0) - (r == 3 ? a.D : 0);
#pragma unroll
            for (int i = 0; i < TS; ++i, x += dir) next[r][i] = get(x);
          }
        }
        return;
      }
#pragma unroll
      for (int i = 0; i < TS; ++i) {
        const int p = p0 + i;
        const bool in = live && p < hi && p >= from && p < to;
#pragma unroll
        for (int r = 0; r < READS; ++r) {
          next[r][i] = r == 0 ? INFINITY : 0.0f;  // a position that is not there holds the state
          if (in) {
            if (r < 3 || p < T - 1) next[r][i] = get(row(src[r], p) - (r == 3 ? a.D : 0));
            else next[r][i] = a.h0 != nullptr ? a.h0[n] : 0.0f;
          }
        }
      }
    };

    double state = 0.0, all = 1.0;
    if (MODE == WHOLE) state = a.first != nullptr ? (double)a.first[n] : 0.0;
    load(lo + tw * TS);
    int turn = 0;
    if (MODE == CHUNK) {
      // the steps of the chunks before: each wave joins consecutive ones, all join the waves'
      state = (double)a.state[n];
      const int64_t share = (piece + NW - 1) / NW, end = min(piece, (tw + 1) * share);
      double run_f = 1.0, run_b = 0.0;
#pragma unroll 4
      for (int64_t i = min(piece, tw * share); i < end; ++i) {
        const double2 g = a.step[i * a.B * a.D + n];
        run_b = fma(g.x, run_b, g.y);
        run_f *= g.x;
      }
      steps[turn][w][lane] = make_double2(run_f, run_b);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NW; ++j) {
        const double2 g = steps[turn][j][lane];
        state = fma(g.x, state, g.y);
      }
      turn ^= 1;
    }
    for (int p0 = lo; p0 < hi; p0 += NW * TS, turn ^= 1) {
      const int q0 = p0 + tw * TS;
      F f[TS], b[TS], k[TS], v[TS], m[TS];
      double run_f = 1.0;
#pragma unroll
      for (int i = 0; i < TS; ++i) {
        double gate;
        float let;
        gates(next[0][i], gate, let);
        f[i] = (F)gate;
        k[i] = (F)let;
        run_f *= gate;
        if (BACK) {
          v[i] = (F)next[1][i];
          if (MODE != STEPS) m[i] = ((F)next[3][i] - (F)next[2][i]) * (f[i] * k[i]);
        } else {
          b[i] = k[i] * (F)next[1][i];
        }
        __builtin_amdgcn_sched_barrier(0);  // one gate's binary64 values at a time
      }
      const bool inside = whole(q0);
      // (what these are without: z = inf, the rest 0. Forming them apart keeps the registers below 128.)
      if (BACK && MODE != STEPS && !inside) {
#pragma unroll
        for (int i = 0; i < TS; ++i) {
          const bool in = q0 + i < hi && q0 + i >= from && q0 + i < to;
          f[i] = in ? f[i] : (F)1;
          m[i] = in ? m[i] : (F)0;
          k[i] = in ? k[i] : (F)0;
          v[i] = in ? v[i] : (F)0;
        }
      }
      if (p0 + NW * TS < hi) load(q0 + NW * TS);
      F s = (F)state;
      if (NW > 1) {
        F run_b = 0;
#pragma unroll
        for (int i = 0; i < TS; ++i) run_b = BACK ? f[i] * (run_b + v[i]) : fma(f[i], run_b, b[i]);
        steps[turn][w][lane] = make_double2(run_f, (double)run_b);
        __syncthreads();
        if (MODE == STEPS && tw != 0) continue;  // (one wave keeps the chunk's step)
#pragma unroll 4  // (all at once take 32 more registers)
        for (int j = 0; j < NW; ++j) {
          const double2 g = steps[turn][j][lane];
          if (j == tw) s = (F)state;
          state = fma(g.x, state, g.y);
          all *= g.x;
        }
      }
      if (MODE != STEPS && live) {
        float* x[2] = {const_cast<float*>(row(a.out[0], q0)), BACK ? const_cast<float*>(row(a.out[1], q0)) : nullptr};
#pragma unroll
        for (int i = 0; i < TS; ++i, x[0] += dir, x[1] += BACK ? dir : 0) {
          if (q0 + i >= hi) break;
          if (BACK) {
            const F g = v[i] + s;
            float dz = (float)(g * m[i]), du = (float)(g * k[i]);
            if (!inside && q0 + i < from) dz = du = 0.0f;  // (a gradient that is not finite stays at the end)
            put(x[0], dz);
            put(x[1], du);
            s = f[i] * g;
          } else {
            s = fma(f[i], s, b[i]);
            put(x[0], q0 + i < to ? (float)s : 0.0f);
          }
        }
      }
      if (NW == 1) state = s;
    }
    if (tw == 0 && live) {
      if (MODE == STEPS) {
        a.step[piece * a.B * a.D + n] = make_double2(all, state);
        if (piece == 0) a.state[n] = a.first != nullptr ? a.first[n] : 0.0f;
      } else if (piece == a.chunks - 1 && a.last != nullptr) {
        a.last[n] = (float)state;  // (which may be `first`: the chunks read its copy)
      }
    }
    if (NW > 1) __syncthreads();  // the steps in LDS have been read
  }
}

// Lanes of a wave for one sequence of D channels: all 64, or the next power of two where several
// sequences' offsets stay within 32 bits.
int scan_lanes(int64_t B, int64_t T, int64_t D) {
  int lanes = 64;
  while (lanes > 1 && lanes / 2 >= D) lanes /= 2;
  return B > 1 && lanes < 64 && T * D <= (1 << 29) / (64 / lanes) ? lanes : 64;
}
int64_t scan_waves(int64_t B, int64_t T, int64_t D) {
  const int64_t pack = 64 / scan_lanes(B, T, D);
  return (B + pack - 1) / pack * ((D + 63) / 64);
}
// Positions of a chunk: all of them from SCAN_SPLIT groups of channels on, where the one pass takes
// no longer than two, whose first reads again two thirds (forward) or a third of what the pass moves:
// a call of [8, 4096, 1024], 128 groups, takes 133 us forward and 203 back in one, 134 and 219 in two. Else as
// many chunks as the CUs hold workgroups at once, three each forward and two back.
constexpr int64_t SCAN_SPLIT = 128, SCAN_LEAST = 128, SCAN_TILE = 64;
int64_t scan_chunk(int64_t B, int64_t T, int64_t D, bool back) {
  const int64_t groups = scan_waves(B, T, D);
  if (groups > SCAN_SPLIT || T < 2 * SCAN_LEAST) return T;
  const int64_t chunks = std::min(T / SCAN_LEAST, (back ? 512 : 768) / groups);
  return ((T + chunks - 1) / chunks + SCAN_TILE - 1) / SCAN_TILE * SCAN_TILE;
}
int64_t scan_bytes(int64_t B, int64_t T, int64_t D, bool back) {
  const int64_t chunk = scan_chunk(B, T, D, back), chunks = (T + chunk - 1) / chunk;
  return chunks > 1 ? 4 * (4 * chunks + 1) * B * D : 0;
}

template <bool BACK>
hipError_t launch_scan(ScanArgs a, float* scratch, hipStream_t s) {
  const int64_t channels = a.B * a.D;
  a.lanes = scan_lanes(a.B, a.T, a.D);
  a.pack = 64 / a.lanes;
  a.parts = (a.D + 63) / 64;
  a.waves = scan_waves(a.B, a.T, a.D);
  auto blocks = [&](int64_t waves) {
    return dim3((unsigned)std::min<int64_t>((a.waves + waves - 1) / waves * a.chunks, 1 << 20));
  };
  constexpr int TS = 8;
  a.chunk = std::max<int64_t>(1, scan_chunk(a.B, a.T, a.D, BACK));
  a.chunks = std::max<int64_t>(1, (a.T + a.chunk - 1) / a.chunk);
  // Whole lines of memory go past the caches where the tensors do not fit them: [16, 4096, 1024] backward
  // 313 us, 331 us with plain writes; [7, 1501, 617], whose waves share lines, 84 us so and 69 us through them.
  // What the chunks' first reading takes stays there for the second.
  const bool lines = a.D % 32 == 0 && (BACK ? 24 : 12) * channels * a.T > 256 << 20;
  if (a.chunks > 1) {
    a.step = reinterpret_cast<double2*>(scratch);
    a.state = scratch + 4 * a.chunks * channels;
    hipLaunchKernelGGL((scan_kernel<BACK, STEPS, 8, 1, TS>), blocks(1), dim3(512), 0, s, a);
    if (lines) hipLaunchKernelGGL((scan_kernel<BACK, CHUNK, 8, 1, TS, true>), blocks(1), dim3(512), 0, s, a);
    else hipLaunchKernelGGL((scan_kernel<BACK, CHUNK, 8, 1, TS>), blocks(1), dim3(512), 0, s, a);
  } else if (a.T <= 8) {
    hipLaunchKernelGGL((scan_kernel<BACK, WHOLE, 1, 4, 4>), blocks(4), dim3(256), 0, s, a);
  } else if (a.T <= 8 * TS) {
    hipLaunchKernelGGL((scan_kernel<BACK, WHOLE, 4, 1, TS>), blocks(1), dim3(256), 0, s, a);
  } else if (a.waves > 256) {
    if (lines) hipLaunchKernelGGL((scan_kernel<BACK, WHOLE, 8, 1, TS, true>), blocks(1), dim3(512), 0, s, a);
    else hipLaunchKernelGGL((scan_kernel<BACK, WHOLE, 8, 1, TS>), blocks(1), dim3(512), 0, s, a);
  } else {
    if (lines) hipLaunchKernelGGL((scan_kernel<BACK, WHOLE, 16, 1, TS, true>), blocks(1), dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((scan_kernel<BACK, WHOLE, 16, 1, TS>), blocks(1), dim3(1024), 0, s, a);
  }
  return hipGetLastError();
}

}  // namespace

int64_t gated_scan_scratch_bytes(int64_t B, int64_t T, int64_t D, bool back) {
  return B <= 0 || T <= 0 || D <= 0 ? 0 : scan_bytes(B, T, D, back);
}

hipError_t launch_gated_scan(const GatedScanParams& p, float* scratch, FlagWord flag, hipStream_t s) {
  if (p.B <= 0 || p.D <= 0) return hipSuccess;
  ScanArgs a{};
  a.z = p.z;
  a.u = p.u;
  a.first = p.h0;
  a.out[0] = p.h;
  a.last = p.last;
  a.lengths = p.lengths;
  a.len64 = p.len64;
  a.flag = flag;
  a.B = p.B;
  a.T = p.T;
  a.D = p.D;
  return launch_scan<false>(a, scratch, s);
}

hipError_t launch_gated_scan_grad(const GatedScanGradParams& p, float* scratch, FlagWord flag, hipStream_t s) {
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
  a.flag = flag;
  a.B = p.B;
  a.T = p.T;
  a.D = p.D;
  return launch_scan<true>(a, scratch, s);
}

}  // namespace shk
