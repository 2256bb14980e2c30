// Y = act(X . W^T + b) of microscaled weights W [N, K] (mx.h) and binary32 activations X [M, K],
// encoded here. The products of stored values (zero or in the normal range, mx.h) are exact in
// bfloat16's matrix instructions, and of e2m1 on both sides in the scaled ones, which run up to four
// times as fast (10 against 2.5 PFLOP/s); sums are binary32.
#include <algorithm>

#include "mx_tiles.h"

namespace shk {
namespace {

typedef int intx8 __attribute__((ext_vector_type(8)));

int64_t pad256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// 16 values of a row of which `rest` are in it.
__device__ __forceinline__ void load16(const float* x, int64_t rest, float (&v)[4][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (rest >= 4 * i + 4) {
      const float4u t = *reinterpret_cast<const float4u*>(x + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = t[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = 4 * i + j < rest ? x[4 * i + j] : 0.0f;
    }
  }
}
// The bits of the largest magnitude that counts for a block's scale (mx_encode).
template <int F>
__device__ __forceinline__ uint32_t largest16(const float (&v)[4][4]) {
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t b = __float_as_uint(v[i][j]) & 0x7fffffffu;
      largest = max(largest, F != MX_E2M1 && b >= 0x7f800000u ? 0u : b);
    }
  return largest;
}
// A block's scale byte.
template <int F>
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest) {
  return F == MX_E2M1 && largest >= 0x7f800000u ? 255u : mx_scale_of<F>(largest);
}

// A block of 32 codes; eight(i): its values 8 i .. 8 i + 7.
template <int F>
struct Codes {
  uint32_t w[F == MX_E2M1 ? 4 : 8];
  __device__ __forceinline__ void set(int half, const uintx4& v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[4 * half + i] = v[i];
  }
  __device__ __forceinline__ void load(const uint8_t* p) {
    set(0, *reinterpret_cast<const uintx4*>(p));
    if constexpr (F != MX_E2M1) set(1, *reinterpret_cast<const uintx4*>(p + 16));
  }
  __device__ __forceinline__ bf16x8 eight(int i, float scale) const {
    uintx4 r;
    if constexpr (F == MX_E2M1)
      r = uintx4{mx_values2<F, 0>(w[i], scale), mx_values2<F, 1>(w[i], scale), mx_values2<F, 2>(w[i], scale),
                 mx_values2<F, 3>(w[i], scale)};
    else
      r = uintx4{mx_values2<F, 0>(w[2 * i], scale), mx_values2<F, 1>(w[2 * i], scale),
                 mx_values2<F, 0>(w[2 * i + 1], scale), mx_values2<F, 1>(w[2 * i + 1], scale)};
    return __builtin_bit_cast(bf16x8, r);
  }
};

struct LinearParams {
  const float* X;
  const uint8_t* x_codes;  // X encoded (null: encoded by the kernel)
  const uint8_t* x_scales;
  const uint8_t* codes;
  const uint8_t* scales;
  const float* bias;
  float* Y;
  int64_t ldx, ldy, K;
  int M, N, G, act;
};

// ---- few rows: the waves of a workgroup share the groups of 128 ----
// A workgroup gives 16 columns n of 16 MB rows m; its waves take every W-th group, and their sums
// are added in wave order. Lane l holds block l / 16 of row l mod 16's group, whose values 8 i ..
// 8 i + 7 go to the i-th of four v_mfma_f32_16x16x32_bf16: which 32 of the group's values an
// instruction contracts does not matter as long as both operands agree. Weights are not staged:
// each is used once. One token by e2m1 weights [4096, 4096] takes 5.8 us (9 MB, 1.5 TB/s): a round of
// loads and its latency, the encoding and the sums.
//
// INLINE: every workgroup encodes its rows of X itself, four values a thread and round, into LDS as
// bfloat16 [rows][128 G] (16-byte pieces of a group in another order for each row, so that rows are
// read from different banks), while its first weights arrive; otherwise X comes encoded.
template <int FX>
__device__ __forceinline__ void encode_rows(const LinearParams& p, char* lds, int row0, int rows) {
  const int q = threadIdx.x & 31, total = rows * p.G;
  for (int t = threadIdx.x >> 5; t < total; t += blockDim.x >> 5) {
    const int m = t / p.G, k = (t - m * p.G) * MX_GROUP + 4 * q;
    const float* x = p.X + (row0 + m) * p.ldx + k;
    float v[4];
    if (k + 4 <= p.K) {
      const float4u f = *reinterpret_cast<const float4u*>(x);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = f[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = k + i < p.K ? x[i] : 0.0f;
    }
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
      largest = max(largest, FX != MX_E2M1 && b >= 0x7f800000u ? 0u : b);
    }
    const uint32_t s = scale_byte<FX>(mx_block_largest(largest));
    // (a lost block's reciprocal is of no account: its scale makes it NaN)
    const uint32_t c = mx_codes4<FX, false>(v, mx_reciprocal(min(s, 254u)));
    const uint2 out = {mx_values2<FX, 0>(c, mx_scale_operand(s)), mx_values2<FX, 1>(c, mx_scale_operand(s))};
    reinterpret_cast<uint2*>(lds)[t * 32 + (q ^ (2 * m))] = out;
  }
}

template <int FX, int FW, int MB, bool INLINE>
__global__ void __launch_bounds__(1024) mx_linear_rows(LinearParams p) {
  constexpr int BW = mx_group_bytes(FW), BX = mx_group_bytes(FX);
  static_assert(!INLINE || MB == 1, "rows of one fragment");
  extern __shared__ __align__(16) char lds[];  // sums [waves][MB][64][4], then INLINE's rows
  const int lane = threadIdx.x & 63, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  float* sums = reinterpret_cast<float*>(lds);
  char* x_rows = lds + waves * MB * 1024;
  const int row0 = blockIdx.y * (16 * MB), rows = min(16 * MB, p.M - row0);
  const int64_t n = min((int)blockIdx.x * 16 + (lane & 15), p.N - 1);
  const uint8_t* w_codes = p.codes + n * p.G * BW + q * (BW / 4);
  const uint8_t* w_scales = p.scales + n * p.G * 4 + q;
  int64_t m[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) m[i] = min((int)blockIdx.y * (16 * MB) + 16 * i + (lane & 15), p.M - 1);
  floatx4 acc[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  bool encoded = false;
  for (int t = wave; INLINE ? !encoded || t < p.G : t < p.G; t += waves) {
    Codes<FW> w;
    uint32_t xs[MB];
    Codes<FX> x[MB];
    const int64_t g = min(t, p.G - 1);
    w.load(w_codes + g * BW);
    const uint32_t ws = w_scales[g * 4];
    if constexpr (!INLINE) {
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        x[i].load(p.x_codes + (m[i] * p.G + g) * BX + q * (BX / 4));
        xs[i] = p.x_scales[(m[i] * p.G + g) * 4 + q];
      }
    }
    if (INLINE && !encoded) {  // (once, every wave)
      encode_rows<FX>(p, x_rows, row0, rows);
      __syncthreads();
      encoded = true;
    }
    if (t >= p.G) break;
    const float wf = mx_scale_operand(ws);
    bf16x8 a[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = w.eight(i, wf);
    if constexpr (INLINE) {
      const int r = min(lane & 15, rows - 1);
      const bf16x8* b = reinterpret_cast<const bf16x8*>(x_rows) + (r * p.G + t) * 16;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j], b[(4 * q + j) ^ r], acc[0], 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const float xf = mx_scale_operand(xs[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j], x[i].eight(j, xf), acc[i], 0, 0, 0);
      }
    }
  }
  // register r of a lane: column n = 4 (lane / 16) + r, row m = lane mod 16 (its four columns' banks
  // apart from those of the other columns of the rows that are read together)
  auto at = [](int quad, int row) { return (quad * 16 + (row ^ (4 * quad))) * 4; };
#pragma unroll
  for (int i = 0; i < MB; ++i)
    *reinterpret_cast<floatx4*>(sums + (wave * MB + i) * 256 + at(q, lane & 15)) = acc[i];
  __syncthreads();
  for (int e = threadIdx.x; e < MB * 256; e += blockDim.x) {
    const int c = e & 15, r = (e >> 4) & 15, from = (e >> 8) * 256 + at(c >> 2, r) + (c & 3);
    float v = sums[from];
    for (int k = 1; k < waves; ++k) v += sums[k * MB * 256 + from];
    const int row = blockIdx.y * (16 * MB) + (e >> 8) * 16 + r, col = blockIdx.x * 16 + c;
    if (row >= p.M || col >= p.N) continue;
    if (p.bias != nullptr) v += p.bias[col];
    p.Y[row * p.ldy + col] = apply_act(p.act, v);
  }
}

// ---- many rows: tiles of codes in LDS ----
// BM x BN results a workgroup, WM x WN waves, one group of 128 a stage, NS stages. Codes are copied
// by global_load_lds_dwordx4, 1 KB of whole rows' groups a copy, so that memory is read in
// contiguous groups. Lane l of a wave takes block 2 h + l / 32 of row l mod 32 for half h of the
// group:
//   * e2m1 on both sides goes to v_mfma_scale_f32_32x32x64_f8f6f4 as it is, with the blocks' scales;
//     sums are exact within a block and binary32 across;
//   * otherwise the codes become bfloat16 on the way from LDS to v_mfma_f32_32x32x16_bf16 (four
//     conversions, which also scale, for eight values of a lane), values 8 i .. 8 i + 7 of each
//     lane's block for the i-th of four. As bfloat16 in LDS the operands would take more of its
//     width than it has.
// The 16-byte chunks of a row are permuted by the row's ordinal so that the 16 lanes that read
// together meet every bank once. Scales come as [group][row] words of four from the launch that
// encodes X. 8192x4096x4096 of e4m3 by e2m1 takes 217 us under steady load, 1.27 PFLOP/s, and 233 in the first
// passes after a pause: the matrix cores are busy 55% of the cycles then, at 2.04 GHz, the vector ALUs'
// conversions (four an instruction of theirs) most of the others. With 8 bits on both sides it takes 230
// us, with 4 bits 106, 2.6 PFLOP/s, a quarter of it the results' store.
template <int F>
struct TileRows {
  static constexpr int BYTES = mx_group_bytes(F), CHUNKS = BYTES / 16, PER_COPY = 64 / CHUNKS;
  // chunk c of row r lies at place c ^ turn(r)
  static __device__ __forceinline__ int turn(int r) {
    return F == MX_E2M1 ? (r >> 2) & 3 : (r >> 1) & 7;
  }
};

struct TileParams {
  LinearParams l;
  const uint32_t* xt;  // scales [G][MP], [G][NP]
  const uint32_t* wt;
  float* partial;      // the slices' sums [slices][M][N] of a product split along K, or null
  int MP, NP, tiles_m, tiles_n, chunk;  // chunk: groups of a slice
};

// Stores act(acc + bias) of a wave's TM x TN blocks whose first row and column are row0 and col0
// (register r of a block: row 8 (r / 4) + 4 (lane / 32) + r mod 4, column lane mod 32). Each band of
// 32 rows goes through `mine`, LDS of this wave alone, so that rows are stored whole and the
// activation, evaluated in binary64, is compiled once a band and not for every register.
template <int TM, int TN>
__device__ __forceinline__ void mx_store_bands(const floatx16 (&acc)[TM][TN], float* mine, float* Y,
                                               int64_t ldy, const float* bias, int act, int row0,
                                               int col0, int M, int N) {
  constexpr int WIDTH = 32 * TN, QUADS = WIDTH / 4;
  const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) mine[(8 * (r >> 2) + 4 * half + (r & 3)) * WIDTH + 32 * j + l32] = acc[i][j][r];
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    for (int e = lane; e < 32 * QUADS; e += 64) {
      const int row = row0 + 32 * i + e / QUADS, col = col0 + e % QUADS * 4;
      floatx4 v = *reinterpret_cast<const floatx4*>(mine + e * 4);
      if (row >= M || col >= N) continue;
      float* y = Y + row * ldy + col;
      const int rest = N - col;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (bias != nullptr && r < rest) v[r] += bias[col + r];
        if (act != ACT_NONE) v[r] = apply_act(act, v[r]);
      }
      if (rest >= 4) {
        *reinterpret_cast<float4u*>(y) = float4u{v[0], v[1], v[2], v[3]};
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (r < rest) y[r] = v[r];
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
  }
}

template <int FX, int FW, int BM, int BN, int WM, int WN, int NS>
__global__ void __launch_bounds__(64 * WM * WN) mx_linear_tile(TileParams t) {
  const LinearParams& p = t.l;
  using RX = TileRows<FX>;
  using RW = TileRows<FW>;
  constexpr bool SCALED = FX == MX_E2M1 && FW == MX_E2M1;
  constexpr int WAVES = WM * WN, TM = BM / 32 / WM, TN = BN / 32 / WN;
  constexpr int CX = BM / RX::PER_COPY, CW = BN / RW::PER_COPY, CODES = (CX + CW) / WAVES;
  static_assert((CX + CW) % WAVES == 0, "whole copies a wave");
  static_assert((BM + BN) / 64 == WAVES, "one copy of 64 rows' scales a wave");
  constexpr int COPIES = CODES + 1;
  constexpr int W_AT = BM * RX::BYTES, S_AT = W_AT + BN * RW::BYTES, STAGE = S_AT + 4 * (BM + BN);
  static_assert(NS >= 2 && NS * STAGE <= 160 * 1024, "LDS");
  static_assert(WAVES * 32 * TN * 32 * 4 <= NS * STAGE, "the epilogue's rows");
  __shared__ __align__(16) uint8_t lds[NS * STAGE];
  const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;
  mx_tile_of(blockIdx.x, t.tiles_m, t.tiles_n, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int g0 = blockIdx.y * t.chunk, groups = min(t.chunk, p.G - g0);

  // this wave's copies: per-lane offsets of the CODES pieces (rows clamped to the operand's last)
  uint32_t voff[CODES];
  const uint8_t* base[CODES];
#pragma unroll
  for (int i = 0; i < CODES; ++i) {
    const int c = wave * CODES + i;
    if (c < CX) {
      const int r = c * RX::PER_COPY + lane / RX::CHUNKS, place = lane % RX::CHUNKS;
      voff[i] = (uint32_t)min(r, p.M - 1 - m0) * (uint32_t)(p.G * RX::BYTES) + (place ^ RX::turn(r)) * 16;
      base[i] = p.x_codes + ((int64_t)m0 * p.G + g0) * RX::BYTES;
    } else {
      const int r = (c - CX) * RW::PER_COPY + lane / RW::CHUNKS, place = lane % RW::CHUNKS;
      voff[i] = (uint32_t)min(r, p.N - 1 - n0) * (uint32_t)(p.G * RW::BYTES) + (place ^ RW::turn(r)) * 16;
      base[i] = p.codes + ((int64_t)n0 * p.G + g0) * RW::BYTES;
    }
  }
  const bool of_x = wave < BM / 64;
  const int64_t sstep = of_x ? t.MP : t.NP;
  const uint32_t* sbase = (of_x ? t.xt + m0 + 64 * wave : t.wt + n0 + 64 * (wave - BM / 64)) + g0 * sstep;
  const uint32_t soff = lane * 4;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  int copied = 0;
  auto copy_next = [&](int stage) {
    const uint32_t at = lds0 + stage * STAGE;
#pragma unroll
    for (int i = 0; i < CODES; ++i)
      asm volatile("global_load_lds_dwordx4 %0, %1"
                   : : "v"(voff[i]), "s"(base[i]), "{m0}"(at + (wave * CODES + i) * 1024) : "memory");
    asm volatile("global_load_lds_dword %0, %1"
                 : : "v"(soff), "s"(sbase), "{m0}"(at + S_AT + wave * 256) : "memory");
    if (++copied < groups) {  // (the last group again behind the end, to keep the count in flight)
#pragma unroll
      for (int i = 0; i < CODES; ++i) base[i] += wave * CODES + i < CX ? RX::BYTES : RW::BYTES;
      sbase += sstep;
    }
  };

  floatx16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  const int wm = wave / WN, wn = wave % WN;
  struct Frags {
    Codes<FX> x[TM];
    Codes<FW> w[TN];
  };
  // the lane's block of half h of the group of each row
  auto block = [&](auto& c, auto fc, const uint8_t* rows, int r, int h) {
    constexpr int F = decltype(fc)::value;
    const uint8_t* row = rows + r * TileRows<F>::BYTES;
    const int turn = TileRows<F>::turn(r), b = 2 * h + half;
    if constexpr (F == MX_E2M1) {
      c.set(0, *reinterpret_cast<const uintx4*>(row + ((b ^ turn) << 4)));
    } else {
      c.set(0, *reinterpret_cast<const uintx4*>(row + (((2 * b) ^ turn) << 4)));
      c.set(1, *reinterpret_cast<const uintx4*>(row + (((2 * b + 1) ^ turn) << 4)));
    }
  };
  constexpr std::integral_constant<int, FX> fx;
  constexpr std::integral_constant<int, FW> fw;
  auto read = [&](int stage, int h, Frags& f) {
    const uint8_t* at = lds + stage * STAGE;
#pragma unroll
    for (int j = 0; j < TN; ++j) block(f.w[j], fw, at + W_AT, (wn * TN + j) * 32 + l32, h);
#pragma unroll
    for (int i = 0; i < TM; ++i) block(f.x[i], fx, at, (wm * TM + i) * 32 + l32, h);
  };
  // the four scales of a row's group, the two that this lane needs in bytes 0 and 2
  struct Scales {
    uint32_t x[TM], w[TN];
  };
  auto read_scales = [&](int stage, Scales& s) {
    const uint32_t* at = reinterpret_cast<const uint32_t*>(lds + stage * STAGE + S_AT);
#pragma unroll
    for (int i = 0; i < TM; ++i) s.x[i] = at[(wm * TM + i) * 32 + l32] >> (8 * half);
#pragma unroll
    for (int j = 0; j < TN; ++j) s.w[j] = at[BM + (wn * TN + j) * 32 + l32] >> (8 * half);
  };
  auto multiply = [&](auto hc, const Frags& f, const Scales& s) {
    constexpr int H = decltype(hc)::value;
    if constexpr (SCALED) {
      auto wide = [](const auto& c) {
        return intx8{(int)c.w[0], (int)c.w[1], (int)c.w[2], (int)c.w[3], 0, 0, 0, 0};
      };
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
              wide(f.x[i]), wide(f.w[j]), acc[i][j], 4, 4, 2 * H, (int)s.x[i], 2 * H, (int)s.w[j]);
    } else {
      float sx[TM], sw[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) sx[i] = mx_scale_operand((s.x[i] >> (16 * H)) & 0xffu);
#pragma unroll
      for (int j = 0; j < TN; ++j) sw[j] = mx_scale_operand((s.w[j] >> (16 * H)) & 0xffu);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        bf16x8 a[TM], b[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) a[i] = f.x[i].eight(e, sx[i]);
#pragma unroll
        for (int j = 0; j < TN; ++j) b[j] = f.w[j].eight(e, sw[j]);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
      }
    }
  };
  // Waits until this wave's reads have returned and its copies into the next stage have landed,
  // for all waves; then refills the stage just read.
  auto advance = [&](int stage) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"((NS - 2) * COPIES) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    copy_next(stage);
  };
#pragma unroll
  for (int s = 0; s < NS - 1; ++s) copy_next(s);
  constexpr std::integral_constant<int, 0> h0;
  constexpr std::integral_constant<int, 1> h1;
  int stage = 0;
  Frags a, b;
  Scales s;
  advance(NS - 1);
  read_scales(0, s);
  read(0, 0, a);
  for (int g = 0; g < groups; ++g) {
    read(stage, 1, b);
    multiply(h0, a, s);
    const Scales now = s;
    advance(stage);
    stage = stage == NS - 1 ? 0 : stage + 1;
    read_scales(stage, s);
    read(stage, 0, a);
    multiply(h1, b, now);
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
  __builtin_amdgcn_s_barrier();  // no copy is in flight and no wave reads: LDS is free
  asm volatile("" : : : "memory");
  const bool whole = t.partial == nullptr;
  mx_store_bands<TM, TN>(acc, reinterpret_cast<float*>(lds) + wave * 32 * TN * 32,
                         whole ? p.Y : t.partial + (int64_t)blockIdx.y * p.M * p.N, whole ? p.ldy : p.N,
                         whole ? p.bias : nullptr, whole ? p.act : (int)ACT_NONE, m0 + wm * TM * 32,
                         n0 + wn * TN * 32, p.M, p.N);
}

// One launch: workgroup (group, y) encodes the group of 32 rows of X, eight lanes a row, scales as
// the tiles take them; the workgroups behind turn W's scales [N][G] likewise.
struct PrepareParams {
  LinearParams l;
  uint8_t* codes;
  uint32_t* xt;
  uint32_t* wt;
  int MP, NP, x_blocks;
};
template <int FX>
__global__ void __launch_bounds__(256) mx_prepare(PrepareParams p) {
  const int g = blockIdx.x;
  if ((int)blockIdx.y < p.x_blocks) {
    const int part = threadIdx.x & 7;
    const int64_t m = (int64_t)blockIdx.y * 32 + (threadIdx.x >> 3), k = (int64_t)g * MX_GROUP + 16 * part;
    if (m >= p.l.M) return;
    float v[4][4];
    load16(p.l.X + m * p.l.ldx + k, p.l.K - k, v);
    uint32_t largest = largest16<FX>(v);
    largest = max(largest, (uint32_t)__builtin_amdgcn_mov_dpp((int)largest, 0xB1, 0xf, 0xf, false));
    const uint32_t s = scale_byte<FX>(largest);
    const float r = mx_reciprocal(min(s, 254u));
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = mx_codes4<FX, false>(v[i], r);
    uint8_t* out = p.codes + (m * p.l.G + g) * mx_group_bytes(FX) + part * (mx_group_bytes(FX) / 8);
    if constexpr (FX == MX_E2M1)
      *reinterpret_cast<uint2*>(out) = uint2{c[0] | (c[1] << 16), c[2] | (c[3] << 16)};
    else
      *reinterpret_cast<uintx4*>(out) = uintx4{c[0], c[1], c[2], c[3]};
    uint32_t word = s << (8 * (part >> 1));  // (the lanes of a block agree)
    word |= (uint32_t)__shfl_xor((int)word, 2, 64);
    word |= (uint32_t)__shfl_xor((int)word, 4, 64);
    if (part == 0) p.xt[(int64_t)g * p.MP + m] = word;
  } else {
    const int64_t n = (int64_t)(blockIdx.y - p.x_blocks) * 256 + threadIdx.x;
    if (n < p.l.N) p.wt[(int64_t)g * p.NP + n] = reinterpret_cast<const uint32_t*>(p.l.scales)[n * p.l.G + g];
  }
}

// act(bias + the sum over the slices, in slice order).
__global__ void __launch_bounds__(256) mx_linear_sum(const float* __restrict__ partial, int64_t plane,
                                                     int slices, LinearParams p) {
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < plane; e += (int64_t)gridDim.x * 256) {
    float v = partial[e];
    for (int s = 1; s < slices; ++s) v += partial[s * plane + e];
    const int64_t row = e / p.N, col = e - row * p.N;
    if (p.bias != nullptr) v += p.bias[col];
    p.Y[row * p.ldy + col] = apply_act(p.act, v);
  }
}

enum Route { ROWS_INLINE, ROWS, TILES };
struct Plan {
  Route route;
  int mb, waves;      // few rows: row fragments and waves of a workgroup
  int large;          // rows of tiles of 256, ahead of those of 128
  int slices, chunk;  // groups of a slice
};
// Which form runs (us on MI355X, e4m3 activations and e2m1 weights, a synchronous run's 13 us
// included, both sides in turn in short runs; under steady load large layers take up to a tenth less):
//   * few rows: INLINE up to 128 groups of X a workgroup, with a wave for every four of them
//     (1x4096x4096 16.6; encoded by a launch of its own 19.6), and for more than 16 rows only while
//     the groups that all workgroups encode stay few (20x1000x500 15.8 against 18.3, 128x1024x128 14.7
//     against 17.9, 362x784x44 17.2 against 17.5; but 2400x512x64 24.8 against 20.5);
//   * ROWS up to 2^30 multiply-adds (500x1021x617 21.8 against 27.2, 300x1024x1024 23.7 against
//     29.2; 1024^3 33.7 against 30.5), 2^31 of up to 64 rows (64x4096x4096 30.9 against 34.6;
//     64x8192x8192 70 against 46), and always up to 16;
//   * tiles of 256, of 128, or the rows of as many rounds of 256 CUs as tiles of 256 fill and then the
//     others on tiles of 128, whichever takes the fewest rounds; a tile of 256 takes 3.6 times one of
//     128, 2.6 times with 4 bits on both sides (8192x4096x4096 290 on 256, 320 on 128; 4096x5120x2048,
//     320 tiles, 122, 102 and mixed 101; 4100x4100x4000 203, 161 and 160, of 4-bit codes 99, 93 and 87;
//     4000x2900x2048, 192 tiles, 74 against 71, of 4-bit codes 46.5 against 50.5);
//   * K split between workgroups when there are fewer than 256 tiles of 128 and 16 groups and more
//     (128x4096x4096 38 in eight, 51 whole; 300x4096x4096 47 in four, 54 whole; but 1024^3, eight
//     groups, 34 in two and 30.5 whole).
constexpr int64_t INLINE_GROUPS = 128, INLINE_WORK = 600000;
Plan plan(int64_t M, int64_t N, int64_t K, bool four) {
  const int64_t G = mx_groups(K);
  Plan w{TILES, 0, 0, 0, 1, (int)G};
  const double work = (double)M * (double)N * (double)K;
  // (tiles address a row within 32 bits)
  if (M <= 16 || work < (M <= 64 ? 2.0 : 1.0) * (1 << 30) || K > (1 << 22)) {
    w.waves = (int)std::min<int64_t>(16, G);
    // as many row fragments as leave three quarters of the CUs a workgroup (48x4096x4096 28.6 us
    // with four, 30.2 with two, 31.4 with one; 128x1024x2048 24.3, 21.5, 22.5; 64x1024x4096 30.6,
    // 25.1, 22.2) and eight waves a CU (362x784x44, one wave each, 20.0 with four, 18.3 with one)
    auto enough = [&](int mb) {
      const int64_t n = ((N + 15) / 16) * ((M + 16 * mb - 1) / (16 * mb));
      return M > 8 * mb && n >= 192 && n * w.waves >= 2048;
    };
    w.mb = enough(4) ? 4 : enough(2) ? 2 : 1;
    const int64_t rows = std::min<int64_t>(M, 16 * w.mb);
    // (with two row fragments and more there is too much to encode)
    const bool in_line = w.mb == 1 && rows * G <= INLINE_GROUPS && (M <= 16 || M * G * N <= INLINE_WORK);
    w.route = in_line ? ROWS_INLINE : ROWS;
    if (in_line) w.waves = (int)std::max<int64_t>(w.waves, std::min<int64_t>(16, rows * G / 4));
  } else if (mx_tiles(M, N, 128) < 256 && G >= 16) {
    const int64_t s = std::max<int64_t>(1, std::min(384 / mx_tiles(M, N, 128), G / 4));
    w.chunk = (int)((G + s - 1) / s);
    w.slices = (int)((G + w.chunk - 1) / w.chunk);
  } else {
    w.large = mx_large_rows(M, N, four ? 2.6 : 3.6);
  }
  return w;
}

template <int FX, int FW>
hipError_t launch(const LinearParams& p, const Plan& w, char* scratch, hipStream_t s) {
  const int G = p.G;
  const Route r = w.route;
  if (r == ROWS_INLINE || r == ROWS) {
    auto go = [&](auto mb, auto in_line) {
      constexpr int MB = decltype(mb)::value;
      constexpr bool INLINE = decltype(in_line)::value;
      hipLaunchKernelGGL((mx_linear_rows<FX, FW, MB, INLINE>),
                         dim3((p.N + 15) / 16, (p.M + 16 * MB - 1) / (16 * MB)), dim3(64 * w.waves),
                         w.waves * MB * 1024 + (INLINE ? (size_t)std::min(p.M, 16 * MB) * G * 256 : 0), s, p);
    };
    if (r == ROWS_INLINE) go(std::integral_constant<int, 1>(), std::true_type());
    else if (w.mb == 4) go(std::integral_constant<int, 4>(), std::false_type());
    else if (w.mb == 2) go(std::integral_constant<int, 2>(), std::false_type());
    else go(std::integral_constant<int, 1>(), std::false_type());
    return hipGetLastError();
  }
  PrepareParams k{};
  k.l = p;
  k.MP = (p.M + 255) / 256 * 256;
  k.NP = (p.N + 255) / 256 * 256;
  k.xt = reinterpret_cast<uint32_t*>(scratch);
  k.wt = k.xt + (int64_t)G * k.MP;
  k.codes = reinterpret_cast<uint8_t*>(k.wt + (int64_t)G * k.NP);
  k.x_blocks = (p.M + 31) / 32;
  hipLaunchKernelGGL(mx_prepare<FX>, dim3(G, k.x_blocks + (p.N + 255) / 256), dim3(256), 0, s, k);
  TileParams t{};
  t.l = p;
  t.l.x_codes = k.codes;
  t.xt = k.xt; t.wt = k.wt; t.MP = k.MP; t.NP = k.NP;
  t.chunk = w.chunk;
  if (w.slices > 1)
    t.partial = reinterpret_cast<float*>(k.codes + (int64_t)p.M * G * mx_group_bytes(FX));
  constexpr int bytes = mx_group_bytes(FX) + mx_group_bytes(FW);
  constexpr int NS = bytes == 256 ? 2 : bytes == 192 ? 3 : 4;
  auto go = [&](auto tile, int row0, int rows) {
    constexpr int T = decltype(tile)::value, WM = T == 256 ? 4 : 2;
    if (rows <= 0) return;
    TileParams q = t;
    q.l.M = rows;
    q.l.x_codes += (int64_t)row0 * G * mx_group_bytes(FX);
    q.l.Y += row0 * p.ldy;
    q.xt += row0;
    q.tiles_m = (rows + T - 1) / T;
    q.tiles_n = (p.N + T - 1) / T;
    hipLaunchKernelGGL((mx_linear_tile<FX, FW, T, T, WM, 2, NS>),
                       dim3((unsigned)(q.tiles_m * q.tiles_n), (unsigned)w.slices), dim3(128 * WM), 0, s, q);
  };
  const int large = std::min(p.M, 256 * w.large);
  go(std::integral_constant<int, 256>(), 0, large);
  go(std::integral_constant<int, 128>(), large, p.M - large);
  if (w.slices > 1) {
    const int64_t plane = (int64_t)p.M * p.N;
    hipLaunchKernelGGL(mx_linear_sum, dim3((unsigned)std::min<int64_t>(8192, (plane + 255) / 256)), dim3(256),
                       0, s, t.partial, plane, w.slices, p);
  }
  return hipGetLastError();
}

}  // namespace

namespace {
// Rows of X and of W that one set of launches takes (grid dimensions).
constexpr int64_t MAX_ROWS = 1 << 20;

int64_t piece_scratch_bytes(int64_t M, int64_t N, int64_t K) {
  const Plan w = plan(M, N, K, false);  // (the tiles' sizes take no scratch)
  if (w.route == ROWS_INLINE) return 0;
  const int64_t G = mx_groups(K);
  if (w.route == ROWS) return pad256(M * G * 128) + M * G * 4;
  return 4 * G * ((M + 255) / 256 * 256 + (N + 255) / 256 * 256) + M * G * 128 +
         (w.slices > 1 ? 4 * w.slices * M * N : 0);
}

hipError_t launch_piece(const MxLinearParams& in, void* scratch, hipStream_t s) {
  const int64_t G = mx_groups(in.K);
  const Plan w = plan(in.M, in.N, in.K, in.x_format == MX_E2M1 && in.w_format == MX_E2M1);
  LinearParams p{};
  p.X = in.X; p.codes = in.codes; p.scales = in.scales; p.bias = in.bias; p.Y = in.Y;
  p.ldx = in.ldx; p.ldy = in.ldy; p.K = in.K;
  p.M = (int)in.M; p.N = (int)in.N; p.G = (int)G; p.act = in.act;
  if (w.route == ROWS) {
    uint8_t* codes = static_cast<uint8_t*>(scratch);
    uint8_t* scales = codes + pad256(in.M * G * 128);
    const hipError_t e = launch_mx_encode(in.X, in.ldx, codes, scales, in.M, in.K, in.x_format, 0, s);
    if (e != hipSuccess) return e;
    p.x_codes = codes;
    p.x_scales = scales;
  }
  hipError_t e = hipSuccess;
  mx_with_format(in.x_format, [&](auto x) {
    mx_with_format(in.w_format, [&](auto f) {
      e = launch<decltype(x)::value, decltype(f)::value>(p, w, static_cast<char*>(scratch), s);
    });
  });
  return e;
}
}  // namespace

int64_t mx_linear_scratch_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0) return 0;
  if (K == 0) return 4 * gemm_workspace_floats(M, N, K);
  int64_t bytes = 0;  // whole pieces and the last ones
  for (int64_t m : {std::min(M, MAX_ROWS), M % MAX_ROWS})
    for (int64_t n : {std::min(N, MAX_ROWS), N % MAX_ROWS})
      if (m > 0 && n > 0) bytes = std::max(bytes, piece_scratch_bytes(m, n, K));
  return bytes;
}

hipError_t launch_mx_linear(const MxLinearParams& in, void* scratch, hipStream_t s) {
  if (in.M <= 0 || in.N <= 0) return hipSuccess;
  if (in.K == 0) {  // no products: act(bias)
    GemmParams g{};
    g.A = g.B = in.X;
    g.C = in.Y;
    g.bias = in.bias;
    g.M = in.M; g.N = in.N;
    g.ldc = in.ldy;
    g.transB = 1;
    g.act = in.act;
    return launch_gemm(g, static_cast<float*>(scratch), s);
  }
  const int64_t G = mx_groups(in.K);
  for (int64_t m = 0; m < in.M; m += MAX_ROWS)
    for (int64_t n = 0; n < in.N; n += MAX_ROWS) {
      MxLinearParams p = in;
      p.M = std::min(MAX_ROWS, in.M - m);
      p.N = std::min(MAX_ROWS, in.N - n);
      p.X += m * in.ldx;
      p.codes += n * G * mx_group_bytes(in.w_format);
      p.scales += n * G * 4;
      if (p.bias != nullptr) p.bias += n;
      p.Y += m * in.ldy + n;
      const hipError_t e = launch_piece(p, scratch, s);
      if (e != hipSuccess) return e;
    }
  return hipSuccess;
}

}  // namespace shk
