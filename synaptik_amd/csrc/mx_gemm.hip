// C = op(A) . B of a binary32 A and a microscaled B [K, N] (mx.h; blocks along N): the weight
// gradient dW = dZ^T . X from X's 8-bit checkpoint, and the input gradient dX = dZ . W through
// microscaled weights.
//
// A code has at most four significant bits and its scale is a power of two, so B's values are exact
// in bfloat16. A binary32 value is the exact sum of three bfloat16 values: its leading eight
// significant bits, the next eight and the last eight. The product of A and B is therefore the sum
// of three bfloat16 products whose terms are exact, accumulated in binary32: what a binary32
// product gives (each term rounded no more often), at a third of the bfloat16 matrix cores' rate
// instead of the binary32 ones', 5.3 times as fast (2.5 / 3 against 0.157 PFLOP/s).
// The matrix cores read subnormal bfloat16 values as zeros, so a value of A counts with an error
// below 2^-126, the smallest normal binary32 value: the first part that is read as zero is below
// it, and so is all that the part leads. A value of B below 2^-126 counts with such an error too;
// those that encoding gives are zero or normal (its scales start at 2^-110). An infinite code of B
// gives NaN, since it meets parts of A that are zero.
#include <algorithm>

#include "launch_limits.h"
#include "mx_tiles.h"

namespace shk {
namespace {

// ---- operands as matrix-instruction fragments ----
// v_mfma_f32_32x32x16_bf16 takes from lane l the eight values k = 8 (l / 32) .. + 7 of row l mod 32.
// Both operands are laid out as the 1 KB fragments it takes, 16 bytes a lane: fragment (kt, block,
// plane) covers k = 16 kt .. + 15 of rows 32 block .. + 31, planes of a block adjacent and the
// blocks of one kt adjacent. Values behind K are zero; rows behind the operand's last are not
// written (they reach only results that are not stored).
constexpr int FRAG = 1024, PLANES = 3;

// (a >> 16) | (b & 0xffff0000): the bfloat16 values that two floats hold exactly.
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}
// Where the eight values k = 8 octet .. + 7 of row r lie in plane 0 of an operand of `blocks`
// blocks and `planes` planes.
__device__ __forceinline__ char* frag_at(char* base, int64_t octet, int64_t r, int64_t blocks, int planes) {
  return base + ((octet >> 1) * blocks + (r >> 5)) * planes * FRAG + (((octet & 1) << 5) + (r & 31)) * 16;
}

// The three parts of eight values. An infinity is its leading part alone; a NaN stays one though
// its low bits are cut off.
struct Planes {
  uintx4 hi, mid, lo;
};
__device__ __forceinline__ Planes split8(const float (&v)[8]) {
  uint32_t h[8], m[8], l[8], largest = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(v[i]);
    largest = max(largest, b & 0x7fffffffu);
    h[i] = b;  // (its high half is cut out below)
    const float r = v[i] - __uint_as_float(b & 0xffff0000u);
    m[i] = __float_as_uint(r);
    l[i] = __float_as_uint(r - __uint_as_float(m[i] & 0xffff0000u));
  }
  if (largest >= 0x7f800000u) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!is_finite(v[i])) {
        h[i] |= v[i] != v[i] ? 0x00400000u : 0u;
        m[i] = l[i] = 0;
      }
  }
  Planes p;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p.hi[i] = high_halves(h[2 * i], h[2 * i + 1]);
    p.mid[i] = high_halves(m[2 * i], m[2 * i + 1]);
    p.lo[i] = high_halves(l[2 * i], l[2 * i + 1]);
  }
  return p;
}
__device__ __forceinline__ void put_planes(char* at, const Planes& p) {
  *reinterpret_cast<uintx4*>(at) = p.hi;
  *reinterpret_cast<uintx4*>(at + FRAG) = p.mid;
  *reinterpret_cast<uintx4*>(at + 2 * FRAG) = p.lo;
}

// A stored [K, M]: a lane takes one row m and eight k (four waves, 32 k a workgroup), so that each
// load of a wave is 256 contiguous bytes.
__device__ __forceinline__ void pack_a_t(const float* __restrict__ a, int64_t lda, char* __restrict__ pa,
                                         int64_t M, int64_t K, int64_t MT, int64_t bk, int64_t bm) {
  const int64_t m = bm * 64 + (threadIdx.x & 63);
  const int64_t octet = bk * 4 + (threadIdx.x >> 6), k = 8 * octet;
  if (m >= M || (octet >> 1) >= (K + 15) / 16) return;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = k + i < K ? a[(k + i) * lda + m] : 0.0f;
  put_planes(frag_at(pa, octet, m, MT, PLANES), split8(v));
}

// A stored [M, K]: a wave takes sixteen rows and four octets, 128 contiguous bytes a row.
__device__ __forceinline__ void pack_a_n(const float* __restrict__ a, int64_t lda, char* __restrict__ pa,
                                         int64_t M, int64_t K, int64_t MT, int64_t bk, int64_t bm) {
  const int lane = threadIdx.x & 63;
  const int64_t m = bm * 64 + (threadIdx.x >> 6) * 16 + (lane & 15);
  const int64_t octet = bk * 4 + (lane >> 4), k = 8 * octet;
  if (m >= M || (octet >> 1) >= (K + 15) / 16) return;
  const float* src = a + m * lda + k;
  float v[8];
  if (k + 8 <= K) {
    const float4u x = *reinterpret_cast<const float4u*>(src), y = *reinterpret_cast<const float4u*>(src + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = x[i]; v[4 + i] = y[i]; }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? src[i] : 0.0f;
  }
  put_planes(frag_at(pa, octet, m, MT, PLANES), split8(v));
}

// Four columns' codes of eight k (a word of four a k, and the scale) as the eight values of each
// column.
template <int F>
__device__ __forceinline__ void fragments_of4(const uint32_t (&w)[8], const uint32_t (&scale)[8],
                                              bf16x8 (&out)[4]) {
  uint32_t lo[8], hi[8];  // columns 0, 1 and 2, 3
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo[i] = mx_values2<F, 0>(w[i], mx_scale_operand(scale[i]));
    hi[i] = mx_values2<F, 1>(w[i], mx_scale_operand(scale[i]));
  }
  uintx4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[0][i] = __builtin_amdgcn_perm(lo[2 * i + 1], lo[2 * i], 0x05040100u);
    v[1][i] = __builtin_amdgcn_perm(lo[2 * i + 1], lo[2 * i], 0x07060302u);
    v[2][i] = __builtin_amdgcn_perm(hi[2 * i + 1], hi[2 * i], 0x05040100u);
    v[3][i] = __builtin_amdgcn_perm(hi[2 * i + 1], hi[2 * i], 0x07060302u);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) out[j] = __builtin_bit_cast(bf16x8, v[j]);
}

// B's codes [K, N] as bfloat16 fragments: a lane takes four columns 4 q .. 4 q + 3 of a block and
// eight k. Column 4 q + j is the fragment's row q + 8 j, so that eight lanes write 128 contiguous
// bytes; the epilogue puts the columns back.
template <int F>
__device__ __forceinline__ void pack_b(const uint8_t* __restrict__ codes,
                                       const uint8_t* __restrict__ scales, char* __restrict__ pb,
                                       int64_t N, int64_t K, int64_t G, int64_t NT, int64_t bk,
                                       int64_t bn) {
  const int64_t n = (bn * 64 + (threadIdx.x & 63)) * 4;
  const int64_t octet = bk * 4 + (threadIdx.x >> 6), k = 8 * octet;
  if (n >= N || (octet >> 1) >= (K + 15) / 16) return;
  uint32_t w[8], sc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = k + i < K ? k + i : K - 1;
    w[i] = mx_load4<F>(codes, row * G * 32 + n / 4);
    sc[i] = scales[row * G * 4 + n / 32];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k + i >= K) w[i] = 0, sc[i] = 127;
  bf16x8 out[4];
  fragments_of4<F>(w, sc, out);
  char* at = frag_at(pb, octet, n / 32 * 32 + (n & 31) / 4, NT, 1);
#pragma unroll
  for (int j = 0; j < 4; ++j) *reinterpret_cast<bf16x8*>(at + 8 * 16 * j) = out[j];
}

// Both operands in one launch: unit (bk, block) is 32 k of 64 rows of A, then of 256 columns of B, the
// blocks of one bk in a row: they read and write neighbouring memory (a transposed 4096^2 A and B 34.5
// us, 219 MB at 6.3 TB/s; a sixth more with the k of one block in a row). A workgroup takes one, or several
// where there are more than a launch has workgroups (launch_limits.h).
struct PackParams {
  const float* A;
  const uint8_t* codes;
  const uint8_t* scales;
  char* pa;
  char* pb;
  int64_t lda, M, N, K, G, MT, NT, units;
  int a_blocks, blocks;
};
template <int F, bool TA>
__global__ void __launch_bounds__(PACK_THREADS) mx_pack(PackParams p) {
  for (int64_t unit = blockIdx.x; unit < p.units; unit += gridDim.x) {
    const int64_t bk = unit / p.blocks, block = unit - bk * p.blocks;
    if (block < p.a_blocks) {
      if (TA) pack_a_t(p.A, p.lda, p.pa, p.M, p.K, p.MT, bk, block);
      else pack_a_n(p.A, p.lda, p.pa, p.M, p.K, p.MT, bk, block);
    } else {
      pack_b<F>(p.codes, p.scales, p.pb, p.N, p.K, p.G, p.NT, bk, block - p.a_blocks);
    }
  }
}

// ---- the product ----
struct WideParams {
  const char* pa;
  const char* pb;
  float* C;        // or the partial sums [slices][M][N] of a product split along K
  int64_t ldc, plane;
  int M, N, KT, MT, NT;         // MT, NT: blocks of the packed operands
  int blocks_m;                 // blocks of A from pa on
  int tiles_m, tiles_n, chunk;  // chunk: fragments along K of a slice
};

// BM x BN results a workgroup, WM x WN waves of (BM / WM) x (BN / WN), 16 k a stage, NS stages in
// LDS. The stages are filled by global_load_lds_dwordx4, which copies 16 bytes a lane without
// passing through registers; fragments lie in memory as in LDS, so every copy and every fragment
// read is linear. A stage is copied NS - 1 stages before it is read; before a stage is read, each
// wave has waited for its own copies into it, and has finished with the stage whose place the next
// copies take. A stage's fragments are read while the one before is multiplied. The matrix cores
// bound it: 4096^3 takes 244 us under steady load, the three products together 1.69 PFLOP/s (a large
// bfloat16 product of the library 1.34), and 266 in the first passes after a pause, when power leaves
// 1.92 GHz and the cores are busy 77% of the cycles. Two by four or four by two waves and three to five
// stages are within 3%; four larger waves are 8% slower.
template <int BM, int BN, int WM, int WN, int NS>
__global__ void __launch_bounds__(64 * WM * WN) mx_wide(WideParams p) {
  constexpr int WAVES = WM * WN, TM = BM / 32 / WM, TN = BN / 32 / WN;
  constexpr int CA = BM / 32 * PLANES, CB = BN / 32, COPIES = (CA + CB) / WAVES;
  static_assert((CA + CB) % WAVES == 0, "whole copies a wave");
  constexpr int STAGE = (CA + CB) * FRAG;
  static_assert(NS >= 2 && NS * STAGE <= 160 * 1024, "LDS");
  __shared__ __align__(16) char lds[NS * STAGE];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;
  mx_tile_of(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
  const int kt0 = blockIdx.y * p.chunk, stages = min(p.chunk, p.KT - kt0);

  // this wave's copies: fragment c of a stage, the operand's blocks clamped to its last
  const char* src[COPIES];
  int64_t step[COPIES];
#pragma unroll
  for (int i = 0; i < COPIES; ++i) {
    const int c = wave * COPIES + i;
    if (c < CA) {
      const int block = min(tm * (BM / 32) + c / PLANES, p.blocks_m - 1);
      src[i] = p.pa + (((int64_t)kt0 * p.MT + block) * PLANES + c % PLANES) * FRAG;
      step[i] = (int64_t)p.MT * PLANES * FRAG;
    } else {
      const int block = min(tn * (BN / 32) + c - CA, p.NT - 1);
      src[i] = p.pb + ((int64_t)kt0 * p.NT + block) * FRAG;
      step[i] = (int64_t)p.NT * FRAG;
    }
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const uint32_t voff = lane * 16;
  int copied = 0;
  auto copy_next = [&](int stage) {
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const uint32_t dst = lds0 + stage * STAGE + (wave * COPIES + i) * FRAG;
      asm volatile("global_load_lds_dwordx4 %0, %1" : : "v"(voff), "s"(src[i]), "{m0}"(dst) : "memory");
    }
    // (behind the last stage it is copied again, which keeps the count of copies in flight)
    if (++copied < stages) {
#pragma unroll
      for (int i = 0; i < COPIES; ++i) src[i] += step[i];
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
    bf16x8 a[TM][PLANES], b[TN];
  };
  auto read = [&](int stage, Frags& f) {
    const char* at = lds + stage * STAGE + lane * 16;
#pragma unroll
    for (int j = 0; j < TN; ++j) f.b[j] = *reinterpret_cast<const bf16x8*>(at + (CA + wn * TN + j) * FRAG);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int q = 0; q < PLANES; ++q)
        f.a[i][q] = *reinterpret_cast<const bf16x8*>(at + ((wm * TM + i) * PLANES + q) * FRAG);
  };
  auto multiply = [&](const Frags& f) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int q = PLANES - 1; q >= 0; --q)
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.a[i][q], f.b[j], acc[i][j], 0, 0, 0);
  };
  int stage = 0;
  // Waits until this wave's reads have returned and its copies into the stage after this one have
  // landed, for all waves; then refills the stage just read.
  auto advance = [&](int s) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"((NS - 2) * COPIES) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    copy_next(s);
    stage = s == NS - 1 ? 0 : s + 1;
  };
#pragma unroll
  for (int s = 0; s < NS - 1; ++s) copy_next(s);
  Frags even, odd;
  advance(NS - 1);
  read(0, even);
  int s = 0;
  for (; s + 2 <= stages; s += 2) {
    advance(stage);
    read(stage, odd);
    multiply(even);
    advance(stage);
    read(stage, even);
    multiply(odd);
  }
  if (s < stages) multiply(even);
  asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // no copy outlives the workgroup's LDS

  // register r of a block: row 8 (r / 4) + 4 (lane / 32) + r mod 4, B's row lane mod 32, which is
  // column 4 q + j for row q + 8 j (pack_b)
  float* c = p.C + blockIdx.y * p.plane;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int col = tn * BN + (wn * TN + j) * 32 + 4 * (lane & 7) + ((lane & 31) >> 3);
      const int row0 = tm * BM + (wm * TM + i) * 32 + 4 * (lane >> 5);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = row0 + 8 * (r >> 2) + (r & 3);
        if (row < p.M && col < p.N) c[row * p.ldc + col] = acc[i][j][r];
      }
    }
}

// The sum over the slices of a product split along K, in slice order.
__global__ void __launch_bounds__(256) mx_gemm_sum(const float* __restrict__ partial, int64_t plane,
                                                   int slices, float* __restrict__ C, int64_t ldc,
                                                   int64_t N) {
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < plane; e += (int64_t)gridDim.x * 256) {
    float v = partial[e];
    for (int s = 1; s < slices; ++s) v += partial[s * plane + e];
    const int64_t row = e / N;
    C[row * ldc + (e - row * N)] = v;
  }
}

// ---- small products: operands straight into registers ----
// A workgroup gives 16 MB rows and 64 columns; its waves take every W-th chunk of 32 k and their sums
// are added in wave order. v_mfma_f32_16x16x32_bf16 takes from lane l the eight values k = 8 (l / 16)
// .. + 7 of row or column l mod 16: the lane loads them of MB rows of A, splits them, and of four
// columns of B (4 (l mod 16) + j is column l mod 16 of product j), whose codes lie four to a word, a
// word for each k. The L1's requests bound it, so of the eight k's scales a lane loads one and takes
// the others from its neighbours, and of a transposed A the two fragments' rows are neighbours, eight
// bytes a k (1024^3 transposed 28.5 -> 25.0 us a run with both, 64x8192x8192 71 -> 66); addresses are
// one base a wave and 32-bit offsets. 1024^3 takes 12.2 us, 176 TFLOP/s of binary32 products.
template <bool TA>
__device__ __forceinline__ void load_a8(const float* __restrict__ a, int64_t lda, int64_t m, int64_t k,
                                        int64_t K, float (&v)[8]) {
  if constexpr (TA) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? a[(k + i) * lda + m] : 0.0f;
  } else if (k + 8 <= K) {
    const float* src = a + m * lda + k;
    const float4u x = *reinterpret_cast<const float4u*>(src), y = *reinterpret_cast<const float4u*>(src + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = x[i]; v[4 + i] = y[i]; }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? a[m * lda + k + i] : 0.0f;
  }
}

struct DirectParams {
  const float* A;
  const uint8_t* codes;
  const uint8_t* scales;
  float* C;  // or the partial sums [slices][M][N] of a product split along K
  int64_t lda, ldc, plane, K, G;
  int M, N, chunks, per_slice, row_tiles;
  int near;  // a chunk's values lie within 2^32 bytes of its first
};
// A buffer from p on, which the wave agrees on.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, -1, 0x00020000);
}
// The value of lane I of this lane's eight.
template <int I>
__device__ __forceinline__ uint32_t of_eight(int v) {
  return (uint32_t)__builtin_amdgcn_ds_swizzle(v, (I << 5) | 0x18);
}
template <int F, bool TA, int MB>
__global__ void __launch_bounds__(512, 4) mx_direct(DirectParams p) {
  extern __shared__ __align__(16) float sums[];  // [waves][MB][4][64][4]
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int64_t n0 = (int64_t)(blockIdx.x / p.row_tiles) * 64;
  const int64_t m0 = (int64_t)(blockIdx.x % p.row_tiles) * (16 * MB);
  const int last = min(p.chunks, (int)(blockIdx.y + 1) * p.per_slice);
  floatx4 acc[MB][4];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  // row c of fragment i
  auto row_of = [&](int i) { return m0 + (TA ? MB * c + i : 16 * i + c); };
  // byte offsets of this lane's first values of a chunk
  const uint32_t row_bytes = (uint32_t)p.G * mx_group_bytes(F), row_scales = (uint32_t)p.G * 4;
  const uint32_t lda4 = (uint32_t)p.lda * 4;
  const uint32_t code_at = 8 * q * row_bytes + c * (F == MX_E2M1 ? 2 : 4);
  const uint32_t scale_at = (8 * q + (c & 7)) * row_scales + (c >> 3);
  uint32_t a_at[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const uint32_t m = (uint32_t)(min(row_of(i), (int64_t)p.M - 1) - m0);
    a_at[i] = TA ? 8 * q * lda4 + 4 * m : m * lda4 + 32 * q;
  }
  const uint8_t* codes0 = p.codes + (n0 / 4) * (F == MX_E2M1 ? 2 : 4);
  const uint8_t* scales0 = p.scales + n0 / MX_BLOCK;
  const bool pairs = TA && MB == 2 && m0 + 32 <= p.M;  // (of rows, eight bytes)
  const float* a0 = TA ? p.A + m0 : p.A + m0 * p.lda;
  for (int t = blockIdx.y * p.per_slice + wave; t < last; t += waves) {
    uint32_t w[8], s[8];
    float a[MB][8];
    const int64_t k0 = (int64_t)t * 32;
    if (k0 + 32 <= p.K && p.near) {
      const auto rw = buffer_at(codes0 + k0 * row_bytes), rs = buffer_at(scales0 + k0 * row_scales);
      const auto ra = buffer_at(a0 + (TA ? k0 * p.lda : k0));
      const int scale = __builtin_amdgcn_raw_buffer_load_b8(rs, scale_at, 0, 0);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i] = F == MX_E2M1 ? (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(rw, code_at, i * row_bytes, 0)
                            : (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rw, code_at, i * row_bytes, 0);
      if (pairs) {
        if constexpr (TA && MB == 2) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const auto x = __builtin_amdgcn_raw_buffer_load_b64(ra, a_at[0], j * lda4, 0);
            a[0][j] = __uint_as_float(x[0]);
            a[1][j] = __uint_as_float(x[1]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          if constexpr (TA) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              a[i][j] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(ra, a_at[i], j * lda4, 0));
          } else {
            const uintx4 x = __builtin_amdgcn_raw_buffer_load_b128(ra, a_at[i], 0, 0);
            const uintx4 y = __builtin_amdgcn_raw_buffer_load_b128(ra, a_at[i], 16, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) { a[i][j] = __uint_as_float(x[j]); a[i][4 + j] = __uint_as_float(y[j]); }
          }
        }
      }
      s[0] = of_eight<0>(scale), s[1] = of_eight<1>(scale), s[2] = of_eight<2>(scale), s[3] = of_eight<3>(scale);
      s[4] = of_eight<4>(scale), s[5] = of_eight<5>(scale), s[6] = of_eight<6>(scale), s[7] = of_eight<7>(scale);
    } else {
      const int64_t k = k0 + 8 * q;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // (behind K the last row again, against zeros of A)
        const int64_t row = min(k + i, p.K - 1);
        w[i] = mx_load4<F>(p.codes, row * p.G * 32 + n0 / 4 + c);
        s[i] = p.scales[row * p.G * 4 + (n0 + 4 * c) / MX_BLOCK];
      }
#pragma unroll
      for (int i = 0; i < MB; ++i)
        load_a8<TA>(p.A, p.lda, min(row_of(i), (int64_t)p.M - 1), k, p.K, a[i]);
    }
    bf16x8 b[4];
    fragments_of4<F>(w, s, b);
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      const Planes x = split8(a[i]);
      const bf16x8 parts[PLANES] = {__builtin_bit_cast(bf16x8, x.lo), __builtin_bit_cast(bf16x8, x.mid),
                                    __builtin_bit_cast(bf16x8, x.hi)};
#pragma unroll
      for (int h = 0; h < PLANES; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(parts[h], b[j], acc[i][j], 0, 0, 0);
    }
  }
  // register r of a lane: row 4 q + r, so that it holds four columns of four rows
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<floatx4*>(sums + (((wave * MB + i) * 4 + r) * 64 + lane) * 4) =
          floatx4{acc[i][0][r], acc[i][1][r], acc[i][2][r], acc[i][3][r]};
  __syncthreads();
  float* out = p.C + blockIdx.y * p.plane;
  for (int e = threadIdx.x; e < MB * 256; e += blockDim.x) {
    floatx4 v = *reinterpret_cast<const floatx4*>(sums + e * 4);
    for (int x = 1; x < waves; ++x) v += *reinterpret_cast<const floatx4*>(sums + (x * MB * 256 + e) * 4);
    const int c = ((e & 63) >> 4) * 4 + ((e >> 6) & 3), i = e >> 8;
    const int64_t row = m0 + (TA ? MB * c + i : 16 * i + c);
    const int64_t col = n0 + 4 * (e & 15);
    if (row >= p.M) continue;
    float* dst = out + row * p.ldc + col;
    if (col + 4 <= p.N) {
      *reinterpret_cast<float4u*>(dst) = float4u{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < p.N) dst[j] = v[j];
    }
  }
}

// How a product runs (us on MI355X, e4m3, a synchronous run's 13 us included, both sides in turn in
// short runs; under steady load large products take up to a tenth less):
//   * straight into registers up to 5 * 2^28 multiply-adds (1024^3 25.2, packed 33.8; 1250x1250x1000
//     32.6 against 37.3; but 1500x1500x1000 52 against 44), 3 * 2^28 where there are tiles of 128 for
//     three quarters of the CUs (2048x2048x200 25.5 against 26.2, but 2000x2000x300 34.4 against 28.8,
//     4000x4000x60 35.5 against 32.1), and whatever the depth for up to 64 rows or 128 columns, where
//     packing the other operand costs most (64x8192x8192 66 against 93, 4096x128x4096 40 against 76;
//     128 rows, 128x4096x4096, 47 against 45); two row fragments a workgroup from 2^28 on (64x4096x4096
//     35 against 41 with one, but 300x300x1000 22.2 against 21.7); eight waves a workgroup, or as few
//     as make eight a CU and have four chunks each (2048x2048x200 25.2 against 34 with seven of one
//     chunk, 3000x3000x100 33.9 against 39.5);
//   * packed on tiles of 256, of 128, or the rows of as many rounds of 256 CUs as tiles of 256 fill and
//     then the others on tiles of 128, whichever takes the fewest rounds; a tile of 256 takes 3.6 times
//     one of 128 (4096^3 342 on 256, 368 on 128; 4000x2900x2048, 192 tiles, 155 against 148;
//     4096x5120x2048, 320 tiles, 284, 250 and mixed 229; 5000x4000x2000 277, 232 and 224).
// Either is split along K into as many slices as bring 256 workgroups, of at least two chunks of 32 k a
// wave (eight fragments): 500x1021x1531 22.6 whole and 26.7 in two, 208x384x6272 26.9 in five and 29.3
// in ten, 16x4096x4096 23.4 in four and 31.1 whole; packed 1024^3 34.5 in four and 40.5 whole.
struct ProductPlan {
  bool direct;
  int mb, waves;            // direct: row fragments and waves a workgroup
  int large;                // packed: rows of tiles of 256, ahead of those of 128
  int slices, chunk;        // chunk: chunks of 32 k, or fragments, of a slice
  int64_t KT, MT, NT;       // packed: fragments along K, blocks of A and of B
};
ProductPlan plan(int64_t M, int64_t N, int64_t K) {
  ProductPlan w{};
  const double work = (double)M * (double)N * (double)K;
  int64_t units, s;
  if (work <= (mx_tiles(M, N, 128) < 192 ? 5.0 : 3.0) * (1 << 28) || M <= 64 || N <= 128) {
    w.direct = true;
    w.mb = work >= (double)(1 << 28) ? 2 : 1;
    units = (K + 31) / 32;
    const int64_t t = ((N + 63) / 64) * ((M + 16 * w.mb - 1) / (16 * w.mb));
    w.waves = (int)std::min<int64_t>({8, units, std::max<int64_t>((units + 3) / 4, (2048 + t - 1) / t)});
    s = std::min(256 / t, units / (2 * w.waves));
  } else {
    w.KT = units = (K + 15) / 16;
    w.MT = (M + 31) / 32;
    w.NT = (N + 31) / 32;
    w.large = mx_large_rows(M, N, 3.6);
    s = w.large ? 1 : std::min(256 / mx_tiles(M, N, 128), units / 8);
  }
  s = std::max<int64_t>(1, s);
  w.chunk = (int)((units + s - 1) / s);
  w.slices = (int)((units + w.chunk - 1) / w.chunk);
  return w;
}

// Rows and columns that one set of launches takes (grid dimensions); a multiple of a group.
constexpr int64_t MAX_EXTENT = 1 << 20;

int64_t piece_scratch_bytes(int64_t M, int64_t N, int64_t K) {
  const ProductPlan w = plan(M, N, K);
  return w.KT * (PLANES * w.MT + w.NT) * FRAG + (w.slices > 1 ? 4 * w.slices * M * N : 0);
}

// p.N columns of a B whose rows have G groups.
hipError_t launch_piece(const MxGemmParams& p, int64_t G, void* scratch, hipStream_t s) {
  const ProductPlan w = plan(p.M, p.N, p.K);
  char* pa = static_cast<char*>(scratch);
  char* pb = pa + w.KT * w.MT * PLANES * FRAG;
  float* partial = reinterpret_cast<float*>(pb + w.KT * w.NT * FRAG);
  float* sums = w.slices > 1 ? partial : p.C;
  const int64_t ld_sums = w.slices > 1 ? p.N : p.ldc, plane = p.M * p.N;
  if (w.direct) {
    DirectParams d{};
    d.A = p.A; d.codes = p.codes; d.scales = p.scales; d.C = sums;
    d.lda = p.lda; d.ldc = ld_sums; d.plane = plane; d.K = p.K; d.G = G;
    d.M = (int)p.M; d.N = (int)p.N; d.chunks = (int)((p.K + 31) / 32); d.per_slice = w.chunk;
    d.row_tiles = (int)((p.M + 16 * w.mb - 1) / (16 * w.mb));
    d.near = p.lda < (1 << 24) && G < (1 << 20);  // (32 rows)
    const dim3 grid((unsigned)((p.N + 63) / 64 * d.row_tiles), (unsigned)w.slices), block(64 * w.waves);
    mx_with_format(p.format, [&](auto f) {
      constexpr int F = decltype(f)::value;
      auto go = [&](auto ta, auto mb) {
        constexpr int MB = decltype(mb)::value;
        hipLaunchKernelGGL((mx_direct<F, decltype(ta)::value, MB>), grid, block, w.waves * MB * 4096, s, d);
      };
      auto by_rows = [&](auto ta) {
        if (w.mb == 1) go(ta, std::integral_constant<int, 1>());
        else go(ta, std::integral_constant<int, 2>());
      };
      if (p.transA) by_rows(std::true_type());
      else by_rows(std::false_type());
    });
  } else {
    PackParams k{p.A, p.codes, p.scales, pa, pb, p.lda, p.M, p.N, p.K, G, w.MT, w.NT,
                 mx_pack_units(p.M, p.N, p.K), (int)((p.M + 63) / 64), (int)mx_pack_blocks(p.M, p.N)};
    const dim3 packs((unsigned)mx_pack_groups(k.units));
    mx_with_format(p.format, [&](auto f) {
      constexpr int F = decltype(f)::value;
      if (p.transA) hipLaunchKernelGGL((mx_pack<F, true>), packs, dim3(PACK_THREADS), 0, s, k);
      else hipLaunchKernelGGL((mx_pack<F, false>), packs, dim3(PACK_THREADS), 0, s, k);
    });
    WideParams q{};
    q.pb = pb;
    q.ldc = ld_sums; q.plane = plane;
    q.N = (int)p.N;
    q.KT = (int)w.KT; q.MT = (int)w.MT; q.NT = (int)w.NT;
    q.chunk = w.chunk;
    auto go = [&](auto tile, int64_t row0, int64_t rows) {
      constexpr int T = decltype(tile)::value;
      if (rows <= 0) return;
      q.pa = pa + row0 / 32 * PLANES * FRAG;
      q.C = sums + row0 * ld_sums;
      q.M = (int)rows;
      q.blocks_m = (int)(w.MT - row0 / 32);
      q.tiles_m = (int)((rows + T - 1) / T);
      q.tiles_n = (int)((p.N + T - 1) / T);
      hipLaunchKernelGGL((mx_wide<T, T, 4, 2, 4>), dim3((unsigned)(q.tiles_m * q.tiles_n), (unsigned)w.slices),
                         dim3(512), 0, s, q);
    };
    const int64_t large = std::min(p.M, 256 * (int64_t)w.large);
    go(std::integral_constant<int, 256>(), 0, large);
    go(std::integral_constant<int, 128>(), large, p.M - large);
  }
  if (w.slices > 1)
    hipLaunchKernelGGL(mx_gemm_sum, dim3((unsigned)std::min<int64_t>(8192, (plane + 255) / 256)), dim3(256),
                       0, s, partial, plane, w.slices, p.C, p.ldc, p.N);
  return hipGetLastError();
}

}  // namespace

int64_t mx_gemm_scratch_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0) return 0;
  if (K == 0) return 4 * gemm_workspace_floats(M, N, K);
  int64_t bytes = 0;  // whole pieces and the last ones
  for (int64_t m : {std::min(M, MAX_EXTENT), M % MAX_EXTENT})
    for (int64_t n : {std::min(N, MAX_EXTENT), N % MAX_EXTENT})
      if (m > 0 && n > 0) bytes = std::max(bytes, piece_scratch_bytes(m, n, K));
  return bytes;
}

hipError_t launch_mx_gemm(const MxGemmParams& in, void* scratch, hipStream_t s) {
  if (in.M <= 0 || in.N <= 0) return hipSuccess;
  if (in.K == 0) {  // no products: zeros
    GemmParams g{};
    g.A = g.B = in.A;
    g.C = in.C;
    g.M = in.M; g.N = in.N;
    g.ldc = in.ldc;
    return launch_gemm(g, static_cast<float*>(scratch), s);
  }
  for (int64_t m = 0; m < in.M; m += MAX_EXTENT)
    for (int64_t n = 0; n < in.N; n += MAX_EXTENT) {
      MxGemmParams p = in;
      p.M = std::min(MAX_EXTENT, in.M - m);
      p.N = std::min(MAX_EXTENT, in.N - n);
      p.A += in.transA ? m : m * in.lda;
      p.codes += n / MX_GROUP * mx_group_bytes(in.format);
      p.scales += n / MX_BLOCK;
      p.C += m * in.ldc + n;
      const hipError_t e = launch_piece(p, mx_groups(in.N), scratch, s);
      if (e != hipSuccess) return e;
    }
  return hipSuccess;
}

}  // namespace shk
