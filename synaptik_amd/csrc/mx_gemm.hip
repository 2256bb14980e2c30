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
#include <algorithm>

#include "mx_tiles.h"

namespace shk {
namespace {

int64_t pad256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

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
  uint32_t h[8], m[8], l[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(v[i]);
    h[i] = b & 0xffff0000u;
    const float r = v[i] - __uint_as_float(h[i]);
    m[i] = __float_as_uint(r) & 0xffff0000u;
    l[i] = __float_as_uint(r - __uint_as_float(m[i]));
    if (!is_finite(v[i])) {
      h[i] = v[i] != v[i] ? b | 0x00400000u : b;
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
  uint32_t w[8], sc[8], b[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = k + i < K ? k + i : K - 1;
    w[i] = mx_load4<F>(codes, row * G * 32 + n / 4);
    sc[i] = scales[row * G * 4 + n / 32];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = mx_factor(sc[i]);
    float v[4];
    mx_values4<F>(w[i], v);
#pragma unroll
    for (int j = 0; j < 4; ++j) b[i][j] = k + i < K ? __float_as_uint(v[j] * f) : 0u;
  }
  char* at = frag_at(pb, octet, n / 32 * 32 + (n & 31) / 4, NT, 1);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uintx4 q;
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = high_halves(b[2 * i][j], b[2 * i + 1][j]);
    *reinterpret_cast<uintx4*>(at + 8 * 16 * j) = q;
  }
}

// Both operands in one launch: workgroup (bk, y) packs 32 k of 64 rows of A, then of 256 columns
// of B.
struct PackParams {
  const float* A;
  const uint8_t* codes;
  const uint8_t* scales;
  char* pa;
  char* pb;
  int64_t lda, M, N, K, MT, NT;
  int a_blocks;
};
template <int F, bool TA>
__global__ void __launch_bounds__(256) mx_pack(PackParams p) {
  if ((int)blockIdx.y < p.a_blocks) {
    if (TA) pack_a_t(p.A, p.lda, p.pa, p.M, p.K, p.MT, blockIdx.x, blockIdx.y);
    else pack_a_n(p.A, p.lda, p.pa, p.M, p.K, p.MT, blockIdx.x, blockIdx.y);
  } else {
    pack_b<F>(p.codes, p.scales, p.pb, p.N, p.K, (p.N + MX_GROUP - 1) / MX_GROUP, p.NT, blockIdx.x,
              blockIdx.y - p.a_blocks);
  }
}

// ---- the product ----
struct WideParams {
  const char* pa;
  const char* pb;
  float* C;        // or the partial sums [slices][M][N] of a product split along K
  int64_t ldc, plane;
  int M, N, KT, MT, NT;
  int tiles_m, tiles_n, chunk;  // chunk: fragments along K of a slice
};

// BM x BN results a workgroup, WM x WN waves of (BM / WM) x (BN / WN), 16 k a stage, NS stages in
// LDS. The stages are filled by global_load_lds_dwordx4, which copies 16 bytes a lane without
// passing through registers; fragments lie in memory as in LDS, so every copy and every fragment
// read is linear. A stage is copied NS - 1 stages before it is read; before a stage is read, each
// wave has waited for its own copies into it, and has finished with the stage whose place the next
// copies take. A stage's fragments are read while the one before is multiplied.
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
      const int block = min(tm * (BM / 32) + c / PLANES, p.MT - 1);
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
__global__ void __launch_bounds__(256) mx_wide_sum(const float* __restrict__ partial, int64_t plane,
                                                   int slices, float* __restrict__ C, int64_t ldc,
                                                   int64_t N) {
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < plane; e += (int64_t)gridDim.x * 256) {
    float v = partial[e];
    for (int s = 1; s < slices; ++s) v += partial[s * plane + e];
    const int64_t row = e / N;
    C[row * ldc + (e - row * N)] = v;
  }
}

// (the packing grids' second dimension)
constexpr int64_t kMaxRows = 1 << 20;

struct WidePlan {
  bool wide;
  int tile, slices, chunk;
  int64_t KT, MT, NT;
};
WidePlan plan(int64_t M, int64_t N, int64_t K) {
  WidePlan w{};
  w.KT = (K + 15) / 16;
  w.MT = (M + 31) / 32;
  w.NT = (N + 31) / 32;
  auto tiles = [&](int64_t t) { return ((M + t - 1) / t) * ((N + t - 1) / t); };
  w.wide = M >= 64 && N >= 64 && K >= 64 && (double)M * N * K >= (double)(1 << 27) &&
           M <= kMaxRows && N <= kMaxRows;
  w.tile = tiles(256) >= 128 ? 256 : 128;
  const int64_t t = tiles(w.tile);
  const int64_t s = t >= 256 ? 1 : std::max<int64_t>(1, std::min<int64_t>(256 / t, w.KT / 8));
  w.chunk = (int)((w.KT + s - 1) / s);
  w.slices = w.chunk > 0 ? (int)((w.KT + w.chunk - 1) / w.chunk) : 1;
  return w;
}

}  // namespace

int64_t mx_gemm_scratch_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0) return 0;
  const WidePlan w = plan(M, N, K);
  if (!w.wide) return pad256(4 * K * N) + 4 * gemm_workspace_floats(M, N, K);
  return w.KT * (PLANES * w.MT + w.NT) * FRAG + (w.slices > 1 ? 4 * w.slices * M * N : 0);
}

hipError_t launch_mx_gemm(const MxGemmParams& p, void* scratch, hipStream_t s) {
  if (p.M <= 0 || p.N <= 0) return hipSuccess;
  const WidePlan w = plan(p.M, p.N, p.K);
  if (!w.wide) {
    float* b = static_cast<float*>(scratch);
    const hipError_t e = launch_mx_decode(p.codes, p.scales, b, p.N, p.K, p.N, p.format, s);
    if (e != hipSuccess) return e;
    GemmParams g{};
    g.A = p.A; g.B = b; g.C = p.C;
    g.M = p.M; g.N = p.N; g.K = p.K;
    g.lda = p.lda; g.ldb = p.N; g.ldc = p.ldc;
    g.transA = p.transA;
    return launch_gemm(g, reinterpret_cast<float*>(static_cast<char*>(scratch) + pad256(4 * p.K * p.N)), s);
  }
  char* pa = static_cast<char*>(scratch);
  char* pb = pa + w.KT * w.MT * PLANES * FRAG;
  float* partial = reinterpret_cast<float*>(pb + w.KT * w.NT * FRAG);
  PackParams k{p.A, p.codes, p.scales, pa, pb, p.lda, p.M, p.N, p.K, w.MT, w.NT, (int)((p.M + 63) / 64)};
  const dim3 packs((unsigned)((w.KT + 1) / 2), (unsigned)(k.a_blocks + (p.N + 255) / 256));
  mx_with_format(p.format, [&](auto f) {
    constexpr int F = decltype(f)::value;
    if (p.transA) hipLaunchKernelGGL((mx_pack<F, true>), packs, dim3(256), 0, s, k);
    else hipLaunchKernelGGL((mx_pack<F, false>), packs, dim3(256), 0, s, k);
  });
  WideParams q{};
  q.pa = pa; q.pb = pb;
  q.C = w.slices > 1 ? partial : p.C;
  q.ldc = w.slices > 1 ? p.N : p.ldc;
  q.plane = p.M * p.N;
  q.M = (int)p.M; q.N = (int)p.N;
  q.KT = (int)w.KT; q.MT = (int)w.MT; q.NT = (int)w.NT;
  q.tiles_m = (int)((p.M + w.tile - 1) / w.tile);
  q.tiles_n = (int)((p.N + w.tile - 1) / w.tile);
  q.chunk = w.chunk;
  const dim3 grid((unsigned)(q.tiles_m * q.tiles_n), (unsigned)w.slices);
  if (w.tile == 256) hipLaunchKernelGGL((mx_wide<256, 256, 4, 2, 4>), grid, dim3(512), 0, s, q);
  else hipLaunchKernelGGL((mx_wide<128, 128, 2, 2, 4>), grid, dim3(256), 0, s, q);
  if (w.slices > 1)
    hipLaunchKernelGGL(mx_wide_sum, dim3((unsigned)std::min<int64_t>(8192, (q.plane + 255) / 256)),
                       dim3(256), 0, s, partial, q.plane, w.slices, p.C, p.ldc, p.N);
  return hipGetLastError();
}

}  // namespace shk
