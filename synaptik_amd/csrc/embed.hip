// Rows of a table by token, and the table's gradient.
//
//   Y[n, :]  = scale * W[t_n, :]                         (zero where t_n is the padding token)
//   dW[v, :] = scale * sum over n with t_n = v of dY[n, :]
//
// A token outside the table flags DEV_INDEX_OUT_OF_BOUNDS; its row of Y is zero and it adds nothing
// to dW. Bound: both move each row once.
//
// The gradient's order of summation is fixed: the rows' ordinals are sorted by token (stable, by
// digits of EG_BITS bits), the sorted list is cut every 8 or 32 rows wherever a token's rows begin
// or end, a wave sums a piece's rows in ascending order in binary64, and a token whose rows lie
// in several pieces gets its parts added in ascending order. So a frequent token costs no more than
// as many rows of different ones, nothing is added by atomics, and results do not depend on what
// runs when.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "flag.h"
#include "kernels.h"
#include "row4.h"

namespace shk {
namespace {

// The token of row n as a table row, or V where there is none (padding, out of bounds).
struct Tokens {
  const void* t;
  int64_t N, V, pad;
  int is64, has_pad;
  FlagWord flag;
  __device__ __forceinline__ uint32_t key(int64_t n, bool flags) const {
    const int64_t v = is64 ? static_cast<const int64_t*>(t)[n] : (int64_t) static_cast<const int32_t*>(t)[n];
    if (has_pad && v == pad) return (uint32_t)V;
    if (v >= 0 && v < V) return (uint32_t)v;
    if (flags) flag_out_of_bounds(flag);
    return (uint32_t)V;
  }
};

// ---- lookup: L lanes a row, each four columns of every 4 L, U rows at once ----
// Bound: memory; the rows' addresses depend on the tokens, so that U rows' loads are in flight in every
// lane. [65536, 1024] of 32003 rows takes 65 us (the 268 MB that it writes past the caches alone 41 us);
// with writes through the caches 103 us.
template <int L, int U>
__global__ void __launch_bounds__(256) embed_rows(Tokens t, const float* __restrict__ w, float* __restrict__ y,
                                                  int64_t D, int64_t ldy, float scale) {
  constexpr int TEAMS = 256 / L;
  const int lane = threadIdx.x % L;
  const int64_t first = ((int64_t)blockIdx.y * L + lane) * 4, step = (int64_t)gridDim.y * L * 4;
  for (int64_t base = (int64_t)blockIdx.x * (TEAMS * U) + threadIdx.x / L; base < t.N;
       base += (int64_t)gridDim.x * (TEAMS * U)) {
    uint32_t key[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t n = base + u * TEAMS;
      key[u] = n < t.N ? t.key(n, first == 0) : (uint32_t)t.V;
    }
    for (int64_t c = first; c < D; c += step) {
      float4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[u] = key[u] < (uint32_t)t.V ? ld4(w + key[u] * D + c, D - c) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t n = base + u * TEAMS;
        if (n < t.N)
          st4<true>(y + n * ldy + c, D - c,
                    make_float4(v[u].x * scale, v[u].y * scale, v[u].z * scale, v[u].w * scale));
      }
    }
  }
}

template <int L, int U>
void launch_rows(const Tokens& t, const float* w, float* y, int64_t D, int64_t ldy, float scale, hipStream_t s) {
  const int64_t rows = 256 / L * U;
  const unsigned gx = (unsigned)std::min<int64_t>((t.N + rows - 1) / rows, 1 << 18);
  const unsigned gy = (unsigned)std::min<int64_t>((D + 4 * L - 1) / (4 * L), 1 << 6);
  hipLaunchKernelGGL((embed_rows<L, U>), dim3(gx, gy), dim3(256), 0, s, t, w, y, D, ldy, scale);
}

// ---- sorting ----
constexpr int EG_BITS = 9, EG_BINS = 1 << EG_BITS;
constexpr int EG_KEYS = 4;                     // keys a thread
constexpr int EG_SORT = 1024 * EG_KEYS;        // keys a workgroup
constexpr int64_t EG_SCAN_TILES = 64;          // up to here a workgroup adds the others' counts itself
constexpr int EG_SMALL_KEYS = 8, EG_SMALL = 1024 * EG_SMALL_KEYS;  // keys that one workgroup sorts
constexpr int64_t EG_FLAGS = 1 << 20;          // table rows up to which a byte each says whether a token names it

// Among the wave's active lanes: those whose digit is this lane's.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, bool active) {
  uint64_t mask = __ballot(active);
#pragma unroll
  for (int b = 0; b < EG_BITS; ++b) {
    const uint64_t set = __ballot((digit >> b) & 1);
    mask &= ((digit >> b) & 1) ? set : ~set;
  }
  return mask;
}

// Rank of each of a wave's keys among its wave's keys of the same digit: nine ballots find the lanes of
// one digit, whose first adds their number to the wave's counter. Bound: latency (a round is some 60
// dependent instructions), so a workgroup has sixteen waves of few keys: 32768 rows' scattering pass
// takes 9.9 us, with four waves of four times the keys 13.8. K rounds of 64 keys in
// order; count: the wave's EG_BINS counters in LDS, zero before, the digits' counts after.
template <int K>
__device__ __forceinline__ void wave_ranks(const uint32_t (&digit)[K], const bool (&active)[K],
                                           uint32_t* count, uint32_t (&rank)[K]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const uint64_t same = same_digit(digit[i], active[i]);
    const int before = __popcll(same & ((1ull << lane) - 1));
    uint32_t old = 0;
    if (active[i] && before == 0) old = atomicAdd(&count[digit[i]], (uint32_t)__popcll(same));
    rank[i] = __shfl(old, active[i] ? __ffsll((unsigned long long)same) - 1 : lane, 64) + before;
  }
}

// Exclusive prefix sums of EG_BINS values in LDS, by NT >= EG_BINS / 2 threads.
template <int NT>
__device__ __forceinline__ void scan_bins(uint32_t* v, uint32_t* wave_sum_lds) {
  constexpr int T = EG_BINS / 2;  // threads that take part: two bins each
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t a = 0, b = 0, x = 0;
  if (threadIdx.x < T) {
    a = v[2 * threadIdx.x];
    b = v[2 * threadIdx.x + 1];
    x = a + b;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t up = __shfl_up(x, o, 64);
      if (lane >= o) x += up;
    }
    if (lane == 63) wave_sum_lds[w] = x;
  }
  __syncthreads();
  if (threadIdx.x < T) {
    uint32_t base = x - a - b;
    for (int i = 0; i < w; ++i) base += wave_sum_lds[i];
    v[2 * threadIdx.x] = base;
    v[2 * threadIdx.x + 1] = base + a;
  }
  __syncthreads();
}

// Zeros in the bytes of `flags` (none: null) that thread `at` of `of` takes.
__device__ __forceinline__ void clear_flags(uint8_t* flags, int64_t V, int64_t at, int64_t of) {
  if (flags == nullptr) return;
  for (int64_t i = 16 * at; i < V; i += 16 * of) *reinterpret_cast<uint4*>(flags + i) = make_uint4(0, 0, 0, 0);
}

// Sorted keys and row ordinals of up to 1024 K rows in one launch, in LDS from digit to digit: 5001 rows by two
// digits take 15.6 us, in four launches 37 us.
template <int K>
__global__ void __launch_bounds__(1024) eg_sort_small(Tokens t, int passes, uint32_t* __restrict__ keys,
                                                      uint32_t* __restrict__ rows, uint8_t* flags) {
  constexpr int NW = 16;
  __shared__ uint32_t count[NW][EG_BINS];
  __shared__ uint32_t base[EG_BINS];
  __shared__ uint32_t sums[EG_BINS / 128];
  __shared__ uint32_t lk[1024 * K];
  __shared__ uint16_t lr[1024 * K];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int N = (int)t.N;
  uint32_t key[K];
  uint16_t row[K];
  bool active[K];
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int n = w * 64 * K + i * 64 + lane;
    active[i] = n < N;
    key[i] = active[i] ? t.key(n, true) : 0u;
    row[i] = (uint16_t)n;
  }
  clear_flags(flags, t.V, threadIdx.x, 1024);
  for (int p = 0; p < passes; ++p) {
    uint32_t digit[K], rank[K];
#pragma unroll
    for (int i = 0; i < K; ++i) digit[i] = (key[i] >> (p * EG_BITS)) & (EG_BINS - 1);
#pragma unroll
    for (int i = 0; i < NW * EG_BINS / 1024; ++i) (&count[0][0])[threadIdx.x + 1024 * i] = 0;
    __syncthreads();
    wave_ranks<K>(digit, active, count[w], rank);
    __syncthreads();
    if (threadIdx.x < EG_BINS) {
      uint32_t c[NW], sum = 0;
#pragma unroll
      for (int i = 0; i < NW; ++i) c[i] = count[i][threadIdx.x];
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        count[i][threadIdx.x] = sum;
        sum += c[i];
      }
      base[threadIdx.x] = sum;
    }
    __syncthreads();
    scan_bins<1024>(base, sums);
#pragma unroll
    for (int i = 0; i < K; ++i) {
      if (active[i]) {
        const uint32_t to = base[digit[i]] + count[w][digit[i]] + rank[i];
        lk[to] = key[i];
        lr[to] = row[i];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int n = w * 64 * K + i * 64 + lane;
      if (active[i]) {
        key[i] = lk[n];
        row[i] = lr[n];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int n = w * 64 * K + i * 64 + lane;
    if (active[i]) {
      keys[n] = key[i];
      rows[n] = row[i];
      if (flags != nullptr && key[i] < t.V) flags[key[i]] = 1;  // (cleared before the barriers above)
    }
  }
}

// Digit counts of each EG_SORT keys: count[tile][bin]. The first pass reads the tokens.
__global__ void __launch_bounds__(1024) eg_count(Tokens t, const uint32_t* __restrict__ keys, int shift,
                                                 uint32_t* __restrict__ count, uint8_t* flags) {
  __shared__ uint32_t h[4][EG_BINS];
  clear_flags(flags, t.V, (int64_t)blockIdx.x * 1024 + threadIdx.x, (int64_t)gridDim.x * 1024);
  for (int i = threadIdx.x; i < 4 * EG_BINS; i += 1024) (&h[0][0])[i] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * EG_SORT;
#pragma unroll
  for (int i = 0; i < EG_KEYS; ++i) {
    const int64_t n = first + i * 1024 + threadIdx.x;
    if (n < t.N) {
      const uint32_t key = keys != nullptr ? keys[n] : t.key(n, true);
      atomicAdd(&h[(threadIdx.x >> 6) & 3][(key >> shift) & (EG_BINS - 1)], 1u);
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < EG_BINS; b += 1024)
    count[(int64_t)blockIdx.x * EG_BINS + b] = (h[0][b] + h[1][b]) + (h[2][b] + h[3][b]);
}

// count[tile][bin] becomes the sum of the bin's counts in the tiles before; row `tiles` the bin's
// whole count. One workgroup for 64 bins, four parts of the tiles.
__global__ void __launch_bounds__(256) eg_scan(uint32_t* __restrict__ count, int64_t tiles) {
  __shared__ uint32_t sum[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t part = (tiles + 3) / 4, lo = min(tiles, w * part), hi = min(tiles, lo + part);
  uint32_t* c = count + blockIdx.x * 64 + lane;
  uint32_t s = 0;
  for (int64_t i = lo; i < hi; ++i) s += c[i * EG_BINS];
  sum[w][lane] = s;
  __syncthreads();
  uint32_t run = 0;
  for (int i = 0; i < w; ++i) run += sum[i][lane];
  for (int64_t i = lo; i < hi; ++i) {
    const uint32_t v = c[i * EG_BINS];
    c[i * EG_BINS] = run;
    run += v;
  }
  if (w == 3) c[tiles * EG_BINS] = run;
}

// Moves each key and its row to its place by one digit.
__global__ void __launch_bounds__(1024) eg_scatter(Tokens t, const uint32_t* __restrict__ keys,
                                                   const uint32_t* __restrict__ rows, int shift,
                                                   const uint32_t* __restrict__ count, int64_t tiles,
                                                   uint32_t* __restrict__ keys_out,
                                                   uint32_t* __restrict__ rows_out, uint8_t* flags) {
  constexpr int K = EG_KEYS, NW = 16;
  __shared__ uint32_t h[NW][EG_BINS];
  __shared__ uint32_t base[EG_BINS], before[EG_BINS];
  __shared__ uint32_t sums[EG_BINS / 128];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t first = (int64_t)blockIdx.x * EG_SORT + w * 64 * K + lane;
  uint32_t key[K], row[K], digit[K], rank[K];
  bool active[K];
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int64_t n = first + i * 64;
    active[i] = n < t.N;
    key[i] = !active[i] ? 0u : keys != nullptr ? keys[n] : t.key(n, false);
    row[i] = !active[i] ? 0u : rows != nullptr ? rows[n] : (uint32_t)n;
    digit[i] = (key[i] >> shift) & (EG_BINS - 1);
  }
  for (int i = threadIdx.x; i < NW * EG_BINS; i += 1024) (&h[0][0])[i] = 0;
  if (threadIdx.x < EG_BINS) {
    const uint32_t* c = count + threadIdx.x;
    uint32_t all = 0, mine = 0;
    if (tiles <= EG_SCAN_TILES) {
#pragma unroll 8
      for (int64_t i = 0; i < tiles; ++i) {
        const uint32_t v = c[i * EG_BINS];
        all += v;
        mine += i < blockIdx.x ? v : 0u;
      }
    } else {
      all = c[tiles * EG_BINS];
      mine = c[(int64_t)blockIdx.x * EG_BINS];
    }
    base[threadIdx.x] = all;
    before[threadIdx.x] = mine;
  }
  __syncthreads();
  wave_ranks<K>(digit, active, h[w], rank);
  scan_bins<1024>(base, sums);
  if (threadIdx.x < EG_BINS) {
    uint32_t run = base[threadIdx.x] + before[threadIdx.x];
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const uint32_t c = h[i][threadIdx.x];
      h[i][threadIdx.x] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < K; ++i) {
    if (active[i]) {
      const uint32_t to = h[w][digit[i]] + rank[i];
      keys_out[to] = key[i];
      rows_out[to] = row[i];
      if (flags != nullptr && key[i] < t.V) flags[key[i]] = 1;
    }
  }
}

// ---- sums ----
struct SumArgs {
  const float* dy;
  const uint32_t* keys;  // sorted
  const uint32_t* rows;  // the row of dY of each
  float* dw;
  double* part;          // [tiles][2][D]: a piece that begins before its tile, one that ends behind it
  const uint8_t* flags;  // [V]: whether a token names the row; null: the sorted keys are searched
  int64_t N, V, D, ldy, tiles, segments;  // segments of 256 columns
  double scale;
  int accumulate;
};

__device__ __forceinline__ void eg_result(const SumArgs& a, uint32_t key, int64_t c, const double (&acc)[4]) {
  float* p = a.dw + key * a.D + c;
  float4 o = make_float4((float)(acc[0] * a.scale), (float)(acc[1] * a.scale), (float)(acc[2] * a.scale),
                         (float)(acc[3] * a.scale));
  if (a.accumulate) {
    const float4 old = ld4(p, a.D - c);
    o = make_float4(old.x + o.x, old.y + o.y, old.z + o.z, old.w + o.w);
  }
  st4<true>(p, a.D - c, o);
}

// A wave's part: EG_TILE rows of the sorted list, 256 columns. The tile's keys and rows are in a lane
// each, so that the control flow is the wave's and eight rows are read at once. Bound: memory. [32768,
// 1024] over 65536 rows takes 83 us: 134 MB read, 276 MB written, of which 223 are the zeros of rows
// without tokens, which the same launch writes.
template <int EG_TILE>
__device__ __forceinline__ void eg_sum_tile(const SumArgs& a, int64_t tile, int64_t segment) {
  const int lane = threadIdx.x & 63;
  const int64_t first = tile * EG_TILE, count = min((int64_t)EG_TILE, a.N - first);
  const int64_t c = segment * 256 + 4 * lane;
  // the keys from the one before the tile to the one behind it, one a lane
  const int64_t at = first - 1 + lane;
  const uint32_t none = (uint32_t)a.V;
  const uint32_t key_l = lane < EG_TILE + 2 && at >= 0 && at < a.N ? a.keys[at] : none;
  const uint32_t row_l = lane < EG_TILE && first + lane < a.N ? a.rows[first + lane] : 0u;
  auto key_of = [&](int i) { return (uint32_t)__builtin_amdgcn_readlane((int)key_l, i + 1); };
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  bool open = first > 0 && key_of(0) == key_of(-1);  // the piece began before this tile
  constexpr int U = 8;
  for (int i0 = 0; i0 < (int)count; i0 += U) {
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + u, (int)count - 1);
      const uint32_t row = (uint32_t)__builtin_amdgcn_readlane((int)row_l, i);
      v[u] = key_of(i) < none ? ld4<true>(a.dy + row * a.ldy + c, a.D - c) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      if (i >= (int)count) break;
      const uint32_t key = key_of(i);
      if (key >= none) return;  // (sorted last)
      acc[0] += (double)v[u].x;
      acc[1] += (double)v[u].y;
      acc[2] += (double)v[u].z;
      acc[3] += (double)v[u].w;
      const bool ends = i + 1 < (int)count && key_of(i + 1) != key;
      if (!ends && i + 1 < (int)count) continue;
      // the piece's end: a token's last row, or the tile's
      const bool goes_on = !ends && first + count < a.N && key_of((int)count) == key;
      if (!open && !goes_on) {
        eg_result(a, key, c, acc);
      } else {
        double* p = a.part + ((2 * tile + (open ? 0 : 1)) * a.D + c);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < a.D) p[j] = acc[j];
      }
      open = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = 0.0;
    }
  }
}

// Zeros in the table rows v0 + j for the bits j of `todo` (the same in the wave).
__device__ __forceinline__ void eg_clear(const SumArgs& a, int64_t v0, uint32_t todo) {
  while (todo != 0) {
    const int j = __ffs(todo) - 1;
    todo &= todo - 1;
    float* row = a.dw + (v0 + j) * a.D;
    for (int64_t c = 4 * (threadIdx.x & 63); c < a.D; c += 256)
      st4<true>(row + c, a.D - c, make_float4(0.f, 0.f, 0.f, 0.f));
  }
}
// Zeros in those of EG_FILL table rows from v0 on that no token names.
constexpr int EG_FILL = 16;
__device__ __forceinline__ void eg_fill_rows(const SumArgs& a, int64_t v0) {
  const int lane = threadIdx.x & 63;
  const int64_t v = v0 + (lane % EG_FILL);
  bool absent = v < a.V;
  if (a.flags != nullptr) {
    absent = absent && a.flags[v] == 0;
  } else {
    // the first of the sorted keys that is not below v
    int64_t lo = 0, hi = a.N;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (a.keys[mid] < v) lo = mid + 1;
      else hi = mid;
    }
    absent = absent && !(lo < a.N && a.keys[lo] == v);
  }
  eg_clear(a, v0, (uint32_t)__ballot(absent) & ((1u << EG_FILL) - 1));
}

template <int EG_TILE>
__global__ void __launch_bounds__(256) eg_sum(SumArgs a, int64_t sum_groups) {
  const int w = threadIdx.x >> 6;
  if (blockIdx.x < sum_groups) {
    const int64_t units = a.tiles * a.segments;
    for (int64_t u = (int64_t)blockIdx.x * 4 + w; u < units; u += sum_groups * 4)
      eg_sum_tile<EG_TILE>(a, u / a.segments, u % a.segments);
    return;
  }
  const int64_t waves = ((int64_t)gridDim.x - sum_groups) * 4;
  for (int64_t v = (((int64_t)blockIdx.x - sum_groups) * 4 + w) * EG_FILL; v < a.V; v += waves * EG_FILL)
    eg_fill_rows(a, v);
}

// Up to EG_DIRECT rows in one launch, without sorting: every wave holds all keys, four a lane. A wave of
// the first `sum_groups` workgroups takes one row of dY and 256 columns, and sums the rows of its
// token if it is the first of them; the others clear table rows. [256, 256] over 2000 rows takes 7.5 us,
// sorted first (257 rows) 16 us in three launches.
constexpr int EG_DIRECT = 256;
__global__ void __launch_bounds__(256) eg_direct(Tokens t, SumArgs a, int64_t sum_groups) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint32_t none = (uint32_t)a.V;
  uint32_t key[EG_DIRECT / 64];
#pragma unroll
  for (int i = 0; i < EG_DIRECT / 64; ++i) {
    const int64_t n = i * 64 + lane;
    key[i] = n < t.N ? t.key(n, blockIdx.x == 0 && w == 0) : none;
  }
  if (blockIdx.x < sum_groups) {
    const int64_t units = a.N * a.segments;
    for (int64_t u = (int64_t)blockIdx.x * 4 + w; u < units; u += sum_groups * 4) {
      const int n = (int)(u / a.segments);
      const int64_t c = (u % a.segments) * 256 + 4 * lane;
      uint32_t mine = none;
#pragma unroll
      for (int i = 0; i < EG_DIRECT / 64; ++i)
        if (i == n / 64) mine = (uint32_t)__builtin_amdgcn_readlane((int)key[i], n % 64);
      if (mine >= none) continue;
      uint64_t same[EG_DIRECT / 64];
      bool first = true;
#pragma unroll
      for (int i = 0; i < EG_DIRECT / 64; ++i) {
        same[i] = __ballot(key[i] == mine);
        if (i < n / 64) first = first && same[i] == 0;
        else if (i == n / 64) first = first && (same[i] & ((1ull << (n % 64)) - 1)) == 0;
      }
      if (!first) continue;
      double acc[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
      for (int i = 0; i < EG_DIRECT / 64; ++i) {
        uint64_t todo = same[i];
        while (todo != 0) {
          constexpr int U = 8;
          float4 v[U];
#pragma unroll
          for (int k = 0; k < U; ++k) {
            v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (todo != 0) {
              const int64_t row = i * 64 + __ffsll((unsigned long long)todo) - 1;
              todo &= todo - 1;
              v[k] = ld4(a.dy + row * a.ldy + c, a.D - c);
            }
          }
#pragma unroll
          for (int k = 0; k < U; ++k) {
            acc[0] += (double)v[k].x;
            acc[1] += (double)v[k].y;
            acc[2] += (double)v[k].z;
            acc[3] += (double)v[k].w;
          }
        }
      }
      if (c < a.D) eg_result(a, mine, c, acc);
    }
    return;
  }
  const int64_t waves = ((int64_t)gridDim.x - sum_groups) * 4;
  for (int64_t v0 = (((int64_t)blockIdx.x - sum_groups) * 4 + w) * EG_FILL; v0 < a.V; v0 += waves * EG_FILL) {
    int named = 0;
#pragma unroll
    for (int i = 0; i < EG_DIRECT / 64; ++i) {
      const uint32_t at = key[i] - (uint32_t)v0;
      if (at < EG_FILL) named |= 1 << at;
    }
    const int rows = (int)min((int64_t)EG_FILL, a.V - v0);
    eg_clear(a, v0, ~(uint32_t)wave_or(named) & ((1u << rows) - 1));
  }
}

// Adds up the parts of a token whose rows lie in several tiles. One workgroup for the tile in which
// the token's rows begin and 256 columns; its four waves take consecutive quarters of the tiles
// behind, whose parts are the first pieces there. Bound: latency; 10 us for 1024 tiles of 1024 columns
// whose most frequent token lies in 64 of them.
template <int EG_TILE>
__global__ void __launch_bounds__(256) eg_join(SumArgs a) {
  __shared__ double part[4][256];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t units = (a.tiles - 1) * a.segments;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t tile = u / a.segments, c = (u % a.segments) * 256 + 4 * lane;
    const int64_t end = (tile + 1) * EG_TILE;  // (a tile that another one follows is full)
    const uint32_t key = a.keys[end - 1];
    if (key >= a.V || a.keys[end] != key) continue;
    const int64_t first = tile * EG_TILE;
    if (first > 0 && a.keys[first - 1] == key) continue;  // began in an earlier tile
    // the first tile behind whose last key is not this token's (64 at a time)
    int64_t lo = tile + 1;
    while (lo < a.tiles) {
      const int64_t i = lo + lane;
      const bool same = i < a.tiles && a.keys[min(a.N, (i + 1) * EG_TILE) - 1] == key;
      const uint64_t other = ~__ballot(same);
      if (other != 0) {
        lo += __ffsll((unsigned long long)other) - 1;
        break;
      }
      lo += 64;
    }
    // the last tile with a part: lo itself if its first row is the token's
    lo = min(lo, a.tiles);
    const int64_t stop = lo < a.tiles && a.keys[lo * EG_TILE] == key ? lo + 1 : lo;
    const int64_t n = stop - (tile + 1), quarter = (n + 3) / 4;
    const int64_t from = tile + 1 + min(n, w * quarter), to = tile + 1 + min(n, (w + 1) * quarter);
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    if (w == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < a.D) acc[j] = a.part[(2 * tile + 1) * a.D + c + j];
    }
    constexpr int U = 8;
    for (int64_t i0 = from; i0 < to; i0 += U) {
      double v[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const double* p = a.part + 2 * min(i0 + u, to - 1) * a.D + c;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[u][j] = i0 + u < to && c + j < a.D ? p[j] : 0.0;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] += v[u][j];
    }
    __syncthreads();  // (the last round's sums have been read)
#pragma unroll
    for (int j = 0; j < 4; ++j) part[w][4 * lane + j] = acc[j];
    __syncthreads();
    if (w == 0 && c < a.D) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc[j] = ((part[0][4 * lane + j] + part[1][4 * lane + j]) + part[2][4 * lane + j]) + part[3][4 * lane + j];
      eg_result(a, key, c, acc);
    }
  }
}

int64_t round16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

// Digits of the keys 0 .. V.
int key_digits(int64_t V) {
  int n = 1;
  while (n * EG_BITS < 32 && (V >> (n * EG_BITS)) != 0) ++n;
  return n;
}
// What embed_grad keeps, for more rows than EG_DIRECT: a list of keys and rows, a second one where a sort
// goes from one to the other, with its digit counts; flags where rows are cleared; parts of sums.
struct Layout {
  int64_t keys[2], rows[2], count, flags, part, bytes;
};
// Sorted rows that a wave sums: 32, or 8 where that leaves fewer than eight waves for each CU.
int64_t tile_rows(int64_t N, int64_t D) { return (N + 31) / 32 * ((D + 255) / 256) < 2048 ? 8 : 32; }
Layout layout(int64_t N, int64_t V, int64_t D, bool accumulate) {
  Layout l{};
  if (N <= EG_DIRECT || V <= 0 || D <= 0) return l;
  const int64_t sort = (N + EG_SORT - 1) / EG_SORT, rows = tile_rows(N, D), tiles = (N + rows - 1) / rows;
  int64_t off = 0;
  auto take = [&](int64_t bytes) {
    const int64_t at = off;
    off += round16(bytes);
    return at;
  };
  const bool launches = N > EG_SMALL;  // one for each digit's counts, one for its places
  for (int i = 0; i < 2; ++i) {
    const int64_t n = i == 0 || (launches && key_digits(V) > 1) ? N : 0;
    l.keys[i] = take(4 * n);
    l.rows[i] = take(4 * n);
  }
  l.count = take(launches ? 4 * (sort + 1) * EG_BINS : 0);
  l.flags = take(!accumulate && V <= EG_FLAGS ? V : 0);
  l.part = take(tiles > 1 ? 16 * tiles * D : 0);
  l.bytes = off;
  return l;
}

Tokens tokens_of(const EmbedParams& p, FlagWord flag) {
  return Tokens{p.tokens, p.N, p.V, p.pad, p.is64, p.has_pad, flag};
}

}  // namespace

hipError_t launch_embed(const EmbedParams& p, FlagWord flag, hipStream_t s) {
  if (p.N <= 0 || p.D <= 0) return hipSuccess;
  const Tokens t = tokens_of(p, flag);
  // lanes for a row's groups of four; four rows at once where there are enough for every CU
  const bool many = (double)p.N * (double)p.D >= (double)(1 << 20);
  auto go = [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    if (many) launch_rows<L, 4>(t, p.w, p.y, p.D, p.ldy, p.scale, s);
    else launch_rows<L, 1>(t, p.w, p.y, p.D, p.ldy, p.scale, s);
  };
  if (p.D <= 16) go(std::integral_constant<int, 4>());
  else if (p.D <= 64) go(std::integral_constant<int, 16>());
  else go(std::integral_constant<int, 64>());
  return hipGetLastError();
}

int64_t embed_grad_scratch_bytes(int64_t N, int64_t V, int64_t D, bool accumulate) {
  return layout(N, V, D, accumulate).bytes;
}

hipError_t launch_embed_grad(const EmbedParams& p, void* scratch, FlagWord flag, hipStream_t s) {
  if (p.V <= 0 || p.D <= 0 || (p.N <= 0 && p.accumulate)) return hipSuccess;
  const Tokens t = tokens_of(p, flag);
  const Layout l = layout(p.N, p.V, p.D, p.accumulate != 0);
  char* base = static_cast<char*>(scratch);
  uint32_t* keys[2] = {reinterpret_cast<uint32_t*>(base + l.keys[0]), reinterpret_cast<uint32_t*>(base + l.keys[1])};
  uint32_t* rows[2] = {reinterpret_cast<uint32_t*>(base + l.rows[0]), reinterpret_cast<uint32_t*>(base + l.rows[1])};
  uint32_t* count = reinterpret_cast<uint32_t*>(base + l.count);
  // (rows are cleared here only where the table's gradient is not added to)
  uint8_t* flags = !p.accumulate && p.V <= EG_FLAGS ? reinterpret_cast<uint8_t*>(base + l.flags) : nullptr;
  const int passes = key_digits(p.V);
  int at = 0;
  SumArgs a{};
  a.dy = p.w;
  a.dw = p.y;
  a.part = reinterpret_cast<double*>(base + l.part);
  a.N = p.N;
  a.V = p.V;
  a.D = p.D;
  a.ldy = p.ldy;
  a.flags = flags;
  const int64_t tile = tile_rows(p.N, p.D);
  a.tiles = (p.N + tile - 1) / tile;
  a.segments = (p.D + 255) / 256;
  a.scale = (double)p.scale;
  a.accumulate = p.accumulate;
  constexpr int64_t MOST = 1 << 20;  // workgroups of either half
  const int64_t fills = p.accumulate ? 0 : std::min<int64_t>((p.V + 4 * EG_FILL - 1) / (4 * EG_FILL), MOST);
  if (p.N <= EG_DIRECT) {
    const int64_t rows_of = std::min<int64_t>((p.N * a.segments + 3) / 4, MOST);
    hipLaunchKernelGGL(eg_direct, dim3((unsigned)(rows_of + fills)), dim3(256), 0, s, t, a, rows_of);
    return hipGetLastError();
  }
  if (p.N <= EG_SMALL) {
    auto sort = [&](auto k) {
      constexpr int K = decltype(k)::value;
      hipLaunchKernelGGL(eg_sort_small<K>, dim3(1), dim3(1024), 0, s, t, passes, keys[0], rows[0], flags);
    };
    if (p.N <= 1024) sort(std::integral_constant<int, 1>());
    else if (p.N <= 2048) sort(std::integral_constant<int, 2>());
    else if (p.N <= 4096) sort(std::integral_constant<int, 4>());
    else if (p.N <= 6144) sort(std::integral_constant<int, 6>());
    else sort(std::integral_constant<int, EG_SMALL_KEYS>());
  } else {
    const int64_t tiles = (p.N + EG_SORT - 1) / EG_SORT;
    for (int i = 0; i < passes; ++i) {
      const uint32_t* ki = i == 0 ? nullptr : keys[at];
      const uint32_t* ri = i == 0 ? nullptr : rows[at];
      const int to = i == 0 ? 0 : 1 - at;
      hipLaunchKernelGGL(eg_count, dim3((unsigned)tiles), dim3(1024), 0, s, t, ki, i * EG_BITS, count,
                         i == 0 ? flags : nullptr);
      if (tiles > EG_SCAN_TILES)
        hipLaunchKernelGGL(eg_scan, dim3(EG_BINS / 64), dim3(256), 0, s, count, tiles);
      hipLaunchKernelGGL(eg_scatter, dim3((unsigned)tiles), dim3(1024), 0, s, t, ki, ri, i * EG_BITS,
                         (const uint32_t*)count, tiles, keys[to], rows[to], i == 0 ? flags : nullptr);
      at = to;
    }
  }
  a.keys = keys[at];
  a.rows = rows[at];
  const int64_t sums = std::min<int64_t>((a.tiles * a.segments + 3) / 4, MOST);
  auto go = [&](auto rows_of_tile) {
    constexpr int TILE = decltype(rows_of_tile)::value;
    hipLaunchKernelGGL(eg_sum<TILE>, dim3((unsigned)(sums + fills)), dim3(256), 0, s, a, sums);
    if (a.tiles > 1)
      hipLaunchKernelGGL(eg_join<TILE>, dim3((unsigned)std::min<int64_t>((a.tiles - 1) * a.segments, MOST)), dim3(256),
                         0, s, a);
  };
  if (tile == 8) go(std::integral_constant<int, 8>());
  else go(std::integral_constant<int, 32>());
  return hipGetLastError();
}

}  // namespace shk
