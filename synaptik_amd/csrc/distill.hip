// Divergence of a model's distribution from a teacher's, of which each row's largest logits are
// known, and its gradient.
//
//   p = softmax(t / T) over a row's entries,  q = softmax(z / T) over all C classes
//   loss = T^2 / n sum over rows of sum_j p_j (log p_j - log q_{i_j}),  dz = g T / n (q - p)
//
// n counts the rows that have an entry. An entry is absent where its index is -1 or its logit is
// -inf; a row without entries has no loss and a zero gradient, and its logits are not read. An
// index outside the classes flags DEV_INDEX_OUT_OF_BOUNDS and counts as absent. An index that a row
// names twice counts with the sum of its entries' p.
//
// Bound: the logits are read once and the gradient is written once. A row is held in registers from
// its load to its gradient. The gradient is first stored as that of a teacher without entries; after
// a barrier the entries' threads store theirs; where a class is named twice (which a table in LDS
// shows), all threads of one class the same sum, in the entries' order. The exponentials of the C
// classes are binary32, their sum and all that concerns the K entries is binary64: the loss is a small
// difference of logarithms.
#include <algorithm>

#include "common.h"
#include "flag.h"
#include "kernels.h"
#include "row4.h"
#include "rowvec.h"
#include "wave_sum.h"

namespace shk {
namespace {

constexpr float NO_LOSS = -0.0f;  // of a row without entries: no row's loss is (one of -0 becomes +0)

struct DistillArgs {
  const float* z;
  const void* index;
  const float* t;
  float* grad;           // null: the loss alone
  float* row_loss;       // [R]
  const uint32_t* count; // [parts]: rows that have an entry; null: counted here
  uint32_t* status;
  int64_t R, C;
  int K, is64, parts, slots, shift;
  float per_T;           // log2(e) / T
  double inv_T, scale;   // 1 / T, g T
};

__device__ __forceinline__ int64_t entry_index(const DistillArgs& a, int64_t at) {
  return a.is64 ? static_cast<const int64_t*>(a.index)[at] : (int64_t) static_cast<const int32_t*>(a.index)[at];
}
__device__ __forceinline__ bool entry_there(const DistillArgs& a, int64_t at) {
  const int64_t i = entry_index(a, at);
  return i >= 0 && i < a.C && a.t[at] != -INFINITY;
}
// Rows with an entry that this thread finds among all of them, R at most COUNT_ROWS: the entries are read
// in order, each that is there marks its row, and the marks are counted. `marks` is read and written by
// the whole workgroup, with barriers.
constexpr int COUNT_ROWS = 1024, COUNT_ENTRIES = 1 << 14;
template <int NT>
__device__ __forceinline__ double count_rows(const DistillArgs& a, uint8_t* marks) {
  const uint32_t R = (uint32_t)a.R, total = R * (uint32_t)a.K;
  const uint32_t inv = (uint32_t)((0x100000000ull + a.K - 1) / a.K);  // ceil(2^32 / K): e / K exactly below 2^22
  for (uint32_t r = threadIdx.x; r < R; r += NT) marks[r] = 0;
  __syncthreads();
#pragma unroll 4
  for (uint32_t e = threadIdx.x; e < total; e += NT)
    if (entry_there(a, e)) marks[a.K == 1 ? e : __umulhi(e, inv)] = 1;
  __syncthreads();
  int n = 0;
  for (uint32_t r = threadIdx.x; r < R; r += NT) n += marks[r];
  return (double)n;
}
// Rows with an entry of each of the launch's parts of the rows: a wave reads a row's entries at once.
__global__ void __launch_bounds__(1024) distill_count(DistillArgs a, uint32_t* count) {
  __shared__ uint32_t found[16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t part = (a.R + gridDim.x - 1) / gridDim.x, first = min(a.R, (int64_t)blockIdx.x * part);
  const int64_t end = min(a.R, first + part);
  uint32_t n = 0;
  for (int64_t r = first + w; r < end; r += 64) {
    bool there[4] = {false, false, false, false};
    for (int j = lane; j < a.K; j += 64) {
#pragma unroll
      for (int u = 0; u < 4; ++u) there[u] |= r + 16 * u < end && entry_there(a, (r + 16 * u) * a.K + j);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) n += __any(there[u]) ? 1u : 0u;
  }
  if (lane == 0) found[w] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) n += found[i];
    count[blockIdx.x] = n;
  }
}

// exp(x / T) for x = z - m <= 0 by the hardware's power of two (1 ulp; a result that is no normal number,
// 2^-126 of the largest weight at most, is zero, NaN stays): six instructions' time where the
// polynomial of fexp.h takes twenty. [4096, 32003] took 247 us with that.
__device__ __forceinline__ float exp_weight(float x, float per_T) { return __builtin_amdgcn_exp2f(x * per_T); }
__device__ __forceinline__ float4 weights(const float4& z, float m, float per_T) {
  return make_float4(exp_weight(z.x - m, per_T), exp_weight(z.y - m, per_T), exp_weight(z.z - m, per_T),
                     exp_weight(z.w - m, per_T));
}
__device__ __forceinline__ double total(const float4& v) {
  return ((double)v.x + (double)v.y) + ((double)v.z + (double)v.w);
}
__device__ __forceinline__ float largest(const float4& v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }
__device__ __forceinline__ float4 scaled(const float4& v, float inv, float scale) {
  return make_float4((v.x * inv) * scale, (v.y * inv) * scale, (v.z * inv) * scale, (v.w * inv) * scale);
}

// The V = ceil(C / 4 NT) groups of four classes of a row of C >= 4 that a thread holds, NT groups apart:
// all but the last lie within the row for every thread; the last is there for some (`mine`), and
// begins at C - 4 at the latest, so that the row's last group overlaps the one before where C is no
// multiple of four. Both hold the same results for the classes they share, which count in sums once.
template <int NT, int V>
struct RowOf {
  int over;  // classes of the last group that the one before has too
  bool mine;
  uint32_t end;    // byte offsets
  __device__ __forceinline__ RowOf(int C) {
    const int c = 4 * ((int)threadIdx.x + (V - 1) * NT);
    mine = c < C;
    over = max(0, c - (C - 4));
    end = 4u * (uint32_t)min(c, C - 4);
  }
  __device__ __forceinline__ uint32_t at(int i) const { return 16u * (threadIdx.x + (uint32_t)(i * NT)); }
  // The sum of what the last group has alone (its classes weigh nothing where it is not this thread's).
  __device__ __forceinline__ double new_part(const float4& v) const {
    return ((over < 1 ? (double)v.x : 0.0) + (over < 2 ? (double)v.y : 0.0)) +
           ((over < 3 ? (double)v.z : 0.0) + (over < 4 ? (double)v.w : 0.0));
  }
};

// A workgroup a row, V groups of four classes a thread. V == 0: the row does not fit; one reading forms
// the largest logit and the sum about the largest so far, a second one the gradient. Four waves on
// each SIMD in every form. [4096, 32003] of 64 entries, 1.0 GB, takes 206 us, 4.8 TB/s: two workgroups a CU,
// whose loads, exponentials and stores overlap only as they happen to fall. One row a workgroup lets
// the next begin where one ends: with 1024 workgroups that take four each the step takes 236 us
// instead of 224.
template <int NT, int V>
__global__ void __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(4))) distill_rows(DistillArgs a) {
  constexpr int NW = NT / 64;
  extern __shared__ double entries[];  // K: p; then K indexes and the table
  __shared__ double red[4 * NW];
  __shared__ float fm[2][NW];
  __shared__ int found[NW];
  __shared__ uint8_t marks[COUNT_ROWS];
  __shared__ int twice;  // whether two entries name one class
  int* index = reinterpret_cast<int*>(entries + a.K);
  int* table = index + a.K;  // a.slots, a power of two of 2 K or more: the classes that were seen
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const bool counts = a.grad != nullptr && a.count == nullptr;  // the rows with an entry, beside the first row's sums
  double n = -1.0;
  if (a.grad != nullptr && a.count != nullptr) {
    n = 0.0;
    for (int i = 0; i < a.parts; ++i) n += (double)a.count[i];
  }
  const int C = (int)a.C;
  for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
    const float* row = a.z + r * a.C;
    float* out = a.grad != nullptr ? a.grad + r * a.C : nullptr;
    const RowGroups view(row, C);
    // the entries: whether there are any, whether a class is named twice, the largest logit
    if (r != blockIdx.x) __syncthreads();  // (the last row's have been read)
    for (int i = threadIdx.x; i < a.slots; i += NT) table[i] = -1;
    if (threadIdx.x == 0) twice = 0;
    __syncthreads();
    int any = 0;
    float mt = -INFINITY;
    for (int j = threadIdx.x; j < a.K; j += NT) {
      const int64_t i = entry_index(a, r * a.K + j);
      const float t = a.t[r * a.K + j];
      const bool inside = i >= 0 && i < a.C;
      if (!inside && i != -1) atomicOr(a.status, (uint32_t)DEV_INDEX_OUT_OF_BOUNDS);
      const bool there = inside && t != -INFINITY;
      index[j] = there ? (int)i : -1;
      any |= there;
      if (!there) continue;
      mt = fmaxf(mt, t);  // (a NaN makes the sums NaN)
      if (a.grad == nullptr) continue;
      for (uint32_t at = (uint32_t)i * 0x9e3779b1u >> a.shift;; at = (at + 1) & (a.slots - 1)) {
        const int old = atomicCAS(&table[at], -1, (int)i);  // (half of the slots stay free: the search ends)
        if (old == (int)i) twice = 1;
        if (old == -1 || old == (int)i) break;
      }
    }
    any = __any(any);
    if (NW > 1) {
      if (lane == 0) found[w] = any;
      __syncthreads();
      any = 0;
#pragma unroll
      for (int i = 0; i < NW; ++i) any |= found[i];
    }
    if (!any) {
      if (threadIdx.x == 0) a.row_loss[r] = NO_LOSS;
      if (out != nullptr)
        for (int q = threadIdx.x; q < view.groups; q += NT) view.store(out, q, make_float4(0.f, 0.f, 0.f, 0.f));
      continue;
    }
    // largest values
    const RowOf<NT, V> in(C);
    float4 v[V > 0 ? V : 1];
    float m = -INFINITY, thread_m = -INFINITY;
    double s[2] = {0.0, 0.0};  // the sum of exp(z - m); the rows counted
    if constexpr (V > 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (i < V - 1) v[i] = ld4_at<true>(row, in.at(i), 4);
        else v[i] = in.mine ? ld4_at<true>(row, in.end, 4) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      }
      if (counts && n < 0.0) s[1] = count_rows<NT>(a, marks);
#pragma unroll
      for (int i = 0; i < V; ++i) m = fmaxf(m, largest(v[i]));
    } else {
      if (counts && n < 0.0) s[1] = count_rows<NT>(a, marks);
      for (int q = threadIdx.x; q < view.groups; q += NT) {
        const float4 x = view.load(row, q, -INFINITY);
        const float top = fmaxf(m, largest(x));
        if (top > m) {  // (the sum so far is zero, or NaN, where m is -inf)
          s[0] *= (double)exp_weight(m - top, a.per_T);
          m = top;
        }
        // about 0 while all logits were -inf, which weigh nothing there (about themselves they are NaN)
        s[0] += total(weights(x, m > -INFINITY ? m : 0.0f, a.per_T));
      }
      thread_m = m;
    }
    m = wave_largest(m);
    mt = wave_largest(mt);
    if (NW > 1) {
      if (lane == 0) { fm[0][w] = m; fm[1][w] = mt; }
      __syncthreads();
      m = fm[0][0];
      mt = fm[1][0];
#pragma unroll
      for (int i = 1; i < NW; ++i) { m = fmaxf(m, fm[0][i]); mt = fmaxf(mt, fm[1][i]); }
    }
    if constexpr (V > 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[i] = weights(v[i], m, a.per_T);
        s[0] += i < V - 1 ? total(v[i]) : in.new_part(v[i]);
        __builtin_amdgcn_sched_barrier(0);  // four exponentials at a time keep the registers down
      }
    } else if (thread_m != m) {
      s[0] *= (double)exp_weight(thread_m - m, a.per_T);  // (zero or NaN already where thread_m is -inf)
    }
    group_sums<NT, 2>(s, red);
    if (counts && n < 0.0) n = s[1];
    const float scale = (float)(a.scale / n);
    if (out != nullptr) {
      const float inv = (float)(1.0 / s[0]);
      if constexpr (V > 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (i < V - 1) st4_at<true>(out, in.at(i), 4, scaled(v[i], inv, scale));
          else if (in.mine) st4_at<true>(out, in.end, 4, scaled(v[i], inv, scale));
        }
      } else {
        for (int q = threadIdx.x; q < view.groups; q += NT)
          view.store(out, q, scaled(weights(view.load(row, q, -INFINITY), m, a.per_T), inv, scale));
      }
    }
    // the entries, whose binary64 values need the registers that held the row
    double e[2] = {0.0, 0.0};  // sums of exp(t - mt) and of that times (t - mt - z + m)
    for (int j = threadIdx.x; j < a.K; j += NT) {
      double p = 0.0;
      if (index[j] >= 0) {
        const double t = ((double)a.t[r * a.K + j] - (double)mt) * a.inv_T;
        p = exp(t);
        const double z = ((double)row[index[j]] - (double)m) * a.inv_T;
        e[0] += p;
        if (p != 0.0) e[1] += p * (t - z);
      }
      entries[j] = p;
    }
    group_sums<NT, 2>(e, red + 2 * NW);
    if (threadIdx.x == 0) {
      const float loss = (float)(e[1] / e[0] - log(e[0]) + log(s[0]));
      a.row_loss[r] = loss == 0.0f ? 0.0f : loss;
    }
    if (out == nullptr) continue;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores above precede those below
    __syncthreads();
    for (int j = threadIdx.x; j < a.K; j += NT) {
      const int mine = index[j];
      if (mine < 0) continue;
      double p = entries[j];
      if (twice) {
        p = 0.0;
        for (int i = 0; i < a.K; ++i) p += index[i] == mine ? entries[i] : 0.0;
      }
      const double q = (double)exp_weight(row[mine] - m, a.per_T) / s[0];
      out[mine] = (float)(q - p / e[0]) * scale;
    }
  }
}

// The loss: binary64 sum of the row losses, over the number of rows that have one. Hands on the flag.
__global__ void __launch_bounds__(1024) distill_finish(const float* __restrict__ row_loss, int64_t R, double T2,
                                                       float* loss, FlagWord flag) {
  __shared__ double lds[2][16];
  double s = 0.0, n = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < R; i += 1024) {
    const float v = row_loss[i];
    s += (double)v;
    n += __float_as_uint(v) == 0x80000000u ? 0.0 : 1.0;
  }
  double v[2] = {s, n};
  group_sums<1024, 2>(v, &lds[0][0]);
  if (threadIdx.x == 0) {
    loss[0] = (float)(v[0] * T2 / v[1]);
    hand_on(flag);
  }
}

constexpr int COUNT_PARTS = 64;

template <int NT, int V>
void launch_rows(const DistillArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((distill_rows<NT, V>), dim3((unsigned)std::min<int64_t>(a.R, 1 << 20)), dim3(NT), 12 * a.K + 4 * a.slots, s, a);
}

// V groups a thread, from V to MOST by the row's width.
template <int NT, int V, int MOST>
void launch_groups(const DistillArgs& a, hipStream_t s) {
  if constexpr (V < MOST) {
    if (a.C > 4 * NT * V) return launch_groups<NT, V + 1, MOST>(a, s);
  }
  launch_rows<NT, V>(a, s);
}

}  // namespace

int64_t distill_scratch_bytes(int64_t R) { return 4 * ((R + 3) / 4 * 4) + 4 * COUNT_PARTS; }

hipError_t launch_distill(const DistillParams& p, void* scratch, FlagWord flag, hipStream_t s) {
  if (p.R <= 0) return hipSuccess;
  DistillArgs a{};
  a.z = p.logits;
  a.index = p.index;
  a.t = p.teacher;
  a.grad = p.grad;
  a.row_loss = static_cast<float*>(scratch);
  a.status = flag.status;
  a.R = p.R;
  a.C = p.C;
  a.K = (int)p.K;
  a.is64 = p.is64;
  a.slots = 2;
  a.shift = 31;
  while (a.slots < 2 * a.K) {
    a.slots *= 2;
    --a.shift;
  }
  a.per_T = (float)(1.4426950408889634 / (double)p.T);
  a.inv_T = 1.0 / (double)p.T;
  a.scale = (double)p.g * (double)p.T;
  if (p.grad != nullptr && (p.R > COUNT_ROWS || p.R * p.K > COUNT_ENTRIES)) {
    uint32_t* count = reinterpret_cast<uint32_t*>(a.row_loss + (p.R + 3) / 4 * 4);
    hipLaunchKernelGGL(distill_count, dim3(COUNT_PARTS), dim3(1024), 0, s, a, count);
    a.count = count;
    a.parts = COUNT_PARTS;
  }
  // The smallest workgroup that holds the row in at most 16 groups (64 registers) a thread, or 8 up to
  // 8192 classes: more waves for the row's latency.
  if (p.C < 4) launch_rows<64, 0>(a, s);
  else if (p.C <= 64 * 4 * 4) launch_groups<64, 1, 4>(a, s);
  else if (p.C <= 256 * 4 * 8) launch_groups<256, 2, 8>(a, s);
  else if (p.C <= 512 * 4 * 16) launch_groups<512, 5, 16>(a, s);
  else if (p.C <= 1024 * 4 * 16) launch_groups<1024, 9, 16>(a, s);
  else launch_rows<1024, 0>(a, s);
  hipLaunchKernelGGL(distill_finish, dim3(1), dim3(1024), 0, s, (const float*)a.row_loss, p.R,
                     (double)p.T * (double)p.T, p.loss, flag);
  return hipGetLastError();
}

}  // namespace shk
