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
// a barrier the entries' threads store theirs (all threads of one index the same sum, in the
// entries' order). The exponentials of the C classes are binary32 (fexp.h), their sum and all that
// concerns the K entries is binary64: the loss is a small difference of logarithms.
#include <algorithm>

#include "common.h"
#include "fexp.h"
#include "kernels.h"
#include "rowvec.h"

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
  int K, is64, parts;
  float inv_T;           // 1 / T
  double inv_T64, scale; // g T
};

__device__ __forceinline__ int64_t entry_index(const DistillArgs& a, int64_t at) {
  return a.is64 ? static_cast<const int64_t*>(a.index)[at] : (int64_t) static_cast<const int32_t*>(a.index)[at];
}
__device__ __forceinline__ bool entry_there(const DistillArgs& a, int64_t at) {
  const int64_t i = entry_index(a, at);
  return i >= 0 && i < a.C && a.t[at] != -INFINITY;
}
// Rows among [first, end) with an entry: thread i's are every NT-th.
template <int NT>
__device__ __forceinline__ double count_rows(const DistillArgs& a, int64_t first, int64_t end, double* dl) {
  int64_t n = 0;
  for (int64_t r = first + threadIdx.x; r < end; r += NT) {
    bool there = false;
    for (int j = 0; j < a.K && !there; ++j) there = entry_there(a, r * a.K + j);
    n += there;
  }
  return block_sum<NT>((double)n, dl);
}
__global__ void __launch_bounds__(256) distill_count(DistillArgs a, uint32_t* count) {
  __shared__ double dl[4];
  const int64_t part = (a.R + gridDim.x - 1) / gridDim.x, first = min(a.R, (int64_t)blockIdx.x * part);
  const double n = count_rows<256>(a, first, min(a.R, first + part), dl);
  if (threadIdx.x == 0) count[blockIdx.x] = (uint32_t)n;
}

// exp(x) for x <= 0: zero where the result is no normal number (a class of such a weight is 2^-126
// of the largest at most), NaN for NaN.
__device__ __forceinline__ float exp_weight(float x) {
  const float e = exp_f32_in_range(fmaxf(x, -87.0f));
  return x != x ? x : x < -87.0f ? 0.0f : e;
}

template <int NT, int V>  // V == 0: the row does not fit, and is read again for each step
__global__ void __launch_bounds__(NT) distill_rows(DistillArgs a) {
  constexpr int NW = NT / 64;
  extern __shared__ double entries[];  // K: p; then K indexes
  __shared__ double red[3][NW];
  __shared__ float fm[2][NW];
  __shared__ int found[NW];
  int* index = reinterpret_cast<int*>(entries + a.K);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  float scale = 0.0f;
  if (a.grad != nullptr) {
    double n = 0.0;
    if (a.count == nullptr) n = count_rows<NT>(a, 0, a.R, red[0]);
    else
      for (int i = 0; i < a.parts; ++i) n += (double)a.count[i];
    scale = (float)(a.scale / n);
  }
  const int C = (int)a.C;
  for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
    const float* row = a.z + r * a.C;
    float* out = a.grad != nullptr ? a.grad + r * a.C : nullptr;
    const RowGroups view(row, C);
    // the entries: their number, the largest logit
    __syncthreads();  // the last row's entries have been read
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
      if (there) mt = fmaxf(mt, t);  // (a NaN makes the sums NaN)
    }
    any = wave_or(any);
    if (lane == 0) found[w] = any;
    __syncthreads();
    any = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) any |= found[i];
    if (!any) {
      if (threadIdx.x == 0) a.row_loss[r] = NO_LOSS;
      if (out != nullptr)
        for (int q = threadIdx.x; q < view.groups; q += NT) view.store(out, q, make_float4(0.f, 0.f, 0.f, 0.f));
      continue;
    }
    // largest values
    float4 v[V > 0 ? V : 1];
    float m = -INFINITY;
    if constexpr (V > 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int q = threadIdx.x + i * NT;
        v[i] = q < view.groups ? view.load(row, q, -INFINITY)
                               : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) m = fmaxf(m, fmaxf(fmaxf(v[i].x, v[i].y), fmaxf(v[i].z, v[i].w)));
    } else {
      for (int q = threadIdx.x; q < view.groups; q += NT) {
        const float4 x = view.load(row, q, -INFINITY);
        m = fmaxf(m, fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)));
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      m = fmaxf(m, __shfl_xor(m, o, 64));
      mt = fmaxf(mt, __shfl_xor(mt, o, 64));
    }
    if (lane == 0) { fm[0][w] = m; fm[1][w] = mt; }
    __syncthreads();
    m = fm[0][0];
    mt = fm[1][0];
#pragma unroll
    for (int i = 1; i < NW; ++i) { m = fmaxf(m, fm[0][i]); mt = fmaxf(mt, fm[1][i]); }
    // sums: of exp(z - m), of e = exp(t - mt), of e (log p - log q) but for the sums' logarithms
    double s[3] = {0.0, 0.0, 0.0};
    if constexpr (V > 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[i].x = exp_weight((v[i].x - m) * a.inv_T);
        v[i].y = exp_weight((v[i].y - m) * a.inv_T);
        v[i].z = exp_weight((v[i].z - m) * a.inv_T);
        v[i].w = exp_weight((v[i].w - m) * a.inv_T);
        s[0] += ((double)v[i].x + (double)v[i].y) + ((double)v[i].z + (double)v[i].w);
      }
    } else {
      for (int q = threadIdx.x; q < view.groups; q += NT) {
        const float4 x = view.load(row, q, -INFINITY);
        s[0] += ((double)exp_weight((x.x - m) * a.inv_T) + (double)exp_weight((x.y - m) * a.inv_T)) +
                ((double)exp_weight((x.z - m) * a.inv_T) + (double)exp_weight((x.w - m) * a.inv_T));
      }
    }
    for (int j = threadIdx.x; j < a.K; j += NT) {
      double e = 0.0;
      if (index[j] >= 0) {
        const double t = ((double)a.t[r * a.K + j] - (double)mt) * a.inv_T64;
        e = exp(t);
        const double z = ((double)row[index[j]] - (double)m) * a.inv_T64;
        s[1] += e;
        if (e != 0.0) s[2] += e * (t - z);
      }
      entries[j] = e;
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) s[k] = wave_sum(s[k]);
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < 3; ++k) red[k][w] = s[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      s[k] = red[k][0];
#pragma unroll
      for (int i = 1; i < NW; ++i) s[k] += red[k][i];
    }
    if (threadIdx.x == 0) {
      const float loss = (float)(s[2] / s[1] - log(s[1]) + log(s[0]));
      a.row_loss[r] = loss == 0.0f ? 0.0f : loss;
    }
    if (out == nullptr) continue;
    const float inv = (float)(1.0 / s[0]);
    if constexpr (V > 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int q = threadIdx.x + i * NT;
        if (q < view.groups)
          view.store(out, q, make_float4((v[i].x * inv) * scale, (v[i].y * inv) * scale, (v[i].z * inv) * scale,
                                         (v[i].w * inv) * scale));
      }
    } else {
      for (int q = threadIdx.x; q < view.groups; q += NT) {
        const float4 x = view.load(row, q, -INFINITY);
        view.store(out, q, make_float4((exp_weight((x.x - m) * a.inv_T) * inv) * scale,
                                       (exp_weight((x.y - m) * a.inv_T) * inv) * scale,
                                       (exp_weight((x.z - m) * a.inv_T) * inv) * scale,
                                       (exp_weight((x.w - m) * a.inv_T) * inv) * scale));
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores above precede those below
    __syncthreads();
    for (int j = threadIdx.x; j < a.K; j += NT) {
      const int mine = index[j];
      if (mine < 0) continue;
      double p = 0.0;
      for (int i = 0; i < a.K; ++i) p += index[i] == mine ? entries[i] : 0.0;
      const double q = (double)exp_weight((row[mine] - m) * a.inv_T) / s[0];
      out[mine] = (float)(q - p / s[1]) * scale;
    }
  }
}

// The loss: binary64 sum of the row losses, over the number of rows that have one.
__global__ void __launch_bounds__(1024) distill_finish(const float* __restrict__ row_loss, int64_t R, double T2,
                                                       float* loss) {
  __shared__ double ds[16], dn[16];
  double s = 0.0, n = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < R; i += 1024) {
    const float v = row_loss[i];
    s += (double)v;
    n += __float_as_uint(v) == 0x80000000u ? 0.0 : 1.0;
  }
  s = wave_sum(s);
  n = wave_sum(n);
  if ((threadIdx.x & 63) == 0) {
    ds[threadIdx.x >> 6] = s;
    dn[threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; ++i) {
    s += ds[i];
    n += dn[i];
  }
  loss[0] = (float)(s * T2 / n);
}

constexpr int64_t COUNT_ROWS = 1024;  // rows that each workgroup counts by itself
constexpr int COUNT_PARTS = 64;

template <int NT, int V>
void launch_rows(const DistillArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((distill_rows<NT, V>), dim3((unsigned)std::min<int64_t>(a.R, 1 << 20)), dim3(NT), 12 * a.K, s, a);
}

}  // namespace

int64_t distill_scratch_bytes(int64_t R) { return 4 * ((R + 3) / 4 * 4) + 4 * COUNT_PARTS; }

hipError_t launch_distill(const DistillParams& p, void* scratch, uint32_t* status, hipStream_t s) {
  if (p.R <= 0) return hipSuccess;
  DistillArgs a{};
  a.z = p.logits;
  a.index = p.index;
  a.t = p.teacher;
  a.grad = p.grad;
  a.row_loss = static_cast<float*>(scratch);
  a.status = status;
  a.R = p.R;
  a.C = p.C;
  a.K = (int)p.K;
  a.is64 = p.is64;
  a.inv_T = (float)(1.0 / (double)p.T);
  a.inv_T64 = 1.0 / (double)p.T;
  a.scale = (double)p.g * (double)p.T;
  if (p.grad != nullptr && p.R > COUNT_ROWS) {
    uint32_t* count = reinterpret_cast<uint32_t*>(a.row_loss + (p.R + 3) / 4 * 4);
    hipLaunchKernelGGL(distill_count, dim3(COUNT_PARTS), dim3(256), 0, s, a, count);
    a.count = count;
    a.parts = COUNT_PARTS;
  }
  if (p.C <= 256 * 4 - 4) launch_rows<256, 1>(a, s);
  else if (p.C <= 256 * 4 * 4 - 4) launch_rows<256, 4>(a, s);
  else if (p.C <= 256 * 4 * 8 - 4) launch_rows<256, 8>(a, s);
  else if (p.C <= 512 * 4 * 8 - 4) launch_rows<512, 8>(a, s);
  else if (p.C <= 512 * 4 * 16 - 4) launch_rows<512, 16>(a, s);
  else if (p.C <= 1024 * 4 * 16 - 4) launch_rows<1024, 16>(a, s);
  else launch_rows<1024, 0>(a, s);
  hipLaunchKernelGGL(distill_finish, dim3(1), dim3(1024), 0, s, (const float*)a.row_loss, p.R,
                     (double)p.T * (double)p.T, p.loss);
  return hipGetLastError();
}

}  // namespace shk
