// Y = act(X . W^T + b) of microscaled weights W [N, K] (mx.h) and binary32 activations X, encoded
// here.
#include <algorithm>

#include "mx.h"

namespace shk {
namespace {

int64_t pad256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace

int64_t mx_linear_scratch_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0) return 0;
  const int64_t G = mx_groups(K);
  return pad256(M * G * 128) + pad256(M * G * 4) + pad256(4 * M * K) + pad256(4 * N * K) +
         4 * gemm_workspace_floats(M, N, K);
}

hipError_t launch_mx_linear(const MxLinearParams& p, void* scratch, hipStream_t s) {
  if (p.M <= 0 || p.N <= 0) return hipSuccess;
  const int64_t G = mx_groups(p.K);
  char* at = static_cast<char*>(scratch);
  auto take = [&](int64_t bytes) {
    char* r = at;
    at += pad256(bytes);
    return r;
  };
  uint8_t* codes = reinterpret_cast<uint8_t*>(take(p.M * G * 128));
  uint8_t* scales = reinterpret_cast<uint8_t*>(take(p.M * G * 4));
  float* x = reinterpret_cast<float*>(take(4 * p.M * p.K));
  float* w = reinterpret_cast<float*>(take(4 * p.N * p.K));
  hipError_t e = launch_mx_encode(p.X, p.ldx, codes, scales, p.M, p.K, p.x_format, 0, s);
  if (e == hipSuccess) e = launch_mx_decode(codes, scales, x, p.K, p.M, p.K, p.x_format, s);
  if (e == hipSuccess) e = launch_mx_decode(p.codes, p.scales, w, p.K, p.N, p.K, p.w_format, s);
  if (e != hipSuccess) return e;
  GemmParams g{};
  g.A = x; g.B = w; g.C = p.Y; g.bias = p.bias;
  g.M = p.M; g.N = p.N; g.K = p.K;
  g.lda = p.K; g.ldb = p.K; g.ldc = p.ldy;
  g.transB = 1;
  g.act = p.act;
  return launch_gemm(g, reinterpret_cast<float*>(at), s);
}

}  // namespace shk
