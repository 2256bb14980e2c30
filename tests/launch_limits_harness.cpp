// Host build of synaptik_amd/csrc/launch_limits.h: every launch it shapes has fewer than 2^32 threads
// along a grid's first dimension and reaches every unit of work. Prints "ok" or the first failure.
#include <cstdio>

#include "../synaptik_amd/csrc/launch_limits.h"

using namespace shk;

static int fail(const char* what, int64_t a, int64_t b, int64_t c) {
  printf("FAIL %s %lld %lld %lld\n", what, (long long)a, (long long)b, (long long)c);
  return 1;
}

// 32 k of every 64 rows and of every 256 columns, each unit in one workgroup's stride
static int check_pack(int64_t M, int64_t N, int64_t K) {
  const int64_t blocks = mx_pack_blocks(M, N), units = mx_pack_units(M, N, K), groups = mx_pack_groups(units);
  if (blocks * 64 < M || groups < 1 || groups > units) return fail("pack extents", M, N, K);
  if (groups * PACK_THREADS > LAUNCH_THREADS) return fail("pack threads", M, N, K);
  if (units % blocks != 0 || units / blocks * 32 < K || (units / blocks - 1) * 32 >= K) return fail("pack depth", M, N, K);
  // workgroup g takes g, g + groups, ...: every unit up to the last once
  const int64_t last = units - 1, g = last % groups;
  if (g + last / groups * groups != last) return fail("pack stride", M, N, K);
  return 0;
}

// pieces of COLSUM_COLS columns, COLSUM_THREADS for every COLSUM_WIDTH of a piece
static int check_colsum(int64_t N) {
  int64_t reached = 0;
  for (int64_t n = 0; n < N; n += COLSUM_COLS) {
    const int64_t cols = N - n < COLSUM_COLS ? N - n : COLSUM_COLS;
    if (colsum_groups(cols) * COLSUM_THREADS > LAUNCH_THREADS) return fail("column sums' threads", N, n, cols);
    if (colsum_groups(cols) * COLSUM_WIDTH < cols) return fail("column sums' width", N, n, cols);
    reached += cols;
  }
  return reached == N ? 0 : fail("column sums' pieces", N, reached, 0);
}

int main() {
  if (LAUNCH_THREADS != 0xffffffffll) return fail("threads", LAUNCH_THREADS, 0, 0);
  const int64_t depths[] = {1, 15, 16, 31, 32, 33, 4096, 700000, 179000000, 1ll << 30, (1ll << 31) - 1};
  const int64_t extents[] = {1, 63, 64, 65, 129, 4096, 1 << 20};
  for (int64_t K : depths)
    for (int64_t M : extents)
      for (int64_t N : extents)
        if (check_pack(M, N, K)) return 1;
  const int64_t widths[] = {1, 65, (1ll << 29) + 1, (1ll << 30) - 64, (1ll << 30) - 63, (1ll << 31) - 257, 1ll << 34};
  for (int64_t N : widths)
    if (check_colsum(N)) return 1;
  // from here on one launch does not do
  if (colsum_groups((1ll << 30) - 63) * COLSUM_THREADS <= LAUNCH_THREADS) return fail("wide", 1ll << 30, 0, 0);
  // the shape whose units alone fill more than a launch: 2^32 threads, one unit each
  if (mx_pack_units(65, 129, 179000000) * PACK_THREADS <= LAUNCH_THREADS) return fail("deep", 65, 129, 179000000);
  // one that a device test runs takes more than one unit a workgroup
  if (mx_pack_units(65, 129, 700001) <= PACK_GROUPS) return fail("two rounds", 65, 129, 700001);
  printf("ok\n");
  return 0;
}
