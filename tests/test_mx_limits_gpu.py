"""Microscaled steps at extents where a launch would exceed what a grid holds, or where its work goes
round more than once (synaptik_amd/csrc/launch_limits.h)."""
import numpy as np
import pytest

from synaptik_amd.program import ProgramBuilder
from tests.gpu_helpers import run_program

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("trans_a", [False, True])
def test_product_deeper_than_one_round_of_packing(ctx, trans_a):
    """65 x 129 by 700001: three units of packing for each 32 k, more than a launch has workgroups.
    Whole numbers of at most two on both sides: every sum is below 2^24, so the result is exact."""
    M, N, K = 65, 129, 700001
    rng = np.random.default_rng(0)
    A = rng.integers(-2, 3, (M, K)).astype(np.float32)
    nibble = np.zeros((K, 256), np.uint8)  # e2m1 codes of 0, 1, 2, -1, -2; zero behind column N
    nibble[:, :N] = rng.choice(np.array([0, 2, 4, 10, 12], np.uint8), (K, N))
    value = np.zeros(16, np.float32)
    value[[2, 4, 10, 12]] = 1, 2, -1, -2
    codes = nibble[:, 0::2] | (nibble[:, 1::2] << 4)
    scales = np.full((K, 8), 127, np.uint8)
    pb = ProgramBuilder()
    a, B, c = pb.input(M * K), pb.mx_tensor(K, N, "e2m1", "input"), pb.output(M * N)
    pb.mx_gemm(a, B, c, M, N, K, format="e2m1", trans_a=trans_a)
    (got,) = run_program(ctx, pb, [A.T if trans_a else A, codes, scales], [c])
    want = A @ value[nibble[:, :N]]
    assert np.array_equal(got.reshape(M, N), want)
