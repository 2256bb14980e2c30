"""How exact the microscaled products are, at shapes of every kernel, with bounds that do not grow
with the depth: a lost part of an operand or a narrow sum stands out by orders of magnitude.

u = 2^-24 is half a unit in the last place of binary32, relative to the value. An addition is off by
at most u when it is rounded and 2 u when it is cut off."""
import numpy as np
import pytest

from tests import mx_oracle as mx
from tests.test_mx_gpu import U, gpu_mx_gemm, gpu_mx_linear

pytestmark = pytest.mark.gpu

# by the rule of mx_linear.hip: few rows that encode X themselves, few rows, tiles of 128 whole and
# split along K, tiles of 256, tiles of 256 ahead of 128
LINEAR_SHAPES = [(1, 300, 1000), (12, 70, 500), (40, 300, 700), (1030, 1031, 1033), (300, 1100, 4100),
                 (4000, 3001, 200), (4400, 4000, 100)]
PAIRS = [(x, w) for x in mx.FORMATS for w in mx.FORMATS]


@pytest.mark.parametrize("x_format,w_format", PAIRS)
@pytest.mark.parametrize("shape", LINEAR_SHAPES, ids=str)
def test_two_blocks_far_apart_add_in_binary32(ctx, shape, x_format, w_format):
    """A row of X has two values, in neighbouring blocks that one instruction contracts, 14 to 20
    binades apart: each result is one addition of two exact products (at most four significant bits
    by four), here allowed to be cut off twice."""
    M, N, K = shape
    rng = np.random.default_rng(M + K)
    X = np.zeros((M, K), np.float32)
    pair = rng.integers(0, K // 64, M) * 64
    k1, k2 = pair + rng.integers(0, 32, M), pair + rng.integers(32, 64, M)
    swap = rng.random(M) < 0.5
    k1, k2 = np.where(swap, k2, k1), np.where(swap, k1, k2)
    rows = np.arange(M)
    X[rows, k1] = rng.standard_normal(M)
    X[rows, k2] = rng.standard_normal(M) * np.exp2(-rng.integers(14, 21, M))
    codes, scales, W = mx.stored(rng.standard_normal((N, K)), w_format)
    Xq = mx.stored(X, x_format)[2]
    got = gpu_mx_linear(ctx, X, (codes, scales), None, M, N, K, x_format, w_format, None)
    p1, p2 = Xq[rows, k1][:, None] * W.T[k1], Xq[rows, k2][:, None] * W.T[k2]
    assert (np.abs(got - (p1 + p2)) <= 4 * U * (np.abs(p1) + np.abs(p2))).all()


@pytest.mark.parametrize("x_format,w_format", PAIRS)
@pytest.mark.parametrize("shape", LINEAR_SHAPES, ids=str)
def test_sums_of_few_bits_are_exact(ctx, shape, x_format, w_format):
    """Values that every format holds, 6 and 0.5 most of them: products are multiples of 0.25 up to
    36, a sum of K <= 4100 of them has at most 144 K < 2^20 such units, so no addition in binary32
    rounds, whatever the order."""
    M, N, K = shape
    rng = np.random.default_rng(N + K)
    values = np.array([6.0, 6.0, 0.5, 0.5, -6.0, -0.5, 1.0, -1.5, 2.0, 3.0, -4.0, 0.0])
    X, Wide = rng.choice(values, (M, K)), rng.choice(values, (N, K))
    X[:, ::32] = 6.0  # (each block's scale follows its largest value)
    Wide[:, ::32] = 6.0
    codes, scales, W = mx.stored(Wide, w_format)
    assert np.array_equal(W, Wide) and np.array_equal(mx.stored(X, x_format)[2], X)
    got = gpu_mx_linear(ctx, X.astype(np.float32), (codes, scales), None, M, N, K, x_format, w_format, None)
    assert np.array_equal(got, X @ W.T)


# by the rule of mx_gemm.hip: one and two row fragments from registers, tiles of 128 whole and split
# along K, tiles of 256, tiles of 256 ahead of 128
GEMM_SHAPES = [(50, 200, 90), (700, 710, 720), (2000, 2000, 300), (1000, 1100, 1500), (4000, 4050, 90),
               (4600, 4000, 90)]


@pytest.mark.parametrize("trans_a", [False, True])
@pytest.mark.parametrize("format", mx.FORMATS)
@pytest.mark.parametrize("shape", GEMM_SHAPES, ids=str)
def test_every_part_of_the_wide_operand_counts(ctx, shape, format, trans_a):
    """One nonzero a row of A: each result is a single product, the sum of its exact parts (three,
    each addition cut off at worst: 6 u). Without the last part it would be off by up to 2^-16."""
    M, N, K = shape
    rng = np.random.default_rng(M + N + K)
    A, at = np.zeros((M, K), np.float32), rng.integers(0, K, M)
    A[np.arange(M), at] = rng.standard_normal(M) * np.exp2(rng.integers(-60, 60, M))
    codes, scales, B = mx.stored(rng.standard_normal((K, N)), format)
    got = gpu_mx_gemm(ctx, A.T if trans_a else A, codes, scales, M, N, K, format, trans_a)
    want = A[np.arange(M), at].astype(np.float64)[:, None] * B[at]
    assert (np.abs(got - want) <= 6 * U * np.abs(want)).all()
