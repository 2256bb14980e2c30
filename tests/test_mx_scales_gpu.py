"""Products of hand-made microscaled tensors: every scale byte below 255, far outside what encoding
gives, at shapes of every kernel.

What a code stands for counts exactly in a product as long as it is zero or of a magnitude from 2^-126
to 2^128, the normal binary32 range: those values are bfloat16 numbers, and a code has at most four
significant bits. A smaller one counts as itself or with an error below 2^-126 (subnormal bfloat16
values are rounded, and read as zeros by the matrix cores)."""
import numpy as np
import pytest

from tests import mx_oracle as mx
from tests.test_mx_gpu import gpu_mx_gemm, gpu_mx_linear
from tests.test_mx_precision_gpu import GEMM_SHAPES, LINEAR_SHAPES, PAIRS

pytestmark = pytest.mark.gpu
LEAST = 2.0 ** -126


def hand_made(rng, R, C, format, scale):
    """(packed codes, scales, values) of random codes under the scale bytes `scale` [R, 4 G]; a code
    that would stand for 2^128 or more is zero."""
    finite = np.arange(16)
    if format != "e2m1":
        n = len(mx.table(format))
        finite = np.concatenate([np.arange(n), 128 + np.arange(n)])
    code = rng.choice(finite, (R, 128 * mx.groups(C))).astype(np.uint8)
    code[np.abs(mx.values(code, scale, code.shape[1], format)) >= 2.0 ** 128] = 0
    code[:, C:] = 0
    return mx.pack(code, format), scale.astype(np.uint8), mx.values(code, scale, C, format)


@pytest.mark.parametrize("trans_a", [False, True])
@pytest.mark.parametrize("format", mx.FORMATS)
@pytest.mark.parametrize("shape", GEMM_SHAPES, ids=str)
def test_wide_products_under_every_scale(ctx, shape, format, trans_a):
    """One power of two a row of A, which brings a row of B back into range: exact products."""
    M, N, K = shape
    rng = np.random.default_rng(M + K)
    s = np.concatenate([np.arange(0, 255, 3)[:K], rng.integers(0, 255, max(0, K - 85))])
    scale = np.repeat(s[:, None], 4 * mx.groups(N), axis=1)
    codes, scales, B = hand_made(rng, K, N, format, scale)
    A, at = np.zeros((M, K), np.float32), np.arange(M) % K
    A[np.arange(M), at] = np.ldexp(1.0, np.clip(127 - s[at], -126, 127))
    got = gpu_mx_gemm(ctx, A.T if trans_a else A, codes, scales, M, N, K, format, trans_a)
    a = A[np.arange(M), at].astype(np.float64)[:, None]
    want, small = a * B[at], np.abs(B[at]) < LEAST
    assert np.array_equal(got[~small], want[~small])
    assert (np.abs(got - want) <= a * LEAST)[small].all()
    assert ((0 < np.abs(B)) & (np.abs(B) < LEAST)).any()


@pytest.mark.parametrize("x_format,w_format", PAIRS)
@pytest.mark.parametrize("shape", LINEAR_SHAPES, ids=str)
def test_linear_layers_under_every_scale(ctx, shape, x_format, w_format):
    """One power of two a row of X, which every format holds. Products in the normal range are exact
    where the weight is; one below it may be lost, one above it is an infinity."""
    M, N, K = shape
    rng = np.random.default_rng(N)
    codes, scales, W = hand_made(rng, N, K, w_format, rng.integers(0, 255, (N, 4 * mx.groups(K))))
    X, at = np.zeros((M, K), np.float32), rng.integers(0, K, M)
    X[np.arange(M), at] = np.ldexp(1.0, rng.integers(-100, 128, M))
    assert np.array_equal(mx.stored(X, x_format)[2], X)
    got = gpu_mx_linear(ctx, X, (codes, scales), None, M, N, K, x_format, w_format, None)
    x, w = X[np.arange(M), at].astype(np.float64)[:, None], W.T[at]
    want = x * w
    exact = (np.abs(w) >= LEAST) & (np.abs(want) >= LEAST) & (np.abs(want) < 2.0 ** 128)
    assert np.array_equal(got[exact], want[exact])
    small = (np.abs(w) < LEAST) & (np.abs(want) >= LEAST)
    assert (np.abs(got - want) <= x * LEAST)[small].all()
    assert (np.abs(got)[np.abs(want) < LEAST] <= LEAST).all()
    assert np.isinf(got[np.abs(want) >= 2.0 ** 128]).all()


@pytest.mark.parametrize("trans_a", [False, True])
@pytest.mark.parametrize("shape", GEMM_SHAPES, ids=str)
def test_an_infinite_code_reaches_its_column_alone(ctx, shape, trans_a):
    """e5m2 has infinities. The wide operand goes to the products in three parts, of which those that
    are zero make NaN of an infinite code, so a result is NaN where a binary32 product would be
    infinite: not finite in its whole column, and nowhere else. The last row of B is one that the
    kernels may read again behind the depth."""
    M, N, K = shape
    rng = np.random.default_rng(K)
    # small whole numbers: sums below 2^24, exact in binary32
    A = rng.integers(-3, 4, (M, K)).astype(np.float32)
    B = rng.integers(-3, 4, (K, N)).astype(np.float64)
    columns = [1, N // 2, N - 1]
    B[K // 2, 1], B[K - 1, N // 2], B[0, N - 1] = np.inf, -np.inf, np.inf
    codes, scales, back = mx.stored(B, "e5m2")
    assert np.array_equal(back, B)
    got = gpu_mx_gemm(ctx, A.T if trans_a else A, codes, scales, M, N, K, "e5m2", trans_a)
    assert not np.isfinite(got[:, columns]).any()
    ok = np.setdiff1d(np.arange(N), columns)
    assert np.array_equal(got[:, ok], A.astype(np.float64) @ B[:, ok])


@pytest.mark.parametrize("x_format", mx.FORMATS)
@pytest.mark.parametrize("shape", LINEAR_SHAPES, ids=str)
def test_an_infinite_weight_is_an_infinity(ctx, shape, x_format):
    """In a linear layer each product is one exact term: an infinite code against values that are not
    zero gives an infinity of the right sign in its column, and touches no other."""
    M, N, K = shape
    rng = np.random.default_rng(M)
    X = (rng.integers(1, 4, (M, K)) * rng.choice([-1, 1], (M, K))).astype(np.float32)
    W = rng.integers(-3, 4, (N, K)).astype(np.float64)
    W[3, K - 1], W[N - 1, 0] = np.inf, -np.inf
    codes, scales, back = mx.stored(W, "e5m2")
    assert np.array_equal(back, W) and np.array_equal(mx.stored(X, x_format)[2], X)
    got = gpu_mx_linear(ctx, X, (codes, scales), None, M, N, K, x_format, "e5m2", None)
    assert np.array_equal(got[:, 3], np.sign(X[:, K - 1]) * np.inf)
    assert np.array_equal(got[:, N - 1], np.sign(X[:, 0]) * -np.inf)
    ok = np.setdiff1d(np.arange(N), [3, N - 1])
    assert np.array_equal(got[:, ok], X.astype(np.float64) @ W[ok].T)
