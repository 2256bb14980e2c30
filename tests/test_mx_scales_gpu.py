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
