"""Microscaled tensors on the GPU against 64-bit forms of the definition (tests/mx_oracle.py).

Tolerances. u = 2^-24 is half a unit in the last place of binary32, relative to the value. A sum
of n products in binary32, in any order, is off by at most (n + 1) u sum |a b| when each addition
is rounded to nearest and 2 (n + 1) u sum |a b| when it is cut off, which is allowed for here. A
product of a binary32 value and a code may be summed in three exact parts (n = 3 K)."""
import numpy as np
import pytest

from synaptik_amd.native import HipBuffer, HipInvalidArgument, HipProgram
from synaptik_amd.program import ProgramBuilder
from tests import mx_oracle as mx
from tests.gpu_helpers import run_program

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def wide_values(rng, R, C):
    """Binary32 values over many binades, with everything that a block can meet."""
    x = (rng.standard_normal((R, C)) * np.exp2(rng.integers(-20, 20, (R, 1)))).astype(np.float32)
    flat = x.reshape(-1)
    special = np.array([0.0, -0.0, np.inf, -np.inf, np.nan, 1e-45, -1e-45, 1.1e-38, 3.4028235e38,
                        448.0, 449.0, 464.0, 57344.0, 6.0, 7.0, 2.5, 0.25, 1.75, 2.0 ** -10,
                        3 * 2.0 ** -10], np.float32)
    at = rng.random(flat.size) < 0.02
    flat[at] = rng.choice(special, at.sum())
    if R > 3:
        x[1] = 0.0
        x[2] = np.nan
        x[3, :] = rng.choice(special[5:7], C)
    return x


def put(ctx, array):
    a = np.ascontiguousarray(array)
    return ctx.upload(a if a.size else np.zeros(1, a.dtype))


# ---- storing ----
SHAPES = [(1, 1), (1, 31), (1, 32), (2, 33), (1, 1024), (3, 127), (5, 128), (4, 129), (7, 1021),
          (131, 300), (2, 4100), (2048, 2049)]


@pytest.mark.parametrize("format", mx.FORMATS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_encoding_and_restoring_are_exact(ctx, shape, format):
    R, C = shape
    rng = np.random.default_rng(R * 131 + C)
    x = wide_values(rng, R, C)
    for keep in ((False,) if format == "e2m1" else (False, True)):
        pb = ProgramBuilder()
        sx = pb.input(R * C)
        out = pb.mx_tensor(R, C, format, "output")
        y = pb.output(R * C)
        pb.mx_encode(sx, out, R, C, format=format, keep_nonzero=keep)
        pb.mx_decode(out, y, R, C, format=format)
        codes, scales, back = run_program(ctx, pb, [x], [*out, y])
        want_codes, want_scales, want = mx.stored(x, format, keep)
        assert np.array_equal(scales.reshape(R, -1), want_scales)
        assert np.array_equal(codes.reshape(R, -1), want_codes)
        assert np.array_equal(back.reshape(R, C).astype(np.float64), want, equal_nan=True)
        if keep:
            assert np.array_equal(want == 0, x == 0)


@pytest.mark.parametrize("format", mx.FORMATS)
def test_encoding_rounds_ties_to_even(ctx, format):
    """Every pair of neighbouring codes' middle, and the floats beside it, of both signs."""
    t = mx.table(format)
    mid = (t[1:] + t[:-1]) / 2
    v = np.concatenate([mid, np.nextafter(mid.astype(np.float32), np.float32(0)),
                        np.nextafter(mid.astype(np.float32), np.float32(np.inf)), t]).astype(np.float32)
    v = np.concatenate([v, -v])
    # a block of 31 of them under the format's largest value, so that the scale is one
    n = -(-v.size // 31)
    rows = np.zeros((n, 32), np.float32)
    rows[:, 0] = t[-1]
    for i, part in enumerate(np.array_split(v, n)):
        rows[i, 1:1 + part.size] = part
    pb = ProgramBuilder()
    sx = pb.input(rows.size)
    out = pb.mx_tensor(n, 32, format, "output")
    pb.mx_encode(sx, out, n, 32, format=format)
    codes, scales = run_program(ctx, pb, [rows], list(out))
    want_codes, want_scales, _ = mx.stored(rows, format)
    assert np.array_equal(scales.reshape(n, -1), want_scales) and (want_scales[:, 0] == 127).all()
    assert np.array_equal(codes.reshape(n, -1), want_codes)


@pytest.mark.parametrize("format", mx.FORMATS)
def test_restoring_every_code_under_every_scale(ctx, format):
    """Hand-made tensors: every code under every scale byte, the extreme ones included."""
    half = 8 if format == "e2m1" else 128
    code = np.tile(np.arange(2 * half), 256 // (2 * half)).astype(np.uint8)
    code = np.tile(code, (256, 1))
    scales = np.tile(np.arange(256, dtype=np.uint8)[:, None], (1, 8))
    pb = ProgramBuilder()
    X = pb.mx_tensor(256, 256, format, "input")
    y = pb.output(256 * 256)
    pb.mx_decode(X, y, 256, 256, format=format)
    (got,) = run_program(ctx, pb, [mx.pack(code, format), scales], [y])
    with np.errstate(over="ignore"):
        want = mx.values(code, scales, 256, format).astype(np.float32)
    assert np.array_equal(got.reshape(256, 256), want, equal_nan=True)


def test_rows_further_apart_than_their_width(ctx):
    R, C, ldx, ldy = 37, 203, 211, 205
    rng = np.random.default_rng(3)
    x = rng.standard_normal((R, ldx)).astype(np.float32)
    pb = ProgramBuilder()
    sx, y = pb.input((R - 1) * ldx + C), pb.input((R - 1) * ldy + C, inout=True)
    t = pb.mx_tensor(R, C, "e4m3")
    pb.mx_encode(sx, t, R, C, ldx=ldx)
    pb.mx_decode(t, y, R, C, ldy=ldy)
    prog = HipProgram(ctx, pb.image())
    bx = ctx.upload(x.reshape(-1)[:(R - 1) * ldx + C])
    by = ctx.upload(np.full((R - 1) * ldy + C, 7.0, np.float32))
    prog.run([bx, by], [])
    got = np.concatenate([by.download(), np.full(ldy - C, 7.0, np.float32)]).reshape(R, ldy)
    assert np.array_equal(got[:, :C], mx.stored(x[:, :C], "e4m3")[2].astype(np.float32))
    assert (got[:, C:] == 7.0).all()
    prog.close()


# ---- the activation's gradient ----
@pytest.mark.parametrize("act", [None, "relu", "tanh", "sigmoid"])
@pytest.mark.parametrize("shape,format", [((1, 1), "e4m3"), ((2, 5), "e5m2"), ((16, 256), "e4m3"),
                                          ((17, 257), "e2m1"), ((300, 130), "e4m3"),
                                          ((64, 70), "e4m3"), ((65, 70), "e4m3"), ((1, 3001), "e5m2"), ((70000, 3), "e4m3"),
                                          ((1000, 1100), "e4m3"), ((1025, 300), "e5m2"), ((1500, 513), "e4m3"),
                                          ((5000, 600), "e5m2")], ids=str)
def test_activation_gradient_from_a_checkpoint(ctx, shape, format, act):
    R, C = shape
    rng = np.random.default_rng(R + C)
    y = mx.activate(act, rng.standard_normal((R, C)) * 2)
    dy = rng.standard_normal((R, C)).astype(np.float32)
    codes, scales, back = mx.stored(y, format)
    back = back.astype(np.float32)
    one = np.float32(1)
    want = {None: lambda: dy, "relu": lambda: np.where(back > 0, dy, np.float32(0)),
            "tanh": lambda: dy * (one - back * back),
            "sigmoid": lambda: (dy * back) * (one - back)}[act]()
    for with_sum in (False, True):
        pb = ProgramBuilder()
        sdy, Y = pb.input(R * C), pb.mx_tensor(R, C, format, "input")
        dz, db = pb.output(R * C), pb.output(C) if with_sum else None
        pb.mx_act_grad(sdy, Y, dz, R, C, act=act, format=format, colsum=db)
        got = run_program(ctx, pb, [dy, codes, scales], [dz] + ([db] if with_sum else []))
        assert np.array_equal(got[0].reshape(R, C), want)  # the same operations in binary32
        if with_sum:  # sums in binary64, rounded once
            exact = want.astype(np.float64).sum(0)
            room = U * np.abs(exact) + 2.0 ** -50 * np.abs(want).astype(np.float64).sum(0)
            assert (np.abs(got[1] - exact) <= room).all()


def test_activation_gradient_in_place_and_with_strides(ctx):
    R, C, ldy = 50, 77, 90
    rng = np.random.default_rng(5)
    dy = rng.standard_normal((R, ldy)).astype(np.float32)
    codes, scales, back = mx.stored(np.maximum(rng.standard_normal((R, C)), 0), "e4m3", True)
    pb = ProgramBuilder()
    d, Y = pb.input(R * ldy, inout=True), pb.mx_tensor(R, C, "e4m3", "input")
    pb.mx_act_grad(d, Y, d, R, C, act="relu", ldy=ldy, ldz=ldy)
    prog = HipProgram(ctx, pb.image())
    buf = ctx.upload(dy)
    prog.run([buf, ctx.upload(codes), ctx.upload(scales)], [])
    got = buf.download().reshape(R, ldy)
    assert np.array_equal(got[:, :C], np.where(back > 0, dy[:, :C], np.float32(0)))
    assert np.array_equal(got[:, C:], dy[:, C:])
    prog.close()


def test_activation_gradient_of_a_very_long_row(ctx):
    """More columns than one launch of a workgroup for every 32 of them takes."""
    C = (1 << 27) + 37
    dy = np.tile(np.arange(-500, 501, dtype=np.float32), C // 1001 + 1)[:C]
    groups = -(-C // 128)
    codes = np.tile(np.arange(256, dtype=np.uint8) % 0x78, groups // 2 + 1)[:groups * 128]  # no NaN
    pb = ProgramBuilder()
    d, Y = pb.input(C), pb.mx_tensor(1, C, "e4m3", "input")
    dz, db = pb.output(C), pb.output(C)
    pb.mx_act_grad(d, Y, dz, 1, C, act="relu", colsum=db)
    got = run_program(ctx, pb, [dy, codes, np.full(groups * 4, 127, np.uint8)], [dz, db])
    want = np.where(codes[:C] > 0, dy, np.float32(0))
    assert np.array_equal(got[0], want) and np.array_equal(got[1], want)


def test_column_sums_of_no_rows_are_zero(ctx):
    pb = ProgramBuilder()
    d, Y = pb.input(0), pb.mx_tensor(0, 5, "e4m3", "input")
    dz, db = pb.output(0), pb.output(5)
    pb.mx_act_grad(d, Y, dz, 0, 5, act="relu", colsum=db)
    prog = HipProgram(ctx, pb.image())
    out = ctx.upload(np.full(5, 3.0, np.float32))
    empty = ctx.buffer(0)
    prog.run([empty, ctx.buffer(0), ctx.buffer(0)], [ctx.buffer(0), out])
    assert np.array_equal(out.download(), np.zeros(5, np.float32))
    prog.close()


# ---- products with one microscaled operand ----
def gpu_mx_gemm(ctx, A, codes, scales, M, N, K, format, trans_a, lda=None, ldc=None):
    pb = ProgramBuilder()
    a, B = pb.input(A.size), pb.mx_tensor(K, N, format, "input")
    ldc = N if ldc is None else ldc
    c = pb.input((M - 1) * ldc + N, inout=True)
    pb.mx_gemm(a, B, c, M, N, K, format=format, trans_a=trans_a, lda=lda, ldc=ldc)
    prog = HipProgram(ctx, pb.image())
    bc = ctx.upload(np.full((M - 1) * ldc + N, 77.0, np.float32))
    prog.run([put(ctx, A), put(ctx, codes), put(ctx, scales), bc], [])
    prog.close()
    got = np.concatenate([bc.download(), np.full(ldc - N, 77.0, np.float32)]).reshape(M, ldc)
    assert (got[:, N:] == 77.0).all()
    return got[:, :N]


PRODUCTS = [(1, 1, 1), (1, 5, 3), (3, 2, 40), (16, 16, 16), (33, 31, 32), (1, 1000, 700), (10, 300, 129),
            (64, 64, 64), (65, 130, 100), (128, 128, 512), (200, 10, 900), (255, 257, 333),
            (257, 513, 65), (512, 512, 512), (700, 390, 1025), (1024, 1030, 260), (130, 4100, 77),
            (1025, 1023, 1027), (2100, 1030, 33), (2000, 1100, 190), (3000, 2900, 95)]
# small tiles whole and split along K, large tiles, and large tiles ahead of small ones
LARGE_PRODUCTS = [(4100, 2100, 70), (4000, 2000, 300), (1600, 1500, 600), (4100, 2100, 200), (4000, 4050, 90), (4600, 4000, 90)]


@pytest.mark.parametrize("trans_a", [False, True])
@pytest.mark.parametrize("format,shape", [(f, s) for s in PRODUCTS for f in mx.FORMATS]
                         + [("e4m3", s) for s in LARGE_PRODUCTS], ids=str)
def test_product_of_a_microscaled_operand(ctx, shape, format, trans_a):
    M, N, K = shape
    rng = np.random.default_rng(M + 7 * N + 31 * K)
    A = (rng.standard_normal((M, K)) * np.exp2(rng.integers(-12, 12, (1, K)))).astype(np.float32)
    codes, scales, B = mx.stored(rng.standard_normal((K, N)) * np.exp2(rng.integers(-6, 6, (K, 1))),
                                 format)
    got = gpu_mx_gemm(ctx, A.T if trans_a else A, codes, scales, M, N, K, format, trans_a)
    want = A.astype(np.float64) @ B
    room = 2 * (3 * K + 1) * U * (np.abs(A).astype(np.float64) @ np.abs(B))
    assert (np.abs(got - want) <= room).all()


@pytest.mark.parametrize("trans_a", [False, True])
@pytest.mark.parametrize("size", [40, 520, 1201])
def test_product_keeps_every_bit_of_the_wide_operand(ctx, size, trans_a):
    """One nonzero a row of A: each result is a single product, off by the rounding of the few
    additions of its exact parts (three, each cut off at worst: 6 u)."""
    rng = np.random.default_rng(size)
    M = N = K = size
    A = np.zeros((M, K), np.float32)
    A[np.arange(M), rng.integers(0, K, M)] = rng.standard_normal(M) * np.exp2(rng.integers(-60, 60, M))
    codes, scales, B = mx.stored(rng.standard_normal((K, N)), "e4m3")
    got = gpu_mx_gemm(ctx, A.T if trans_a else A, codes, scales, M, N, K, "e4m3", trans_a)
    want = A.astype(np.float64) @ B
    assert (np.abs(got - want) <= 6 * U * np.abs(want)).all()


@pytest.mark.parametrize("size", [40, 520, 1201])
def test_product_of_the_smallest_wide_values(ctx, size):
    """Wide values down to the least subnormal one, against large microscaled values.

    The matrix cores read subnormal bfloat16 values as zeros. Of a wide value's three exact parts,
    each the leading eight bits of what the ones before it leave, those read as zeros are the last
    ones; the first of them is below 2^-126, so what it leads, the sum of it and the ones behind it,
    is too (2^-126 has one bit: a remainder of at least 2^-126 leads with at least 2^-126). A wide
    value therefore counts with an error below 2^-126."""
    rng = np.random.default_rng(size)
    M = N = K = size
    A = np.ldexp(rng.integers(-(1 << 24), 1 << 24, (M, K)), rng.integers(-149, -130, (M, 1))).astype(np.float32)
    codes, scales, B = mx.stored(np.ldexp(rng.standard_normal((K, N)), 100), "e4m3")
    room = 2 * (3 * K + 1) * U * (np.abs(A).astype(np.float64) @ np.abs(B)) + 2.0 ** -126 * np.abs(B).sum(0)
    for trans_a in (False, True):
        got = gpu_mx_gemm(ctx, A.T if trans_a else A, codes, scales, M, N, K, "e4m3", trans_a)
        assert (np.abs(got - A.astype(np.float64) @ B) <= room).all()


@pytest.mark.parametrize("trans_a", [False, True])
def test_products_longer_than_a_piece(ctx, trans_a):
    """More rows, and more columns, than one set of launches takes."""
    rng = np.random.default_rng(1)
    for M, N, K in (((1 << 20) + 37, 5, 6), (3, (1 << 20) + 200, 2)):
        A = rng.standard_normal((M, K)).astype(np.float32)
        codes, scales, B = mx.stored(rng.standard_normal((K, N)), "e2m1")
        got = gpu_mx_gemm(ctx, A.T if trans_a else A, codes, scales, M, N, K, "e2m1", trans_a)
        A = A.astype(np.float64)
        assert (np.abs(got - A @ B) <= 2 * (3 * K + 1) * U * (np.abs(A) @ np.abs(B))).all()


@pytest.mark.parametrize("trans_a", [False, True])
def test_product_with_strides_and_a_matrix_of_no_depth(ctx, trans_a):
    rng = np.random.default_rng(11)
    for M, N, K, pad_a, ldc in ((45, 70, 130, 9, 77), (600, 530, 520, 3, 531), (1150, 1290, 1203, 5, 1295)):
        shape = (K, M) if trans_a else (M, K)
        wide = rng.standard_normal((shape[0], shape[1] + pad_a)).astype(np.float32)
        A = wide[:, :shape[1]]
        codes, scales, B = mx.stored(rng.standard_normal((K, N)), "e5m2")
        got = gpu_mx_gemm(ctx, wide, codes, scales, M, N, K, "e5m2", trans_a, lda=wide.shape[1], ldc=ldc)
        A = (A.T if trans_a else A).astype(np.float64)
        assert (np.abs(got - A @ B) <= 2 * (3 * K + 1) * U * (np.abs(A) @ np.abs(B))).all()
    empty = np.zeros((0,), np.float32)
    got = gpu_mx_gemm(ctx, empty, empty.astype(np.uint8), empty.astype(np.uint8), 5, 6, 0, "e4m3", trans_a)
    assert np.array_equal(got, np.zeros((5, 6), np.float32))


def test_product_of_rows_far_apart(ctx):
    """Rows of A 64 MiB apart: a wave's 32 lie further than a 32-bit offset reaches."""
    M, N, K, lda = 20, 70, 100, (1 << 24) + 8
    rng = np.random.default_rng(6)
    A = rng.standard_normal((M, K)).astype(np.float32)
    codes, scales, B = mx.stored(rng.standard_normal((K, N)), "e4m3")
    wide = np.zeros((M - 1) * lda + K, np.float32)
    for m in range(M):
        wide[m * lda:m * lda + K] = A[m]
    got = gpu_mx_gemm(ctx, wide, codes, scales, M, N, K, "e4m3", False, lda=lda)
    A = A.astype(np.float64)
    assert (np.abs(got - A @ B) <= 2 * (3 * K + 1) * U * (np.abs(A) @ np.abs(B))).all()


@pytest.mark.parametrize("size", [48, 560, 1209])
def test_product_with_infinities_and_nans(ctx, size):
    """A value that is not finite makes every result that it contributes to not finite, and no
    other; a masked sample's row of zeros gives zeros."""
    rng = np.random.default_rng(size)
    M, N, K = size, size + 3, size - 5
    A = rng.standard_normal((M, K)).astype(np.float32)
    A[3, 4], A[9, 1], A[11, 0] = np.inf, -np.inf, np.nan
    A.view(np.uint32)[13, 2] = 0x7f800001  # a NaN whose payload is its last bit
    A[20] = 0.0
    x = rng.standard_normal((K, N))
    x[6, 8] = np.nan
    codes, scales, B = mx.stored(x, "e4m3")
    for trans_a in (False, True):
        got = gpu_mx_gemm(ctx, A.T if trans_a else A, codes, scales, M, N, K, "e4m3", trans_a)
        bad = np.zeros((M, N), bool)
        bad[[3, 9, 11, 13]] = True
        bad[:, 8] = True
        assert not np.isfinite(got[bad]).any()
        assert np.isnan(got[[11, 13]]).all()
        ok = ~bad
        A0, B0 = np.where(np.isfinite(A), A, 0).astype(np.float64), np.where(np.isnan(B), 0, B)
        room = 2 * (3 * K + 1) * U * (np.abs(A0) @ np.abs(B0))
        assert (np.abs(got - A0 @ B0) <= room)[ok].all()
        assert (got[20][np.arange(N) != 8] == 0).all()


# ---- linear layers ----
def gpu_mx_linear(ctx, X, W, bias, M, N, K, x_format, w_format, act, ldx=None, ldy=None):
    pb = ProgramBuilder()
    x, w = pb.input(X.size), pb.mx_tensor(N, K, w_format, "input")
    ldy = N if ldy is None else ldy
    b = pb.input(N) if bias is not None else None
    y = pb.input((M - 1) * ldy + N, inout=True)
    pb.mx_linear(x, w, y, M, N, K, x_format=x_format, w_format=w_format, bias=b, act=act, ldx=ldx,
                 ldy=ldy)
    prog = HipProgram(ctx, pb.image())
    by = ctx.upload(np.full((M - 1) * ldy + N, 77.0, np.float32))
    prog.run([put(ctx, X), put(ctx, W[0]), put(ctx, W[1])]
             + ([put(ctx, bias)] if bias is not None else []) + [by], [])
    prog.close()
    got = np.concatenate([by.download(), np.full(ldy - N, 77.0, np.float32)]).reshape(M, ldy)
    assert (got[:, N:] == 77.0).all()
    return got[:, :N]


def linear_room(X, W, bias, act, z):
    """Of the sum, the bias's addition and the activation (whose slope is at most one, evaluated
    in binary64 and rounded once)."""
    K = X.shape[1]
    room = 2 * (K + 2) * U * (np.abs(X) @ np.abs(W.T) + np.abs(bias))
    return room + (U * np.abs(mx.activate(act, z)) if act in ("tanh", "sigmoid") else 0.0)


LINEARS = [(1, 1, 1), (1, 7, 33), (1, 300, 1000), (1, 1030, 4096), (2, 130, 128), (3, 64, 129),
           (4, 17, 600), (5, 33, 257), (15, 65, 64), (16, 1030, 300), (17, 16, 2100), (33, 100, 31),
           (64, 512, 1024), (100, 333, 200), (129, 127, 130), (256, 256, 512), (300, 1021, 617),
           (1030, 520, 260), (16, 70, 1100), (3, 40, 6000), (20, 3100, 130), (40, 3100, 300), (90, 1100, 200), (20, 3100, 1500),
           (40, 3100, 1500), (700, 30, 130)]
# tiles in LDS: whole, split along K, of 256, and of 256 ahead of 128
LARGE_LINEARS = [(1030, 1031, 1033), (70, 2000, 8300), (4000, 3001, 200), (4000, 4050, 70), (4400, 4000, 100)]


@pytest.mark.parametrize("x_format", mx.FORMATS)
@pytest.mark.parametrize("w_format", mx.FORMATS)
@pytest.mark.parametrize("shape", LINEARS + LARGE_LINEARS, ids=str)
def test_linear_layer_of_microscaled_weights(ctx, shape, w_format, x_format):
    M, N, K = shape
    rng = np.random.default_rng(3 * M + 5 * N + K)
    X = (rng.standard_normal((M, K)) * np.exp2(rng.integers(-3, 3, (M, 1)))).astype(np.float32)
    codes, scales, W = mx.stored(rng.standard_normal((N, K)) * np.sqrt(1.0 / K), w_format)
    Xq = mx.stored(X, x_format)[2]
    act = [None, "relu", "tanh", "sigmoid"][(M + N + K) % 4]
    bias = rng.standard_normal(N).astype(np.float32) if (M + K) % 3 else None
    got = gpu_mx_linear(ctx, X, (codes, scales), bias, M, N, K, x_format, w_format, act)
    b = np.zeros(N) if bias is None else bias.astype(np.float64)
    z = Xq @ W.T + b
    assert (np.abs(got - mx.activate(act, z)) <= linear_room(Xq, W, b, act, z)).all()


@pytest.mark.parametrize("x_format", mx.FORMATS)
@pytest.mark.parametrize("w_format", mx.FORMATS)
@pytest.mark.parametrize("shape", [(3, 50, 700), (40, 50, 700), (1100, 1050, 1000)], ids=str)
def test_linear_layer_of_blocks_of_different_sizes(ctx, shape, w_format, x_format):
    """Blocks 24 binades apart beside each other, on both sides: the small ones' products still count
    to binary32 where the large ones of the other side are small or zero."""
    M, N, K = shape
    rng = np.random.default_rng(K + M)
    blocks = -(-K // 32)

    def spread(rows):
        f = np.exp2(rng.choice([-24, -12, 0], (rows, blocks))) * (rng.random((rows, blocks)) < 0.7)
        return rng.standard_normal((rows, K)) * np.repeat(f, 32, axis=1)[:, :K]

    X = spread(M).astype(np.float32)
    codes, scales, W = mx.stored(spread(N), w_format)
    Xq = mx.stored(X, x_format)[2]
    got = gpu_mx_linear(ctx, X, (codes, scales), None, M, N, K, x_format, w_format, None)
    z = Xq @ W.T
    assert (np.abs(got - z) <= linear_room(Xq, W, np.zeros(N), None, z)).all()


def test_linear_layer_with_strides_and_without_depth(ctx):
    rng = np.random.default_rng(2)
    for M, ldx, N, ldy in ((1, 200, 150, 161), (7, 203, 150, 161), (40, 201, 150, 161),
                           (300, 207, 150, 161), (2500, 203, 2501, 2511)):
        K = 190
        wide = rng.standard_normal((M, ldx)).astype(np.float32)
        codes, scales, W = mx.stored(rng.standard_normal((N, K)), "e2m1")
        got = gpu_mx_linear(ctx, wide, (codes, scales), None, M, N, K, "e4m3", "e2m1", None, ldx, ldy)
        Xq = mx.stored(wide[:, :K], "e4m3")[2]
        z = Xq @ W.T
        assert (np.abs(got - z) <= linear_room(Xq, W, np.zeros(N), None, z)).all()
    bias = rng.standard_normal(9).astype(np.float32)
    e = np.zeros(0, np.uint8)
    for M in (1, 40):
        got = gpu_mx_linear(ctx, np.zeros(0, np.float32), (e, e), bias, M, 9, 0, "e4m3", "e2m1", "relu")
        assert np.array_equal(got, np.tile(np.maximum(bias, 0), (M, 1)))


def test_linear_layers_longer_than_a_piece(ctx):
    rng = np.random.default_rng(6)
    for M, N, K in (((1 << 20) + 37, 3, 8), (2, (1 << 20) + 70, 5)):
        X = rng.standard_normal((M, K)).astype(np.float32)
        codes, scales, W = mx.stored(rng.standard_normal((N, K)), "e4m3")
        bias = rng.standard_normal(N).astype(np.float32)
        got = gpu_mx_linear(ctx, X, (codes, scales), bias, M, N, K, "e4m3", "e4m3", "relu")
        Xq = mx.stored(X, "e4m3")[2]
        z = Xq @ W.T + bias
        assert (np.abs(got - np.maximum(z, 0)) <= linear_room(Xq, W, bias, "relu", z)).all()


@pytest.mark.parametrize("x_format,w_format", [("e4m3", "e2m1"), ("e2m1", "e2m1"), ("e5m2", "e4m3"),
                                               ("e4m3", "e5m2")])
@pytest.mark.parametrize("M,N", [(1, 140), (8, 140), (40, 140), (300, 140), (2000, 2001)])
def test_linear_layer_with_infinities_and_nans(ctx, M, N, x_format, w_format):
    rng = np.random.default_rng(M)
    K = 300
    X = rng.standard_normal((M, K)).astype(np.float32)
    w = rng.standard_normal((N, K))
    w[5, 70] = np.nan  # (e2m1: its block of 32, all of row 5's results either way)
    codes, scales, W = mx.stored(w, w_format)
    bad = np.zeros((M, N), bool)
    bad[:, 5] = True
    if M > 1:
        X[1, 299] = np.inf
        X[M - 1, 0] = np.nan
        bad[[1, M - 1]] = True
    got = gpu_mx_linear(ctx, X, (codes, scales), None, M, N, K, x_format, w_format, None)
    Xq = mx.stored(X, x_format)[2]
    assert not np.isfinite(got[bad]).any()
    Xq, W = np.where(np.isfinite(Xq), Xq, 0), np.where(np.isfinite(W), W, 0)
    z = Xq @ W.T
    assert (np.abs(got - z) <= linear_room(Xq, W, np.zeros(N), None, z))[~bad].all()


# ---- the operators together, and the calls around them ----
def layer_program(R, I, O, act="tanh"):
    """A trained layer's pass with checkpoints: forward, both checkpoints, backward."""
    pb = ProgramBuilder()
    x, W, b, dy = pb.input(R * I), pb.input(O * I), pb.input(O), pb.input(R * O)
    y, dz, db, dw = pb.output(R * O), pb.output(R * O), pb.output(O), pb.output(O * I)
    kx, ky = pb.mx_tensor(R, I, "e4m3"), pb.mx_tensor(R, O, "e4m3")
    pb.gemm(x, W, y, R, O, I, trans_b=True, bias=b, act=act)
    pb.mx_encode(x, kx, R, I, keep_nonzero=True)
    pb.mx_encode(y, ky, R, O, keep_nonzero=True)
    pb.mx_act_grad(dy, ky, dz, R, O, act=act, colsum=db)
    pb.mx_gemm(dz, kx, dw, O, I, R, trans_a=True)
    return pb, [y, dz, db, dw]


@pytest.mark.parametrize("shape", [(20, 30, 25), (700, 640, 580)], ids=str)
def test_layer_trained_from_checkpoints(ctx, shape):
    R, I, O = shape
    rng = np.random.default_rng(R)
    x, W = rng.standard_normal((R, I)), rng.standard_normal((O, I)) / np.sqrt(I)
    b, dy = rng.standard_normal(O) * 0.1, rng.standard_normal((R, O)) / R
    ins = [a.astype(np.float32) for a in (x, W, b, dy)]
    pb, outs = layer_program(R, I, O)
    y, dz, db, dw = [o.reshape(s) for o, s in zip(run_program(ctx, pb, ins, outs),
                                                 [(R, O), (R, O), (O,), (O, I)])]
    X, Y = mx.stored(ins[0], "e4m3", True)[2], mx.stored(y, "e4m3", True)[2]
    Y32, one = Y.astype(np.float32), np.float32(1)
    assert np.array_equal(dz, ins[3] * (one - Y32 * Y32))
    d = dz.astype(np.float64)
    assert (np.abs(db - d.sum(0)) <= U * np.abs(d.sum(0)) + 2.0 ** -50 * np.abs(d).sum(0)).all()
    assert (np.abs(dw - d.T @ X) <= 2 * (3 * R + 1) * U * (np.abs(d).T @ np.abs(X))).all()


def test_weight_gradient_against_differences(ctx):
    """The loss sum(dY . act(X^ W^T)) of the stored input moves by dW as W does: a central
    difference in 64 bits, off by its third-order term (bounded by the step's cube)."""
    R, I, O = 24, 20, 18
    rng = np.random.default_rng(4)
    x, W = rng.standard_normal((R, I)), rng.standard_normal((O, I)) / np.sqrt(I)
    codes, scales, X = mx.stored(x, "e4m3")
    dy = rng.standard_normal((R, O))
    dz = (dy * (1 - np.tanh(X @ W.T) ** 2)).astype(np.float32)
    got = gpu_mx_gemm(ctx, dz, codes, scales, O, I, R, "e4m3", True)
    h = 2.0 ** -12
    for o, i in ((0, 0), (7, 3), (17, 19)):
        def loss(t):
            V = W.copy()
            V[o, i] += t
            return (dy * np.tanh(X @ V.T)).sum()
        diff = (loss(h) - loss(-h)) / (2 * h)
        # |tanh'''| <= 2, in the direction X[:, i]; dz's rounding; the product's sum; the loss's own
        room = (h * h / 6 * 2 * (np.abs(dy[:, o]) * np.abs(X[:, i]) ** 3).sum()
                + (2 * (3 * R + 1) + 1) * U * (np.abs(dy[:, o]) * np.abs(X[:, i])).sum()
                + 2.0 ** -50 * np.abs(dy).sum() * R * O / h)
        assert abs(got[o, i] - diff) <= room


@pytest.mark.parametrize("shape", [(300, 260, 280), (2100, 1300, 1290)], ids=str)
def test_repeated_runs_graphs_and_the_static_entry_agree(ctx, shape):
    """The same bits from plain runs, graph replays with other work between them, an asynchronous
    run and the entry that allocates nothing."""
    R, I, O = shape
    rng = np.random.default_rng(8)
    ins = [a.astype(np.float32) for a in (rng.standard_normal((R, I)), rng.standard_normal((O, I)) / 16,
                                          rng.standard_normal(O), rng.standard_normal((R, O)))]
    pb, outs = layer_program(R, I, O, "relu")
    prog = HipProgram(ctx, pb.image())
    b_in, b_out = [ctx.upload(a) for a in ins], [ctx.buffer(s.nbytes) for s in outs]
    prog.set_graph_mode(False)
    prog.run(b_in, b_out)
    want = [b.download() for b in b_out]

    def same():
        for b, w in zip(b_out, want):
            assert np.array_equal(b.download(), w)
            b.upload(np.zeros_like(w))

    same()
    prog.set_graph_mode(True)
    for _ in range(4):
        prog.run(b_in, b_out)
        same()
    prog.run_async(b_in, b_out)
    prog.wait()
    same()
    prog.run_static(b_in, b_out)
    same()
    other = HipProgram(ctx, pb.image())  # two programs' graphs, run in turn
    other.set_graph_mode(True)
    for _ in range(2):
        for p in (prog, other):
            p.run(b_in, b_out)
            same()
    prog.close()
    other.close()


@pytest.mark.parametrize("shape", [(40, 200, 300), (70, 200, 5000), (600, 1100, 1700)], ids=str)
def test_concurrent_runs_of_one_program(ctx, shape):
    import threading
    M, N, K = shape
    rng = np.random.default_rng(1)
    codes, scales, _ = mx.stored(rng.standard_normal((N, K)), "e2m1")
    pb = ProgramBuilder()
    x, w, y = pb.input(M * K), pb.mx_tensor(N, K, "e2m1", "input"), pb.output(M * N)
    pb.mx_linear(x, w, y, M, N, K)
    prog = HipProgram(ctx, pb.image())
    bw = [ctx.upload(codes), ctx.upload(scales)]
    xs = [rng.standard_normal((M, K)).astype(np.float32) for _ in range(6)]
    bufs = [(ctx.upload(v), ctx.buffer(4 * M * N)) for v in xs]
    want = []
    for bx, by in bufs:
        prog.run([bx] + bw, [by])
        want.append(by.download())
    errors = []

    def work(i):
        try:
            for _ in range(20):
                prog.run([bufs[i][0]] + bw, [bufs[i][1]])
                if not np.array_equal(bufs[i][1].download(), want[i]):
                    errors.append(i)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(len(bufs))]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not errors
    prog.close()


def test_codes_that_are_not_aligned_are_refused(ctx):
    pb = ProgramBuilder()
    X, y = pb.mx_tensor(2, 128, "e4m3", "input"), pb.output(256)
    pb.mx_decode(X, y, 2, 128)
    prog = HipProgram(ctx, pb.image())
    store, scales, out = ctx.buffer(1024), ctx.buffer(64), ctx.buffer(1024)
    at = store.device_pointer()
    for off, s_off in ((1, 0), (8, 0), (0, 2)):
        odd = HipBuffer(ctx, 256, at + off)
        s = HipBuffer(ctx, 8, scales.device_pointer() + s_off)
        with pytest.raises(HipInvalidArgument, match="alignment"):
            prog.run([odd, s], [out])
    prog.run([HipBuffer(ctx, 256, at + 16), HipBuffer(ctx, 8, scales.device_pointer() + 4)], [out])
    prog.close()
