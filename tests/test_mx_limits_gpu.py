"""Microscaled steps at extents where a launch would exceed what a grid holds, or where its work goes
round more than once (synaptik_amd/csrc/launch_limits.h)."""
import numpy as np
import pytest

from synaptik_amd.native import HipProgram
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


def sums_of_a_row(ctx, C, add):
    """The column sums, at places, of one row of C floats: 1.5 but for a hundred numbers from each
    place on. add(pb, row slot) adds the step and gives (its other inputs, the slot of the sums, the
    other outputs)."""
    places = [0, (1 << 29) - 50, (1 << 30) - 100, C - 100]
    pb = ProgramBuilder()
    row = pb.output(C)
    pb.fill(row, C, 1.5)
    prog = HipProgram(ctx, pb.image())
    buf = ctx.buffer(4 * C)
    prog.run([], [buf])
    prog.close()
    for i, at in enumerate(places):
        buf.upload(np.arange(100, dtype=np.float32) + 100 * i, 4 * at)
    pb = ProgramBuilder()
    ins, sums, outs = add(pb, pb.input(C))
    prog = HipProgram(ctx, pb.image())
    made = {id(s): ctx.buffer(s.nbytes) for s in ins + outs + [sums]}
    made[id(sums)].upload(np.full(200, -7.0, np.float32), 4 * (C - 200))
    prog.run([buf] + [made[id(s)] for s in ins], [made[id(s)] for s in outs + [sums]])
    prog.close()
    for i, at in enumerate(places):
        got = made[id(sums)].download(count=100, offset=4 * at)
        assert np.array_equal(got, np.arange(100, dtype=np.float32) + 100 * i), at
    got = made[id(sums)].download(count=100, offset=4 * (C - 200))
    assert np.array_equal(got, np.full(100, 1.5, np.float32))


def test_column_sums_of_more_columns_than_a_launch_finishes(ctx):
    """2^30 columns and more: 256 threads for every 64 of them are more than a launch has."""
    C = (1 << 30) + 300

    def act_grad(pb, row):
        Y, dz, db = pb.mx_tensor(1, C, "e2m1", "input"), pb.output(C), pb.output(C)
        pb.mx_act_grad(row, Y, dz, 1, C, act=None, format="e2m1", colsum=db)
        return list(Y), db, [dz]

    def colsum(pb, row):
        db = pb.output(C)
        pb.colsum(row, db, 1, C)
        return [], db, []

    sums_of_a_row(ctx, C, act_grad)
    sums_of_a_row(ctx, C, colsum)
