"""Steps for models of tokens where element offsets pass 32 bits and where rows outnumber a launch's
workgroups."""
import numpy as np
import pytest

from synaptik_amd.native import HipProgram
from synaptik_amd.program import ProgramBuilder
from tests import token_oracle as o

pytestmark = pytest.mark.gpu
N, D, V = (1 << 21) + 5, 1030, 7  # 2.16e9 elements


@pytest.fixture(scope="module")
def rows(ctx):
    """A large matrix whose every row is one of seven: (the seven, the row numbers, its buffer)."""
    rng = np.random.default_rng(0)
    W = rng.standard_normal((V, D)).astype(np.float32)
    tokens = rng.integers(0, V, N).astype(np.int32)
    pb = ProgramBuilder()
    sw, st, sy = pb.input(V * D), pb.input(N, "i32"), pb.output(N * D)
    pb.embed(sw, st, sy, N, V, D)
    prog = HipProgram(ctx, pb.image())
    big = ctx.buffer(4 * N * D)
    prog.run([ctx.upload(W), ctx.upload(tokens)], [big])
    prog.close()
    yield W, tokens, big
    big.close()


PLACES = [0, 1, N // 2, (1 << 31) // D, (1 << 31) // D + 1, N - 2, N - 1]


def row(buf, r):
    return buf.download(count=D, offset=4 * D * r)


def test_embed(rows):
    W, tokens, big = rows
    for r in PLACES:
        assert np.array_equal(row(big, r), W[tokens[r]])


def test_embed_grad(ctx, rows):
    W, tokens, big = rows
    pb = ProgramBuilder()
    sd, st, sw = pb.input(N * D), pb.input(N, "i32"), pb.output(V * D)
    pb.embed_grad(sd, st, sw, N, V, D)
    prog = HipProgram(ctx, pb.image())
    bw = ctx.buffer(4 * V * D)
    prog.run([big, ctx.upload(tokens)], [bw])
    prog.close()
    # equal terms: a sum of n of them in binary64 is off by n 2^-53 of itself, the rounding by 2^-24
    want = np.bincount(tokens, minlength=V)[:, None] * W.astype(np.float64)
    o.within(bw.download(), want, np.abs(want) * (o.U + N * 2.0 ** -52))


def test_layer_norm_and_its_gradient(ctx, rows):
    W, tokens, big = rows
    pb = ProgramBuilder()
    sx, sy, dx, dg, db = pb.input(N * D), pb.output(N * D), pb.output(N * D), pb.output(D), pb.output(D)
    pb.layer_norm(sx, sy, N, D)
    pb.layer_norm_grad(sx, sx, dx, N, D, dgamma=dg, dbeta=db)
    prog = HipProgram(ctx, pb.image())
    outs = [ctx.buffer(s.nbytes) for s in (sy, dx, dg, db)]
    prog.run([big], outs)
    prog.close()
    y, by = o.layer_norm(W, None, None, 1e-5)
    (d, _, _), (bd, _, _) = o.layer_norm_grad(W, W, None, 1e-5)
    for r in PLACES:
        o.within(row(outs[0], r), y[tokens[r]], by[tokens[r]])
        o.within(row(outs[1], r), d[tokens[r]], bd[tokens[r]])
    n = np.bincount(tokens, minlength=V)[:, None]
    W = W.astype(np.float64)
    xh = o.normalised(W, 1e-5)[0]
    for got, terms in ((outs[2], W * xh), (outs[3], W)):
        # partial sums of some thousand rows in binary64, added in binary64, rounded once
        want, mass = (n * terms).sum(0), (n * np.abs(terms)).sum(0)
        o.within(got.download(), want, o.U * np.abs(want) + mass * (2.0 ** -40 + (D + 16) * 2.0 ** -50))


def test_gated_scan_and_its_gradient(ctx):
    """f = 1/2, u = 1, dh = 1: h_t = 1 - 2^-(t+1) and G_t = 2 - 2^-(T-1-t), both exactly until they are 1 and
    2; du = G / 2, dz = G (h_(t-1) - 1) / 4."""
    pb = ProgramBuilder()
    z, one, h, last = pb.internal(N * D), pb.internal(N * D), pb.output(N * D), pb.output(D)
    dz, du = pb.output(N * D), pb.output(N * D)
    pb.fill(z, N * D, 0.0)
    pb.fill(one, N * D, 1.0)
    pb.gated_scan(z, one, h, 1, N, D, last=last)
    pb.gated_scan_grad(one, z, one, h, dz, du, 1, N, D)
    prog = HipProgram(ctx, pb.image())
    outs = [ctx.buffer(s.nbytes) for s in (h, last, dz, du)]
    prog.run([], outs)
    prog.close()
    assert (outs[1].download() == 1).all()
    for t in PLACES:
        state = np.float32(1 - 2.0 ** -(t + 1.0)) if t < 24 else np.float32(1)
        before = 0.0 if t == 0 else 1 - 2.0 ** -float(t) if t <= 24 else 1.0
        G = np.float32(2 - 2.0 ** -float(N - 1 - t)) if N - 1 - t < 24 else np.float32(2)
        assert (row(outs[0], t) == state).all(), t
        assert (row(outs[3], t) == G / 2).all(), t
        assert (row(outs[2], t) == np.float32(float(G) * (before - 1) / 4)).all(), t


def test_distill(ctx, rows):
    W, tokens, big = rows
    index = (tokens * 3).astype(np.int32)
    pb = ProgramBuilder()
    sz, si, st, sl, sg = pb.input(N * D), pb.input(N, "i32"), pb.input(N), pb.output(1), pb.output(N * D)
    pb.distill(sz, si, st, sl, N, D, 1, grad=sg, g=float(N))
    prog = HipProgram(ctx, pb.image())
    outs = [ctx.buffer(4), ctx.buffer(4 * N * D)]
    prog.run([big, ctx.upload(index), ctx.upload(np.zeros(N, np.float32))], outs)
    prog.close()
    each = [o.distill(W[v:v + 1], np.array([[3 * v]]), np.zeros((1, 1), np.float32)) for v in range(V)]
    count = np.bincount(tokens, minlength=V)
    loss = sum(c * e[0] for c, e in zip(count, each)) / N
    o.within(outs[0].download(), np.array([loss]), np.array([sum(c * e[2] for c, e in zip(count, each)) / N + o.U * abs(loss)]))
    for r in PLACES:
        _, grad, _, bound = each[tokens[r]]
        o.within(row(outs[1], r), grad[0], bound[0] + 2 * o.U * np.abs(grad[0]))  # (g T / n is 1 but for two roundings)


def test_distill_of_more_rows_than_a_launch_has_workgroups(ctx):
    R, C = (1 << 20) + 1501, 5
    rng = np.random.default_rng(1)
    z, t = rng.standard_normal((R, C)).astype(np.float32), rng.standard_normal((R, 2)).astype(np.float32)
    index = np.stack([rng.integers(0, 3, R), rng.integers(3, C, R)], 1).astype(np.int32)
    index[rng.random(R) < 0.25] = -1
    pb = ProgramBuilder()
    sz, si, st, sl, sg = pb.input(R * C), pb.input(2 * R, "i32"), pb.input(2 * R), pb.output(1), pb.output(R * C)
    pb.distill(sz, si, st, sl, R, C, 2, grad=sg, g=float(R))
    prog = HipProgram(ctx, pb.image())
    outs = [ctx.buffer(4), ctx.buffer(4 * R * C)]
    prog.run([ctx.upload(z), ctx.upload(index), ctx.upload(t)], outs)
    prog.close()
    there = index[:, 0] >= 0
    n = there.sum()
    q = np.exp(z.astype(np.float64) - z.max(1, keepdims=True))
    q /= q.sum(1, keepdims=True)
    p = np.exp(t.astype(np.float64) - t.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    grad = q.copy()
    at = np.arange(R)
    losses = 0.0
    for j in range(2):
        grad[at, np.maximum(index[:, j], 0)] -= p[:, j]
        losses = losses + p[:, j] * (np.log(p[:, j]) - np.log(q[at, np.maximum(index[:, j], 0)]))
    grad = np.where(there[:, None], grad * (R / n), 0.0)
    # the bounds of tests/token_oracle.py, exponents of at most 10
    o.within(outs[1].download(), grad, o.U * (R / n) * (q * (2 * (3 * 10 + 2) + 2) + 3))
    loss = losses[there].mean()
    o.within(outs[0].download(), np.array([loss]), np.array([o.U * (3 * 10 + 2 + 2 * abs(loss))]))


def test_classes_named_twice_in_more_rows_than_a_launch_has_workgroups(ctx):
    """A workgroup's rows with a class named twice beside rows without: each by its own entries."""
    R, C, K = (1 << 20) + 70000, 300, 3
    rng = np.random.default_rng(3)
    kinds = 64
    z, t = rng.standard_normal((kinds, C)).astype(np.float32), rng.standard_normal((kinds, K)).astype(np.float32)
    index = np.stack([rng.permutation(C)[:K] for _ in range(kinds)]).astype(np.int32)
    index[::2, 2] = index[::2, 0]
    kind = rng.integers(0, kinds, R).astype(np.int32)
    pb = ProgramBuilder()
    sw, sk, sz = pb.input(kinds * C), pb.input(R, "i32"), pb.internal(R * C)
    si, st, sl, sg = pb.input(R * K, "i32"), pb.input(R * K), pb.output(1), pb.output(R * C)
    pb.embed(sw, sk, sz, R, kinds, C)
    pb.distill(sz, si, st, sl, R, C, K, grad=sg, g=float(R))
    prog = HipProgram(ctx, pb.image())
    outs = [ctx.buffer(4), ctx.buffer(4 * R * C)]
    prog.run([ctx.upload(z), ctx.upload(kind), ctx.upload(index[kind]), ctx.upload(t[kind])], outs)
    prog.close()
    each = [o.distill(z[v:v + 1], index[v:v + 1], t[v:v + 1]) for v in range(kinds)]
    want = np.concatenate([e[1] for e in each])
    bound = np.concatenate([e[3] for e in each]) + 2 * o.U * np.abs(want)  # (g T / n is 1 but for two roundings)
    for first in (0, 70000 - 500, 1 << 19, 1 << 20, R - 1000):
        got = outs[1].download(count=1000 * C, offset=4 * C * first).reshape(1000, C)
        o.within(got, want[kind[first:first + 1000]], bound[kind[first:first + 1000]])


def test_layer_norm_of_more_rows_than_a_launch_has_workgroups(ctx):
    R, C = 65536 + 70, 1025
    rng = np.random.default_rng(2)
    x = rng.standard_normal((R, C), dtype=np.float32)
    pb = ProgramBuilder()
    sx, sy = pb.input(R * C), pb.output(R * C)
    pb.layer_norm(sx, sy, R, C)
    prog = HipProgram(ctx, pb.image())
    by = ctx.buffer(4 * R * C)
    prog.run([ctx.upload(x)], [by])
    prog.close()
    for first in (0, 65500):
        got = by.download(count=100 * C, offset=4 * C * first).reshape(100, C)
        want, bound = o.layer_norm(x[first:first + 100], None, None, 1e-5)
        o.within(got, want, bound)
