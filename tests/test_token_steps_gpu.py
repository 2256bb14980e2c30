"""Embeddings, layer norm, gated recurrences and distillation on the GPU against 64-bit forms of their
definitions; the tolerances are derived in tests/token_oracle.py."""
import numpy as np
import pytest

from synaptik_amd.native import HipBackendError, HipProgram
from synaptik_amd.program import ProgramBuilder
from tests import token_oracle as o
from tests.gpu_helpers import run_program

pytestmark = pytest.mark.gpu
INT = {"i32": np.int32, "i64": np.int64}


def run(ctx, pb, inputs, outputs):
    """run_program with buffers for empty arrays too."""
    return run_program(ctx, pb, [a if np.size(a) else np.zeros(1, np.asarray(a).dtype) for a in inputs], outputs)


def floats(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


# ---- embeddings ----
@pytest.mark.parametrize("index", ["i32", "i64"])
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 7, 4), (3, 5, 17), (5, 2, 64), (130, 9, 65), (64, 1000, 1024),
                                   (700, 33, 257), (2000, 4099, 1021), (1, 3, 40000)])
@pytest.mark.parametrize("pad", [None, 0, -1])
def test_embed(ctx, N, V, D, index, pad):
    rng = np.random.default_rng(N + V + D)
    W, tokens = floats(rng, V, D), rng.integers(0, V, N).astype(INT[index])
    if pad is not None:
        tokens[rng.random(N) < 0.3] = pad
    scale = 1.0 if pad is None else 2.5
    pb = ProgramBuilder()
    sw, st, sy = pb.input(V * D), pb.input(N, index), pb.output(N * D)
    pb.embed(sw, st, sy, N, V, D, scale=scale, pad=pad)
    (got,) = run(ctx, pb, [W, tokens], [sy])
    assert np.array_equal(got.reshape(N, D), o.embed(W, tokens, scale, pad))


def test_embed_keeps_what_lies_between_rows(ctx):
    N, V, D, ldy = 37, 11, 70, 75
    rng = np.random.default_rng(0)
    W, tokens = floats(rng, V, D), rng.integers(0, V, N).astype(np.int32)
    pb = ProgramBuilder()
    sw, st, sy = pb.input(V * D), pb.input(N, "i32"), pb.input((N - 1) * ldy + D, inout=True)
    pb.embed(sw, st, sy, N, V, D, ldy=ldy)
    prog = HipProgram(ctx, pb.image())
    by = ctx.upload(np.full(N * ldy, 7.0, np.float32))
    prog.run([ctx.upload(W), ctx.upload(tokens), by], [])
    got = by.download().reshape(N, ldy)
    assert np.array_equal(got[:, :D], o.embed(W, tokens, 1.0)) and (got[:, D:] == 7.0).all()
    prog.close()


def bad_tokens(rng, N, V, dtype):
    t = rng.integers(0, V, N).astype(dtype)
    t[[1, N // 2, N - 1]] = [-1, V, np.iinfo(dtype).max]
    return t


@pytest.mark.parametrize("index", ["i32", "i64"])
@pytest.mark.parametrize("N", [10, 9000])
def test_tokens_out_of_bounds_fail_the_run(ctx, N, index):
    V, D = 13, 20
    rng = np.random.default_rng(1)
    tokens = bad_tokens(rng, N, V, INT[index])
    W, dY = floats(rng, V, D), floats(rng, N, D)
    for grad in (False, True):
        pb = ProgramBuilder()
        a, st, y = pb.input(N * D if grad else V * D), pb.input(N, index), pb.output(V * D if grad else N * D)
        (pb.embed_grad if grad else pb.embed)(a, st, y, N, V, D)
        prog = HipProgram(ctx, pb.image())
        by = ctx.buffer(y.nbytes)
        with pytest.raises(HipBackendError, match="out of bounds"):
            prog.run([ctx.upload(dY if grad else W), ctx.upload(tokens)], [by])
        if grad:
            want, bound = o.embed_grad(dY, tokens.astype(np.int64), V, 1.0)
            o.within(by.download(), want, bound)
        else:
            assert np.array_equal(by.download().reshape(N, D), o.embed(W, tokens.astype(np.int64), 1.0))
        # the same program goes on with tokens in bounds
        prog.run([ctx.upload(dY if grad else W), ctx.upload(np.zeros(N, INT[index]))], [by])
        prog.close()


def tokens_like(rng, kind, N, V):
    """Token lists: even, with frequent ones, one alone, one in two, in order."""
    if kind == "even":
        return rng.integers(0, V, N)
    if kind == "frequent":
        return rng.permutation(V)[np.minimum(V - 1, (np.exp(rng.random(N) * np.log(V + 1)) - 1).astype(np.int64))]
    if kind == "one":
        return np.full(N, V - 1)
    if kind == "half":
        return np.where(rng.random(N) < 0.5, V // 2, rng.integers(0, V, N))
    return np.sort(rng.integers(0, V, N))


@pytest.mark.parametrize("kind", ["even", "frequent", "one", "half", "sorted"])
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 600, 5), (31, 4, 3), (32, 2, 260), (33, 1, 8), (64, 7, 64), (65, 512, 300),
                                   (300, 513, 17), (4096, 1000, 12), (4097, 70000, 5), (5001, 511, 61),
                                   (9000, 262144, 4), (20000, 300000, 3), (256, 300, 40), (257, 40, 33), (1024, 77, 20),
                                   (1025, 5, 9), (2049, 1100, 30), (6145, 90, 7), (8192, 2000, 11), (8193, 33, 6),
                                   (130, 1200000, 3), (600, 1200000, 2)])
def test_embed_grad(ctx, N, V, D, kind):
    rng = np.random.default_rng(N + V)
    tokens = tokens_like(rng, kind, N, V)
    dY = (floats(rng, N, D) * np.exp2(rng.integers(-8, 8, (N, 1)))).astype(np.float32)
    for index, pad, accumulate in (("i32", None, False), ("i64", V - 1, False), ("i64", None, True), ("i32", -5, True)):
        t = tokens.copy()
        if pad is not None and pad < 0:
            t[rng.random(N) < 0.2] = pad
        scale = 1.0 if pad is None else 0.75
        old = floats(rng, V, D) if accumulate else np.full((V, D), np.nan, np.float32)
        pb = ProgramBuilder()
        sd, st, sw = pb.input(N * D), pb.input(N, index), pb.input(V * D, inout=True)
        pb.embed_grad(sd, st, sw, N, V, D, scale=scale, pad=pad, accumulate=accumulate)
        prog = HipProgram(ctx, pb.image())
        bw = ctx.upload(old)
        prog.run([ctx.upload(dY), ctx.upload(t.astype(INT[index])), bw], [])
        want, bound = o.embed_grad(dY, t, V, scale, pad)
        if accumulate:
            bound = bound + o.U * np.abs(old + want)
            named = np.isin(np.arange(V), t[(t >= 0) & (t != (V if pad is None else pad))])
            want = old + want
            assert np.array_equal(bw.download().reshape(V, D)[~named], old[~named])
        o.within(bw.download(), want, bound)
        prog.close()


def test_embed_grad_of_rows_apart(ctx):
    N, V, D, ldy = 100, 30, 33, 40
    rng = np.random.default_rng(3)
    dY, tokens = floats(rng, N, ldy), rng.integers(0, V, N).astype(np.int32)
    pb = ProgramBuilder()
    sd, st, sw = pb.input((N - 1) * ldy + D), pb.input(N, "i32"), pb.output(V * D)
    pb.embed_grad(sd, st, sw, N, V, D, ldy=ldy)
    (got,) = run(ctx, pb, [dY.reshape(-1)[:(N - 1) * ldy + D], tokens], [sw])
    want, bound = o.embed_grad(dY[:, :D], tokens, V, 1.0)
    o.within(got, want, bound)


def test_embed_grad_of_many_sorting_groups(ctx):
    """More than 64 groups of 4096 rows: their digits' counts are added by a launch of their own."""
    N, V, D = 300001, 70001, 2
    rng = np.random.default_rng(4)
    dY, tokens = floats(rng, N, D), tokens_like(rng, "frequent", N, V).astype(np.int32)
    pb = ProgramBuilder()
    sd, st, sw = pb.input(N * D), pb.input(N, "i32"), pb.output(V * D)
    pb.embed_grad(sd, st, sw, N, V, D)
    (got,) = run(ctx, pb, [dY, tokens], [sw])
    want, bound = o.embed_grad(dY, tokens, V, 1.0)
    o.within(got, want, bound)


def test_embed_grad_of_nothing(ctx):
    V, D = 50, 30
    pb = ProgramBuilder()
    sw = pb.input(V * D, inout=True)
    pb.embed_grad(pb.input(1), pb.input(1, "i32"), sw, 0, V, D)
    prog = HipProgram(ctx, pb.image())
    bw = ctx.upload(np.full(V * D, 3.0, np.float32))
    prog.run([bw, ctx.buffer(4), ctx.buffer(4)], [])
    assert (bw.download() == 0).all()
    prog.close()


# ---- layer norm ----
NORM_SHAPES = [(1, 1), (5, 2), (3, 8), (130, 9), (2, 16), (7, 31), (9, 64), (33, 65), (1, 127), (6, 256), (200, 257),
               (3, 512), (5, 1000), (1, 1024), (2, 1025), (700, 1021), (3, 2048), (5, 3001), (1, 4096), (2, 4097),
               (3, 8192), (2, 8195), (1, 16384), (2, 16385), (3, 40001), (2100, 12), (5000, 300)]


def rows_like(rng, R, C):
    """Rows of very different sizes, some far from zero, one constant."""
    x = floats(rng, R, C) * np.exp2(rng.integers(-10, 10, (R, 1))).astype(np.float32)
    x += np.where(rng.random((R, 1)) < 0.3, 1000.0, 0.0).astype(np.float32)
    if R > 2:
        x[1] = 3.25
    return x.astype(np.float32)


@pytest.mark.parametrize("R,C", NORM_SHAPES)
@pytest.mark.parametrize("weights", ["both", "gamma", "beta", "none"])
def test_layer_norm(ctx, R, C, weights):
    rng = np.random.default_rng(R * 7 + C)
    x = rows_like(rng, R, C)
    gamma = floats(rng, C) if weights in ("both", "gamma") else None
    beta = floats(rng, C) if weights in ("both", "beta") else None
    eps = 1e-5 if weights == "both" else 0.125
    pb = ProgramBuilder()
    sx, sy = pb.input(R * C), pb.output(R * C)
    pb.layer_norm(sx, sy, R, C, gamma=None if gamma is None else pb.input(C),
                  beta=None if beta is None else pb.input(C), eps=eps)
    (got,) = run(ctx, pb, [x] + [w for w in (gamma, beta) if w is not None], [sy])
    want, bound = o.layer_norm(x, gamma, beta, eps)
    o.within(got, want, bound)


@pytest.mark.parametrize("C", [70, 1500, 20000])
def test_layer_norm_in_place_and_of_rows_apart(ctx, C):
    R, ld = 9, C + 3
    rng = np.random.default_rng(C)
    x = floats(rng, R, ld)
    pb = ProgramBuilder()
    s = pb.input((R - 1) * ld + C, inout=True)
    pb.layer_norm(s, s, R, C, ldx=ld, ldy=ld)
    prog = HipProgram(ctx, pb.image())
    b = ctx.upload(x)
    prog.run([b], [])
    got = b.download().reshape(R, ld)
    want, bound = o.layer_norm(x[:, :C], None, None, 1e-5)
    o.within(got[:, :C], want, bound)
    assert np.array_equal(got[:, C:], x[:, C:])
    prog.close()


@pytest.mark.parametrize("C", [50, 1100, 17000])
def test_layer_norm_of_values_that_are_not_finite(ctx, C):
    rng = np.random.default_rng(C)
    x = floats(rng, 4, C)
    x[0, C // 2], x[1, 0], x[3, C - 1] = np.nan, np.inf, -np.inf
    dy = floats(rng, 4, C)
    pb = ProgramBuilder()
    sx, sd, sy, dx = pb.input(4 * C), pb.input(4 * C), pb.output(4 * C), pb.output(4 * C)
    pb.layer_norm(sx, sy, 4, C)
    pb.layer_norm_grad(sd, sx, dx, 4, C)
    y, d = run(ctx, pb, [x, dy], [sy, dx])
    for v in (y.reshape(4, C), d.reshape(4, C)):
        assert np.isnan(v[[0, 1, 3]]).all() and np.isfinite(v[2]).all()


def test_layer_norm_without_epsilon(ctx):
    """A constant row is 0 / 0."""
    x = np.array([[1, 2, 3, 4], [5, 5, 5, 5]], np.float32)
    pb = ProgramBuilder()
    sx, sy = pb.input(8), pb.output(8)
    pb.layer_norm(sx, sy, 2, 4, eps=0.0)
    (y,) = run(ctx, pb, [x], [sy])
    o.within(y[:4], *[v[0] for v in o.layer_norm(x[:1], None, None, 0.0)])
    assert np.isnan(y[4:]).all()


@pytest.mark.parametrize("R,C", NORM_SHAPES)
@pytest.mark.parametrize("wanted", ["both", "gamma", "beta", "none"])
def test_layer_norm_grad(ctx, R, C, wanted):
    rng = np.random.default_rng(R + 31 * C)
    x, dy = rows_like(rng, R, C), floats(rng, R, C)
    gamma = floats(rng, C) if wanted in ("both", "gamma") else None
    eps = 1e-5 if wanted == "both" else 0.125
    pb = ProgramBuilder()
    sd, sx, dx = pb.input(R * C), pb.input(R * C), pb.output(R * C)
    dg = pb.output(C) if wanted in ("both", "gamma") else None
    db = pb.output(C) if wanted in ("both", "beta") else None
    pb.layer_norm_grad(sd, sx, dx, R, C, gamma=None if gamma is None else pb.input(C), dgamma=dg, dbeta=db, eps=eps)
    slots = [s for s in (dx, dg, db) if s is not None]
    got = dict(zip([s.index for s in slots], run(ctx, pb, [dy, x] + ([] if gamma is None else [gamma]), slots)))
    want, bound = o.layer_norm_grad(dy, x, gamma, eps)
    for slot, w, b in zip((dx, dg, db), want, bound):
        if slot is not None:
            o.within(got[slot.index], w, b)


@pytest.mark.parametrize("C", [60, 900, 3000, 18000])
def test_layer_norm_grad_in_place_and_of_rows_apart(ctx, C):
    R, ldx, ld = 13, C + 1, C + 6
    rng = np.random.default_rng(C)
    x, dy, gamma = floats(rng, R, ldx), floats(rng, R, ld), floats(rng, C)
    pb = ProgramBuilder()
    sd, sx, sg = pb.input((R - 1) * ld + C, inout=True), pb.input((R - 1) * ldx + C), pb.input(C)
    dg, db = pb.output(C), pb.output(C)
    pb.layer_norm_grad(sd, sx, sd, R, C, gamma=sg, dgamma=dg, dbeta=db, lddy=ld, ldx=ldx, lddx=ld)
    prog = HipProgram(ctx, pb.image())
    bd, bg, bb = ctx.upload(dy), ctx.buffer(4 * C), ctx.buffer(4 * C)
    prog.run([bd, ctx.upload(x), ctx.upload(gamma)], [bg, bb])
    want, bound = o.layer_norm_grad(dy[:, :C], x[:, :C], gamma, 1e-5)
    got = bd.download().reshape(R, ld)
    o.within(got[:, :C], want[0], bound[0])
    o.within(bg.download(), want[1], bound[1])
    o.within(bb.download(), want[2], bound[2])
    assert np.array_equal(got[:, C:], dy[:, C:])
    prog.close()


def test_layer_norm_grad_of_no_rows(ctx):
    pb = ProgramBuilder()
    dg, db = pb.output(5), pb.output(5)
    pb.layer_norm_grad(pb.input(1), pb.input(1), pb.output(1), 0, 5, dgamma=dg, dbeta=db)
    prog = HipProgram(ctx, pb.image())
    b = [ctx.upload(np.ones(5, np.float32)) for _ in range(3)]
    prog.run([ctx.buffer(4), ctx.buffer(4)], b)
    assert (b[0].download() == 0).all() and (b[1].download() == 0).all()
    prog.close()


# ---- gated recurrence ----
SCANS = [(1, 1, 1), (3, 1, 70), (64, 1, 128), (2, 2, 5), (1, 7, 300), (5, 8, 33), (2, 9, 64), (3, 33, 65), (1, 64, 130),
         (4, 65, 7), (2, 129, 100), (1, 256, 64), (2, 257, 61), (1, 1000, 3), (1, 1024, 40), (3, 1500, 70), (1, 5003, 130),
         (300, 40, 64)]


def scan_inputs(rng, B, T, D):
    """Gates that forget at once, remember for long, and saturate."""
    z = floats(rng, B, T, D) * 2 + (rng.random(D).astype(np.float32) * 12 - 3)
    z.reshape(-1)[rng.random(z.size) < 0.01] = 40.0
    z.reshape(-1)[rng.random(z.size) < 0.01] = -120.0
    return z, floats(rng, B, T, D)


def some_lengths(rng, B, T):
    n = rng.integers(0, T + 1, B)
    n[rng.integers(B)] = T
    if B > 2:
        n[1], n[2] = 0, 1
    return n


@pytest.mark.parametrize("B,T,D", SCANS)
@pytest.mark.parametrize("given", ["all", "state", "lengths", "none"])
def test_gated_scan(ctx, B, T, D, given):
    rng = np.random.default_rng(B + T + D)
    z, u = scan_inputs(rng, B, T, D)
    h0 = floats(rng, B, D) if given in ("all", "state") else None
    index = "i32" if given == "all" else "i64"
    lengths = some_lengths(rng, B, T) if given in ("all", "lengths") else None
    h, last, off, off_last = o.gated_scan(z, u, h0, lengths)
    if lengths is not None:  # behind a sequence's end nothing is read
        behind = np.arange(T)[None] >= lengths[:, None]
        z[behind], u[behind] = np.nan, np.inf
    pb = ProgramBuilder()
    sz, su = pb.input(z.size), pb.input(u.size)
    s0 = None if h0 is None else pb.input(B * D)
    sl = None if lengths is None else pb.input(B, index)
    sh, slast = pb.output(z.size), pb.output(B * D) if given != "lengths" else None
    pb.gated_scan(sz, su, sh, B, T, D, h0=s0, last=slast, lengths=sl)
    ins = [z, u] + ([] if h0 is None else [h0]) + ([] if lengths is None else [lengths.astype(INT[index])])
    got = run(ctx, pb, ins, [s for s in (sh, slast) if s is not None])
    o.within(got[0], h, off)
    if slast is not None:
        o.within(got[1], last, off_last)


@pytest.mark.parametrize("B,T,D", SCANS)
@pytest.mark.parametrize("given", ["all", "state", "lengths", "none"])
def test_gated_scan_grad(ctx, B, T, D, given):
    rng = np.random.default_rng(B * 3 + T + D)
    z, u = scan_inputs(rng, B, T, D)
    full = given in ("all", "state")
    h0, dlast = (floats(rng, B, D), floats(rng, B, D)) if full else (None, None)
    index = "i64" if given == "all" else "i32"
    lengths = some_lengths(rng, B, T) if given in ("all", "lengths") else None
    h = o.gated_scan(z, u, h0, lengths)[0].astype(np.float32)
    dh = floats(rng, B, T, D)
    want, bound = o.gated_scan_grad(dh, z, u, h, h0, dlast, lengths)
    if lengths is not None:
        behind = np.arange(T)[None] >= lengths[:, None]
        z[behind], u[behind], dh[behind], h[behind] = np.nan, np.inf, np.nan, np.nan
    pb = ProgramBuilder()
    slots = [pb.input(z.size) for _ in range(4)]
    s0, sd = (pb.input(B * D), pb.input(B * D)) if full else (None, None)
    sl = None if lengths is None else pb.input(B, index)
    dz, du = pb.output(z.size), pb.output(z.size)
    dh0 = pb.output(B * D) if given != "none" else None
    pb.gated_scan_grad(*slots, dz, du, B, T, D, h0=s0, dlast=sd, dh0=dh0, lengths=sl)
    ins = [dh, z, u, h] + ([h0, dlast] if full else []) + ([] if lengths is None else [lengths.astype(INT[index])])
    got = run(ctx, pb, ins, [s for s in (dz, du, dh0) if s is not None])
    for g, w, b in zip(got, want, bound):
        o.within(g, w, b)


@pytest.mark.parametrize("B,T,D", [(3, 1, 40), (2, 6, 70), (1, 1300, 65)])
def test_states_in_place(ctx, B, T, D):
    """A server's states, moved on twice; and gradients of states in place."""
    rng = np.random.default_rng(T)
    z, u = scan_inputs(rng, B, T, D)
    pb = ProgramBuilder()
    sz, su, state, sh = pb.input(z.size), pb.input(z.size), pb.input(B * D, inout=True), pb.output(z.size)
    pb.gated_scan(sz, su, sh, B, T, D, h0=state, last=state)
    prog = HipProgram(ctx, pb.image())
    h0 = floats(rng, B, D)
    bufs = [ctx.upload(z), ctx.upload(u), ctx.upload(h0)]
    bh = ctx.buffer(z.nbytes)
    for _ in range(2):
        h, last, off, off_last = o.gated_scan(z, u, h0)
        prog.run(bufs, [bh])
        o.within(bh.download(), h, off)
        h0 = bufs[2].download().reshape(B, D)
        o.within(h0, last, off_last)
    prog.close()
    h0, dh, dl = floats(rng, B, D), floats(rng, B, T, D), floats(rng, B, D)
    h = o.gated_scan(z, u, h0)[0].astype(np.float32)
    pb = ProgramBuilder()
    ins = [pb.input(z.size) for _ in range(4)]
    s0, sd = pb.input(B * D), pb.input(B * D, inout=True)
    dz, du = pb.output(z.size), pb.output(z.size)
    pb.gated_scan_grad(*ins, dz, du, B, T, D, h0=s0, dlast=sd, dh0=sd)
    prog = HipProgram(ctx, pb.image())
    bd, outs = ctx.upload(dl), [ctx.buffer(z.nbytes), ctx.buffer(z.nbytes)]
    prog.run([ctx.upload(a) for a in (dh, z, u, h, h0)] + [bd], outs)
    want, bound = o.gated_scan_grad(dh, z, u, h, h0, dl)
    for b, w, off in zip(outs + [bd], want, bound):
        o.within(b.download(), w, off)
    prog.close()


@pytest.mark.parametrize("T,D", [(4, 20), (50, 70), (1300, 64)])
def test_values_that_are_not_finite_stay_within_their_sequence(ctx, T, D):
    """A NaN or infinity in one channel of one sequence, in its inputs, its first state or its last state's
    gradient: other channels are finite, and behind a sequence's end all is zero."""
    B = 4
    rng = np.random.default_rng(T)
    z, u = floats(rng, B, T, D), floats(rng, B, T, D)
    lengths = np.array([T, T // 2, 0, T - 1])
    h0, dlast, dh = floats(rng, B, D), floats(rng, B, D), floats(rng, B, T, D)
    h = o.gated_scan(z, u, h0, lengths)[0].astype(np.float32)
    z[0, 1, 3], h0[1, 5], dlast[1, 6], dlast[2, 7], dlast[3, 8], u[3, 0, 9] = np.nan, np.inf, np.nan, np.inf, np.inf, np.nan
    pb = ProgramBuilder()
    sz, su, sd, sh = (pb.input(z.size) for _ in range(4))
    s0, sl, sn = pb.input(B * D), pb.input(B * D), pb.input(B, "i32")
    out, last, dz, du, dh0 = pb.output(z.size), pb.output(B * D), pb.output(z.size), pb.output(z.size), pb.output(B * D)
    pb.gated_scan(sz, su, out, B, T, D, h0=s0, last=last, lengths=sn)
    pb.gated_scan_grad(sd, sz, su, sh, dz, du, B, T, D, h0=s0, dlast=sl, dh0=dh0, lengths=sn)
    got = run(ctx, pb, [z, u, dh, h, h0, dlast, lengths.astype(np.int32)], [out, last, dz, du, dh0])
    behind = np.arange(T)[None] >= lengths[:, None]
    touched = np.zeros((B, D), bool)
    for b, c in ((0, 3), (1, 5), (1, 6), (2, 7), (3, 8), (3, 9)):
        touched[b, c] = True
    for i in (0, 2, 3):
        a = got[i].reshape(B, T, D)
        assert (a[behind] == 0).all()
        assert np.isfinite(a[np.broadcast_to(~touched[:, None], a.shape)]).all()
    for i in (1, 4):
        assert np.isfinite(got[i].reshape(B, D)[~touched]).all()
    assert np.isnan(got[0].reshape(B, T, D)[0, 1:, 3]).all() and not np.isfinite(got[1].reshape(B, D)[1, 5])
    assert not np.isfinite(got[4].reshape(B, D)[[1, 2, 3], [6, 7, 8]]).any()


@pytest.mark.parametrize("T,D", [(5, 20), (1200, 64)])
def test_lengths_out_of_bounds_fail_the_run(ctx, T, D):
    rng = np.random.default_rng(T)
    z, u = scan_inputs(rng, 3, T, D)
    lengths = np.array([-1, T + 1, T // 2])
    pb = ProgramBuilder()
    sz, su, sl, sh = pb.input(z.size), pb.input(z.size), pb.input(3, "i64"), pb.output(z.size)
    pb.gated_scan(sz, su, sh, 3, T, D, lengths=sl)
    prog = HipProgram(ctx, pb.image())
    bh = ctx.buffer(z.nbytes)
    with pytest.raises(HipBackendError, match="out of bounds"):
        prog.run([ctx.upload(z), ctx.upload(u), ctx.upload(lengths)], [bh])
    h, _, off, _ = o.gated_scan(z, u, None, np.clip(lengths, 0, T))
    o.within(bh.download(), h, off)
    prog.close()


@pytest.mark.parametrize("T", [0, 3])
def test_states_of_empty_sequences(ctx, T):
    B, D = 3, 70
    rng = np.random.default_rng(T)
    h0 = floats(rng, B, D)
    pb = ProgramBuilder()
    s0, last = pb.input(B * D), pb.output(B * D)
    sl = pb.input(B, "i32")
    pb.gated_scan(pb.input(max(1, B * T * D)), pb.input(max(1, B * T * D)), pb.output(max(1, B * T * D)), B, T, D, h0=s0,
                  last=last, lengths=sl)
    prog = HipProgram(ctx, pb.image())
    bl = ctx.buffer(4 * B * D)
    pad = [ctx.buffer(4 * max(1, B * T * D)) for _ in range(3)]
    prog.run([ctx.upload(h0), ctx.upload(np.zeros(B, np.int32))] + pad[:2], [bl, pad[2]])
    assert np.array_equal(bl.download().reshape(B, D), h0)
    prog.close()


# ---- distillation ----
def entries(rng, R, C, K, absent=0.3):
    """Distinct classes for each row; absent entries; rows without any (not the first)."""
    index = np.stack([rng.permutation(C)[:K] if C < 4096 else rng.choice(C, K, replace=False) for _ in range(R)])
    t = floats(rng, R, K) * 3
    index = np.where(rng.random((R, K)) < absent, -1, index)
    t[rng.random((R, K)) < absent / 4] = -np.inf
    index[rng.random(R) < 0.2] = -1
    index[0, 0], t[0, 0] = (index[0, 0] if index[0, 0] >= 0 else (index[0].max() + 1) % C if C > K else 0), 1.5
    if C <= K:
        index[0] = rng.permutation(C)[:K] if K <= C else index[0]
    return index, t


def check_distill(ctx, z, index, t, T=1.0, g=1.0, dtype="i32", grad=True):
    R, C = z.shape
    K = index.shape[1]
    pb = ProgramBuilder()
    sz, si, st, sl = pb.input(R * C), pb.input(R * K, dtype), pb.input(R * K), pb.output(1)
    sg = pb.output(R * C) if grad else None
    pb.distill(sz, si, st, sl, R, C, K, grad=sg, temperature=T, g=g)
    got = run(ctx, pb, [z, index.astype(INT[dtype]), t], [sl] + ([sg] if grad else []))
    loss, want, off, bound = o.distill(z, index, t, T, g)
    o.within(got[0], np.array([loss]), np.array([off]))
    if grad:
        o.within(got[1], want, bound)


@pytest.mark.parametrize("R,C,K", [(1, 1, 1), (1, 2, 2), (3, 5, 3), (2, 16, 16), (70, 63, 7), (5, 64, 1), (9, 65, 8), (4, 255, 40),
                                   (3, 256, 256), (5, 1000, 13), (6, 1020, 5), (3, 1021, 64), (2, 4096, 9), (3, 4099, 300),
                                   (2, 8191, 8), (2, 10007, 17), (2, 16380, 4), (3, 32003, 64), (2, 65532, 3),
                                   (2, 65533, 30), (2, 100001, 1024), (1500, 33, 3), (1025, 130, 2)])
@pytest.mark.parametrize("T,dtype", [(1.0, "i32"), (2.5, "i64")])
def test_distill(ctx, R, C, K, T, dtype):
    rng = np.random.default_rng(R + C + K)
    index, t = entries(rng, R, C, K)
    z = (floats(rng, R, C) * 4).astype(np.float32)
    check_distill(ctx, z, index, t, T, 1.0 if T == 1.0 else -0.5, dtype)
    check_distill(ctx, z, index, t, T, dtype=dtype, grad=False)


@pytest.mark.parametrize("C,K", [(12, 30), (700, 90), (5000, 1000)])
def test_an_entry_of_one_class_twice(ctx, C, K):
    rng = np.random.default_rng(C)
    index = rng.integers(0, min(C, 20), (5, K))
    index[2] = 7
    check_distill(ctx, floats(rng, 5, C) * 3, index, floats(rng, 5, K))


@pytest.mark.parametrize("C", [40, 3000, 70000])
def test_distill_of_extreme_logits(ctx, C):
    """Far apart, the type's lowest value, infinities, NaN."""
    rng = np.random.default_rng(C)
    low = -np.finfo(np.float32).max
    z = floats(rng, 9, C) * 30
    index = np.tile(np.arange(4), (9, 1))
    t = floats(rng, 9, 4) * 30
    z[0] = low
    z[1, 5:] = low
    z[2, 1] = -np.inf                     # a class with an entry, of probability zero
    z[3, 9:] = -np.inf                    # classes without
    t[4] = low
    t[5, 1:] = low
    t[6, 2] = np.nan
    z[7, 3] = np.nan
    z[8, 20] = np.inf
    for r in range(9):  # each by itself: a row that is not finite takes the loss
        check_distill(ctx, z[r:r + 1], index[r:r + 1], t[r:r + 1])
    check_distill(ctx, z[:6], index[:6], t[:6], 0.5)


def test_distill_without_any_entry(ctx):
    """0 / 0, as the mean cross-entropy of no sample; logits are not read."""
    C = 100
    pb = ProgramBuilder()
    sz, si, st, sl, sg = pb.input(3 * C), pb.input(6, "i32"), pb.input(6), pb.output(1), pb.output(3 * C)
    pb.distill(sz, si, st, sl, 3, C, 2, grad=sg)
    t = np.array([[1, 2], [-np.inf, -np.inf], [0, 0]], np.float32)
    index = np.array([[-1, -1], [4, 5], [-1, -1]], np.int32)
    loss, grad = run(ctx, pb, [np.full((3, C), np.nan, np.float32), index, t], [sl, sg])
    assert np.isnan(loss[0]) and (grad == 0).all()


def test_classes_out_of_bounds_fail_the_run(ctx):
    R, C, K = 4, 300, 3
    rng = np.random.default_rng(0)
    z, t = floats(rng, R, C), floats(rng, R, K)
    index = rng.integers(0, 100, (R, 1)) + np.arange(K)
    index[1, 2], index[2, 0] = C, -2
    pb = ProgramBuilder()
    sz, si, st, sl, sg = pb.input(R * C), pb.input(R * K, "i64"), pb.input(R * K), pb.output(1), pb.output(R * C)
    pb.distill(sz, si, st, sl, R, C, K, grad=sg)
    prog = HipProgram(ctx, pb.image())
    bl, bg = ctx.buffer(4), ctx.buffer(4 * R * C)
    with pytest.raises(HipBackendError, match="out of bounds"):
        prog.run([ctx.upload(z), ctx.upload(index), ctx.upload(t)], [bl, bg])
    loss, want, off, bound = o.distill(z, index, t)
    o.within(bg.download(), want, bound)
    prog.close()
