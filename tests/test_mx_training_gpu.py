"""Training from 8-bit checkpoints and inference through microscaled weights on the GPU.

Gradients are compared with their formulas in 64 bits over the values that the step keeps: the
hidden outputs come from a forward program of the same GEMMs (the same bits) and are stored by the
oracle (tests/mx_oracle.py), so no rounding of a code can differ. The error of each quantity is
bounded along the way: u = 2^-24; a product of depth n is off by at most 2 (n + 2) u |A| |B| (each
addition may be cut off, three exact parts of a term count as three), and errors of its operands
pass through it."""
import numpy as np
import pytest

from synaptik_amd.native import HipProgram
from synaptik_amd.program import ProgramBuilder
from synaptik_amd.training import (Adam, AdamW, GradientMode, HipTrainingSession, MlpSpec, Sgd,
                                   encode_mx_weights, init_parameters, lower_mx_forward)
from tests import mx_oracle as mx
from tests.gpu_helpers import run_program

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def problem(dims, act, loss, batch, seed):
    spec = MlpSpec.chain(dims, hidden=act, loss=loss)
    Ws, bs = init_parameters(spec, seed, "xavier_uniform")
    rng = np.random.default_rng(seed + 1)
    bs = [(0.1 * rng.standard_normal(b.size)).astype(np.float32) for b in bs]
    x = rng.standard_normal((batch, dims[0])).astype(np.float32)
    y = (rng.standard_normal((batch, dims[-1])).astype(np.float32) if loss == "mse"
         else rng.integers(0, dims[-1], batch))
    return spec, Ws, bs, x, y


def forward_values(ctx, spec, Ws, bs, x):
    """Every layer's output, from the GEMMs of a training step's forward pass."""
    pb = ProgramBuilder()
    sW, sb = [pb.input(w.size) for w in Ws], [pb.input(b.size) for b in bs]
    cur, outs = pb.input(x.size), []
    for i, l in enumerate(spec.layers):
        outs.append(pb.output(len(x) * l.fan_out))
        pb.gemm(cur, sW[i], outs[-1], len(x), l.fan_out, l.fan_in, trans_b=True, bias=sb[i],
                act=l.activation)
        cur = outs[-1]
    got = run_program(ctx, pb, list(Ws) + list(bs) + [x], outs)
    return [g.reshape(len(x), -1) for g in got]


def product(A, eA, B, eB, parts=1):
    """A . B with error bounds of both operands and of the product itself."""
    n = parts * A.shape[1]
    aA, aB = np.abs(A), np.abs(B)
    return A @ B, 2 * (n + 2) * U * (aA @ aB) + (eA @ (aB + eB)) + aA @ eB


def expected_gradients(ctx, spec, Ws, bs, x, y, checkpoint):
    """[(gradient, bound)] of W_1.., b_1.. by the formulas over the kept values."""
    outs = forward_values(ctx, spec, Ws, bs, x)
    kept = [x.astype(np.float64)] + [mx.stored(o, checkpoint, True)[2] for o in outs[:-1]]
    z, batch = outs[-1].astype(np.float64), len(x)
    if spec.loss == "mse":
        t = y.astype(np.float64)
        dz = 2 * (z - t) / z.size
        # the difference, its double and the factor are each rounded; z is the step's own
        e = 4 * U * np.abs(dz)
    else:
        # logits of a fused head may be summed in another order
        last = spec.layers[-1]
        h = outs[-2].astype(np.float64) if len(outs) > 1 else x.astype(np.float64)
        ez = 4 * (last.fan_in + 2) * U * (np.abs(h) @ np.abs(Ws[-1].T.astype(np.float64)) + np.abs(bs[-1]))
        s = np.exp(z - z.max(1, keepdims=True))
        s /= s.sum(1, keepdims=True)
        dz = s.copy()
        dz[np.arange(batch), y] -= 1
        dz /= batch
        # softmax moves by at most twice the logits' error; its own roundings beside
        e = (s * 2 * ez.max(1, keepdims=True) + 16 * U * (s + np.abs(dz) * batch)) / batch
    L = len(spec.layers)
    gW, gb = [None] * L, [None] * L
    for i in reversed(range(L)):
        zero = np.zeros_like(kept[i])
        gW[i] = product(dz.T, e.T, kept[i], zero, parts=3)
        gb[i] = (dz.sum(0), U * np.abs(dz.sum(0)) + e.sum(0) + 2.0 ** -45 * np.abs(dz).sum(0))
        if i > 0:
            W = Ws[i].astype(np.float64)
            d, ed = product(dz, e, W, np.zeros_like(W))
            slope = mx.slope(spec.layers[i - 1].activation, kept[i])
            dz = d * slope
            e = ed * np.abs(slope) + 4 * U * np.abs(d)  # (1 - y^2 or y (1 - y), and the product)
    return gW + gb


CASES = [([7, 5, 3], "relu", "mse", 4), ([24, 33, 40, 5], "relu", "ce", 50),
         ([24, 33, 40, 5], "tanh", "ce", 129), ([30, 65, 20], "sigmoid", "ce", 77),
         ([16, 64, 64, 64, 1], "tanh", "mse", 256), ([200, 520, 600, 31], "relu", "mse", 1100)]


@pytest.mark.parametrize("checkpoint", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dims,act,loss,batch", CASES, ids=str)
def test_gradients_are_those_of_the_kept_values(ctx, dims, act, loss, batch, checkpoint):
    spec, Ws, bs, x, y = problem(dims, act, loss, batch, 3)
    want = expected_gradients(ctx, spec, Ws, bs, x, y, checkpoint)
    sess = HipTrainingSession.open(ctx, spec, Ws, bs, Sgd(0.5), batch, checkpoint=checkpoint)
    plain = HipTrainingSession.open(ctx, spec, Ws, bs, Sgd(0.5), batch)
    loss_kept = sess.run(x, y, GradientMode.ACCUMULATE).objective
    assert loss_kept == plain.run(x, y, GradientMode.ACCUMULATE).objective
    for a, (g, room) in zip(sess.state().accumulators, want):
        assert (np.abs(a.reshape(g.shape) - g) <= room).all()
    sess.zero_grad()
    # the step: w - rate g, with g's bound and the two roundings
    sess.run(x, y)
    st = sess.state()
    for w0, w1, (g, room) in zip(Ws + bs, st.weights + st.biases, want):
        target = w0 - 0.5 * g
        assert (np.abs(w1 - target) <= 0.5 * room + 2 * U * (np.abs(w0) + np.abs(0.5 * g))).all()
    sess.close()
    plain.close()


@pytest.mark.parametrize("opt", [Sgd(0.1, momentum=0.9), Adam(1e-2), AdamW(1e-2, weight_decay=0.1)],
                         ids=lambda o: type(o).__name__)
def test_modes_agree(ctx, opt):
    """A step that updates at once and one that accumulates a single run first use the same
    gradients up to their products' rounding; pipelined, graph and plain runs give the same bits."""
    spec, Ws, bs, x, y = problem([40, 70, 50, 12], "tanh", "ce", 90, 5)
    batches = [(x, y), (x[::-1].copy(), y[::-1].copy()), (x * 0.5, y)]

    def train(run):
        sess = HipTrainingSession.open(ctx, spec, Ws, bs, opt, 90, checkpoint="e4m3")
        run(sess)
        st = sess.state()
        sess.close()
        return st

    plain = train(lambda s: [s.run(*b) for b in batches])
    piped = train(lambda s: s.run_pipelined(batches))

    def with_graphs(s):
        s.program.set_graph_mode(True)
        for b in batches:
            s.run(*b)
    graphs = train(with_graphs)
    for st in (piped, graphs):
        assert st.optimizer_steps == 3
        for a, b in zip(plain.weights + plain.biases + plain.first + plain.second,
                        st.weights + st.biases + st.first + st.second):
            assert np.array_equal(a, b)
    # one accumulated run with its step: the first slots are the gradient times a factor, each within
    # the gradient's bound and the roundings of the factor and its product
    acc = train(lambda s: s.run(x, y, GradientMode.ACCUMULATE_AND_STEP))
    one = train(lambda s: s.run(x, y))
    factor = 1.0 if isinstance(opt, Sgd) else 1.0 - opt.beta1
    for a, b, (g, room) in zip(acc.first, one.first, expected_gradients(ctx, spec, Ws, bs, x, y, "e4m3")):
        room = factor * (2 * room + 6 * U * np.abs(g))
        assert (np.abs(a - b).reshape(g.shape) <= room).all()
    assert acc.optimizer_steps == one.optimizer_steps == 1


def test_accumulated_runs_add(ctx):
    spec, Ws, bs, x, y = problem([24, 33, 40, 5], "relu", "ce", 50, 9)
    x2 = x[::-1].copy()
    a = expected_gradients(ctx, spec, Ws, bs, x, y, "e4m3")
    b = expected_gradients(ctx, spec, Ws, bs, x2, y, "e4m3")
    sess = HipTrainingSession.open(ctx, spec, Ws, bs, Sgd(0.5), 50, checkpoint="e4m3")
    sess.run(x, y, GradientMode.ACCUMULATE)
    sess.run(x2, y, GradientMode.ACCUMULATE)
    for g, (ga, ra), (gb, rb) in zip(sess.state().accumulators, a, b):
        room = ra + rb + U * (np.abs(ga + gb) + ra + rb)
        assert (np.abs(g.reshape(ga.shape) - (ga + gb)) <= room).all()
    # a step that ignores and empties the pending gradients
    sess.run(x, y)
    st = sess.state()
    assert st.accumulated_gradient_runs == 0
    assert all((acc.download() == 0).all() for acc in sess.accum)
    for w0, w1, (g, room) in zip(Ws + bs, st.weights + st.biases, a):
        assert (np.abs(w1 - (w0 - 0.5 * g)) <= 0.5 * room + 2 * U * (np.abs(w0) + np.abs(0.5 * g))).all()
    sess.close()


def test_a_failed_step_changes_nothing(ctx):
    spec, Ws, bs, x, y = problem([8, 9, 7], "relu", "mse", 16, 2)
    sess = HipTrainingSession.open(ctx, spec, Ws, bs, Sgd(0.5), 16, checkpoint="e4m3")
    sess.run(x, y)
    before = sess.state()
    bad = y.copy()
    bad[3, 2] = np.inf
    with pytest.raises(ArithmeticError):
        sess.run(x, bad)
    after = sess.state()
    assert after.optimizer_steps == before.optimizer_steps == 1
    for a, b in zip(before.weights + before.biases, after.weights + after.biases):
        assert np.array_equal(a, b)
    sess.run(x, y)
    assert sess.optimizer_steps == 2
    sess.close()


@pytest.mark.parametrize("weights,activations", [("e2m1", "e4m3"), ("e2m1", "e2m1"), ("e4m3", "e4m3"),
                                                 ("e5m2", "e4m3")])
@pytest.mark.parametrize("batch", [1, 5, 70])
def test_inference_through_microscaled_weights(ctx, batch, weights, activations):
    """Each layer against its 64-bit form over the input that it had."""
    spec, Ws, bs, x, _ = problem([130, 257, 100, 9], "tanh", "ce", batch, 1)
    bufs = encode_mx_weights(ctx, spec, Ws, weights)
    stored = [mx.stored(w, weights) for w in Ws]
    for i, (c, s, _) in enumerate(stored):
        assert np.array_equal(bufs[2 * i].download(np.uint8).reshape(c.shape), c)
        assert np.array_equal(bufs[2 * i + 1].download(np.uint8).reshape(s.shape), s)
    prog = HipProgram(ctx, lower_mx_forward(spec, batch, weights=weights, activations=activations).image())
    out = ctx.buffer(4 * batch * 9)
    prog.run(bufs + [ctx.upload(b) for b in bs] + [ctx.upload(x)], [out])
    got = out.download().reshape(batch, 9)
    prog.close()
    # the same layers one by one, each output published
    pb = ProgramBuilder()
    sW = [pb.mx_tensor(l.fan_out, l.fan_in, weights, "input") for l in spec.layers]
    sb = [pb.input(b.size) for b in bs]
    cur, outs = pb.input(x.size), []
    for i, l in enumerate(spec.layers):
        outs.append(pb.output(batch * l.fan_out))
        pb.mx_linear(cur, sW[i], outs[-1], batch, l.fan_out, l.fan_in, x_format=activations,
                     w_format=weights, bias=sb[i], act=l.activation)
        cur = outs[-1]
    prog = HipProgram(ctx, pb.image())
    layer_out = [ctx.buffer(s.nbytes) for s in outs]
    prog.run(bufs + [ctx.upload(b) for b in bs] + [ctx.upload(x)], layer_out)
    prog.close()
    layers = [b.download().reshape(batch, -1) for b in layer_out]
    assert np.array_equal(got, layers[-1])
    before = x
    for l, y, (_, _, W), b in zip(spec.layers, layers, stored, bs):
        X = mx.stored(before, activations)[2]
        z = X @ W.T + b
        room = 2 * (l.fan_in + 2) * U * (np.abs(X) @ np.abs(W.T) + np.abs(b))
        want = mx.activate(l.activation, z)
        assert (np.abs(y - want) <= room + U * np.abs(want)).all()
        before = y


def test_encoding_weights_takes_device_buffers(ctx):
    spec, Ws, bs, _, _ = problem([64, 32, 8], "relu", "mse", 4, 0)
    host = encode_mx_weights(ctx, spec, Ws, "e2m1")
    device = encode_mx_weights(ctx, spec, [ctx.upload(w) for w in Ws], "e2m1")
    for a, b in zip(host, device):
        assert np.array_equal(a.download(np.uint8), b.download(np.uint8))
