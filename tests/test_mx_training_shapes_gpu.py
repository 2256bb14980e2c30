"""Checkpointed steps of chains that are not uniform: layers with and without biases and activations,
one row, one unit, widths that are no multiple of a block, and the sum as the loss's reduction."""
import numpy as np
import pytest

from synaptik_amd.training import Dense, GradientMode, HipTrainingSession, MlpSpec, Sgd
from tests.test_mx_training_gpu import U, expected_gradients

pytestmark = pytest.mark.gpu

CHAINS = [([Dense(20, 33, "relu", bias=False), Dense(33, 40, None), Dense(40, 17, "tanh", bias=False), Dense(17, 5)], 50),
          ([Dense(7, 1, "sigmoid"), Dense(1, 129, "relu"), Dense(129, 3, bias=False)], 1),
          ([Dense(130, 300, None, bias=False), Dense(300, 31, bias=False)], 1030)]


@pytest.mark.parametrize("checkpoint", ["e4m3", "e5m2"])
@pytest.mark.parametrize("layers,batch", CHAINS, ids=lambda v: str(v) if isinstance(v, int) else f"{len(v)} layers")
def test_chains_of_mixed_layers(ctx, layers, batch, checkpoint):
    rng = np.random.default_rng(batch)
    spec = MlpSpec(layers, "mse")
    Ws = [(rng.standard_normal((l.fan_out, l.fan_in)) / np.sqrt(l.fan_in)).astype(np.float32) for l in layers]
    bs = [(0.1 * rng.standard_normal(l.fan_out) * l.bias).astype(np.float32) for l in layers]
    x = rng.standard_normal((batch, layers[0].fan_in)).astype(np.float32)
    y = rng.standard_normal((batch, layers[-1].fan_out)).astype(np.float32)
    # the same chain with every bias, zero where the layer has none: the same values everywhere
    want = expected_gradients(ctx, spec, Ws, bs, x, y, checkpoint)
    want = want[:len(layers)] + [w for w, l in zip(want[len(layers):], layers) if l.bias]
    sess = HipTrainingSession.open(ctx, spec, Ws, bs, Sgd(0.25), batch, checkpoint=checkpoint)
    sess.run(x, y, GradientMode.ACCUMULATE)
    for a, (g, room) in zip(sess.state().accumulators, want):
        assert (np.abs(a.reshape(g.shape) - g) <= room).all()
    sess.zero_grad()
    sess.run(x, y)
    st = sess.state()
    before = Ws + [b for b, l in zip(bs, layers) if l.bias]
    for w0, w1, (g, room) in zip(before, st.weights + st.biases, want):
        step = 0.25 * np.abs(g)
        assert (np.abs(w1 - (w0 - 0.25 * g)) <= 0.25 * room + 2 * U * (np.abs(w0) + step)).all()
    sess.close()


def test_a_summed_loss(ctx):
    """reduction="sum": the gradients of the mean times the number of outputs, a power of two here, so
    every rounding is the same."""
    rng = np.random.default_rng(1)
    batch, layers = 32, [Dense(12, 40, "tanh"), Dense(40, 8)]
    Ws = [(rng.standard_normal((l.fan_out, l.fan_in)) / 4).astype(np.float32) for l in layers]
    bs = [np.zeros(l.fan_out, np.float32) for l in layers]
    x, y = rng.standard_normal((batch, 12)).astype(np.float32), rng.standard_normal((batch, 8)).astype(np.float32)
    grads = []
    for reduction in ("mean", "sum"):
        sess = HipTrainingSession.open(ctx, MlpSpec(layers, "mse", reduction), Ws, bs, Sgd(0.1), batch,
                                       checkpoint="e4m3")
        sess.run(x, y, GradientMode.ACCUMULATE)
        grads.append(sess.state().accumulators)
        sess.close()
    for a, b in zip(*grads):
        assert np.array_equal(a * np.float32(batch * 8), b)
