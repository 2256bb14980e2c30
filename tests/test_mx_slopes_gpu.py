"""What 8-bit checkpoints do to the slopes of tanh and sigmoid units, and with them to a step's
gradients, against the uncompressed step."""
import numpy as np
import pytest

from synaptik_amd.program import ProgramBuilder
from synaptik_amd.training import GradientMode, HipTrainingSession, MlpSpec, Sgd, init_parameters
from tests import mx_oracle as mx
from tests.gpu_helpers import run_program

pytestmark = pytest.mark.gpu

# (the output from which on it is kept as 1, the kept value's largest error relative to it): codes
# between a half and one are 1/16 and 1/8 apart
FORMATS = {"e4m3": (1 - 1 / 32, 2.0 ** -4), "e5m2": (1 - 1 / 16, 2.0 ** -3)}


@pytest.mark.parametrize("act", ["tanh", "sigmoid"])
@pytest.mark.parametrize("format", FORMATS)
def test_slopes_vanish_from_a_threshold_on(ctx, format, act):
    """Outputs in steps of 2^-10: the slope of a kept output is zero from the threshold on, and not
    below it (but for sigmoid's zero)."""
    threshold = FORMATS[format][0]
    y = (np.arange(-1024 if act == "tanh" else 0, 1025) / 1024.0).astype(np.float32)
    n = y.size
    pb = ProgramBuilder()
    sy, one, kept, dz = pb.input(n), pb.input(n), pb.mx_tensor(1, n, format), pb.output(n)
    pb.mx_encode(sy, kept, 1, n, format=format, keep_nonzero=True)
    pb.mx_act_grad(one, kept, dz, 1, n, act=act, format=format)
    (slope,) = run_program(ctx, pb, [y, np.ones(n, np.float32)], [dz])
    gone = np.abs(y) >= threshold
    if act == "sigmoid":
        gone |= y == 0
    assert np.array_equal(slope == 0, gone)


@pytest.mark.parametrize("act", ["tanh", "sigmoid"])
@pytest.mark.parametrize("format", FORMATS)
def test_gradients_against_the_uncompressed_step(ctx, format, act):
    """One hidden layer with units on both sides of the threshold. Both steps have the same dY, so the
    cotangent of the hidden layer differs by |dY| times the slopes' difference, and W_1's and W_2's
    gradients by the cotangents' and the kept outputs' differences. With y^ = y + d and |d| <= r |y| +
    t, where t is the smallest code's size: 1 - y^2 moves by |d| |2 y + d|, y (1 - y) by |d| |1 - 2 y - d|.
    Binary32 sums beside it: both steps' products, 2 (3 n + 2) u of the magnitudes each (u = 2^-24)."""
    dims, batch = [12, 70, 9], 130
    spec = MlpSpec.chain(dims, hidden=act, loss="mse")
    Ws, bs = init_parameters(spec, 3, "xavier_uniform")
    rng = np.random.default_rng(2)
    x = (rng.standard_normal((batch, dims[0])) * 2).astype(np.float32)
    target = rng.standard_normal((batch, dims[2])).astype(np.float32)
    grads = []
    for checkpoint in (None, format):
        sess = HipTrainingSession.open(ctx, spec, Ws, bs, Sgd(0.1), batch, checkpoint=checkpoint)
        sess.run(x, target, GradientMode.ACCUMULATE)
        grads.append([a.astype(np.float64) for a in sess.state().accumulators])
        sess.close()
    W1, W2, b1, b2 = [np.asarray(v, np.float64) for v in (*Ws, *bs)]
    X = x.astype(np.float64)
    y = mx.activate(act, X @ W1.T + b1)
    dz2 = 2 * (y @ W2.T + b2 - target) / target.size
    dy = dz2 @ W2
    t = 2.0 ** -9 * 2.0 ** -8  # e4m3's smallest code under a scale of at most 2^-8 (e5m2's is less)
    d = FORMATS[format][1] * np.abs(y) + t
    moved = d * (2 * np.abs(y) + d) if act == "tanh" else d * (np.abs(1 - 2 * y) + d)
    assert (np.abs(y) >= FORMATS[format][0]).any() and (np.abs(y) < 0.5).any()
    u = 2.0 ** -24

    def room(a, b):  # a product's own binary32 sum, in both steps
        return 2 * 2 * (3 * a.shape[0] + 2) * u * (np.abs(a).T @ np.abs(b))
    dz1 = dy * mx.slope(act, y)
    # roundings upstream: of y, the logits, dz2, dy (depths 12, 70, 9) and the slope, in either step
    early = 64 * (12 + 70 + 9) * u * (np.abs(dz2) @ np.abs(W2) + np.abs(dy))
    bounds = [(np.abs(dy) * moved + early).T @ np.abs(X) + room(dz1, X),
              np.abs(dz2).T @ d + room(dz2, y) + 64 * 91 * u * (np.abs(dz2).sum(0)[:, None] + np.abs(dz2).T @ np.abs(y)),
              (np.abs(dy) * moved + early).sum(0)]
    for a, b, bound in zip(grads[0], grads[1], bounds):
        assert (np.abs(a - b).reshape(bound.shape) <= bound).all()
    # not a bound that everything passes: below the gradients themselves, as norms
    assert np.linalg.norm(bounds[1]) < np.linalg.norm(grads[0][1])
