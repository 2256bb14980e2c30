"""What a server's states hold after a run that a token out of bounds fails."""
import numpy as np
import pytest

from synaptik_amd.native import HipBackendError, HipProgram
from synaptik_amd.program import ProgramBuilder
from tests import token_oracle as o

pytestmark = pytest.mark.gpu
B, D, V = 5, 40, 11


def step(in_place):
    """Z and U are rows of a table by token; one position."""
    pb = ProgramBuilder()
    table, tokens = pb.input(V * D), pb.input(B, "i32")
    state = pb.input(B * D, inout=in_place)
    z, h = pb.internal(B * D), pb.output(B * D)
    last = state if in_place else pb.output(B * D)
    pb.embed(table, tokens, z, B, V, D)
    pb.gated_scan(z, z, h, B, 1, D, h0=state, last=last)
    return pb


def moved(table, tokens, state):
    x = o.embed(table, tokens, 1.0)[:, None]
    _, last, _, off = o.gated_scan(x, x, state)
    return last, off


def arrays():
    rng = np.random.default_rng(0)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    good = rng.integers(0, V, B).astype(np.int32)
    bad = good.copy()
    bad[2] = V
    return f(V, D), f(B, D), good, bad


def test_states_in_place_have_moved_on(ctx):
    """Every request's: that of the token out of bounds by a row of zeros."""
    table, state, good, bad = arrays()
    prog = HipProgram(ctx, step(True).image())
    bt, bs, bh = ctx.upload(bad), ctx.upload(state), ctx.buffer(4 * B * D)
    with pytest.raises(HipBackendError, match="out of bounds"):
        prog.run([ctx.upload(table), bt, bs], [bh])
    want, off = moved(table, bad, state)
    o.within(bs.download().reshape(B, D), want, off)
    prog.close()


def test_states_from_one_buffer_to_another_can_be_repeated(ctx):
    """The first states are as they were; the run with its token mended moves every request on once."""
    table, state, good, bad = arrays()
    prog = HipProgram(ctx, step(False).image())
    tb, bt, bh = ctx.upload(table), ctx.upload(bad), ctx.buffer(4 * B * D)
    now, then = ctx.upload(state), ctx.buffer(4 * B * D)
    with pytest.raises(HipBackendError, match="out of bounds"):
        prog.run([tb, bt, now], [bh, then])
    assert np.array_equal(now.download().reshape(B, D), state)
    bt.upload(good)
    for _ in range(2):
        prog.run([tb, bt, now], [bh, then])
        want, off = moved(table, good, now.download().reshape(B, D))
        o.within(then.download().reshape(B, D), want, off)
        now, then = then, now
    prog.close()
