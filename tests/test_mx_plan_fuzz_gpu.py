"""Random programs of microscaled and plain steps (tests/mx_programs.py) give the same bits on one
stream, on two, and replayed as a graph, with the programs' runs in turn."""
import numpy as np
import pytest

from synaptik_amd.native import HipProgram
from tests.mx_programs import random_program

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(24))
def test_random_microscaled_programs_on_one_and_two_streams(ctx, seed):
    pb, arrays, outs = random_program(seed)
    prog = HipProgram(ctx, pb.image())
    ins = [ctx.upload(a) for a in arrays]

    def run():
        bufs = [ctx.upload(np.full(s.count, 9.0, np.float32)) for s in outs]
        prog.run(ins, bufs)
        return [b.download().view(np.uint32) for b in bufs]

    prog.set_graph_mode(False)
    prog.set_concurrent(False)
    want = run()
    prog.set_concurrent(True)
    for graphs in (False, True, True, False):
        prog.set_graph_mode(graphs)
        for got, w in zip(run(), want):
            assert np.array_equal(got, w)
    prog.close()
