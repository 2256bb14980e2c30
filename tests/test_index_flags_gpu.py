"""Indexes out of bounds, run after run: each run reports its own, by every way to run a program, and the next
one starts clear."""
import threading

import numpy as np
import pytest

from synaptik_amd.native import HipBackendError, HipProgram
from synaptik_amd.program import ProgramBuilder

pytestmark = pytest.mark.gpu


def embed(pb, N=9, V=7, D=5):
    st = pb.input(N, "i32")
    pb.embed(pb.input(V * D), st, pb.output(N * D), N, V, D)
    return st, np.full(N, V - 1, np.int32), V


def embed_grad(pb, N=9, V=7, D=5):
    st = pb.input(N, "i64")
    pb.embed_grad(pb.input(N * D), st, pb.output(V * D), N, V, D)
    return st, np.full(N, V - 1, np.int64), -1


def scan(pb, T=6, B=9, D=5):
    st = pb.input(B, "i64")
    pb.gated_scan(pb.input(B * T * D), pb.input(B * T * D), pb.output(B * T * D), B, T, D, lengths=st)
    return st, np.full(B, T, np.int64), T + 1


def scan_grad(pb, T=6, B=9, D=5):
    st = pb.input(B, "i32")
    n = B * T * D
    pb.gated_scan_grad(*(pb.input(n) for _ in range(4)), pb.output(n), pb.output(n), B, T, D, lengths=st)
    return st, np.full(B, T, np.int32), -1


def distill(pb, R=9, C=30):
    st = pb.input(R, "i32")
    pb.distill(pb.input(R * C), st, pb.input(R), pb.output(1), R, C, 1, grad=pb.output(R * C))
    return st, np.full(R, C - 1, np.int32), C


STEPS = dict(embed=embed, embed_grad=embed_grad, embed_grad_sorted=lambda pb: embed_grad(pb, 700),
             embed_grad_many=lambda pb: embed_grad(pb, 9000), scan=scan, scan_chunks=lambda pb: scan(pb, 1000, 2, 40),
             scan_grad=scan_grad, distill=distill, distill_many=lambda pb: distill(pb, 1200))


class Flagging:
    """A program of one such step (and `more` copies, which make it one that is replayed as a graph)."""

    def __init__(self, ctx, name, more=0):
        pb = ProgramBuilder()
        st, self.good, bad = STEPS[name](pb)
        for _ in range(more):
            pb.fill(pb.output(16), 16)
        self.bad = self.good.copy()
        self.bad[-1] = bad
        self.prog = HipProgram(ctx, pb.image())
        ins = [s for s in sorted((s for s in pb.slots if s.kind == 1), key=lambda s: s.ext_index)]
        outs = [s for s in sorted((s for s in pb.slots if s.kind == 2), key=lambda s: s.ext_index)]
        self.ins = [ctx.upload(self.good) if s is st else ctx.upload(np.zeros(s.nbytes // 4, np.float32)) for s in ins]
        self.at = [s is st for s in ins].index(True)
        self.outs = [ctx.buffer(s.nbytes) for s in outs]

    def bind(self, good):
        self.ins[self.at].upload(self.good if good else self.bad)


def expect(good, call):
    if good:
        call()
    else:
        with pytest.raises(HipBackendError, match="out of bounds"):
            call()


ORDER = [True, False, True, False, False, True, True]


@pytest.mark.parametrize("name", STEPS)
@pytest.mark.parametrize("more", [0, 7])
def test_each_run_reports_its_own(ctx, name, more):
    f = Flagging(ctx, name, more)
    for good in ORDER:
        f.bind(good)
        expect(good, lambda: f.prog.run(f.ins, f.outs))
    for good in ORDER:
        f.bind(good)
        f.prog.run_async(f.ins, f.outs)
        expect(good, f.prog.wait)
    for good in ORDER:
        f.bind(good)
        expect(good, lambda: f.prog.run_static(f.ins, f.outs))
    # the ways beside each other
    for good in ORDER:
        f.bind(good)
        expect(good, lambda: f.prog.run(f.ins, f.outs))
        expect(good, lambda: f.prog.run_static(f.ins, f.outs))
    f.prog.close()


def test_two_programs_share_the_static_run(ctx):
    """A failing one of either kind (its own host word, the published device word) beside a good one."""
    f, g = Flagging(ctx, "embed"), Flagging(ctx, "scan")
    pb = ProgramBuilder()
    N, C = 4, 6
    z, t, loss, dz = pb.input(N * C), pb.input(N, "i32"), pb.output(1), pb.output(N * C)
    pb.index_ce(z, t, loss, N, C, grad=dz)
    p = HipProgram(ctx, pb.image())
    bz, bt, outs = ctx.upload(np.zeros(N * C, np.float32)), ctx.upload(np.full(N, C, np.int32)), [ctx.buffer(s.nbytes) for s in pb.slots if s.kind == 2]
    for good in ORDER:
        f.bind(good)
        expect(False, lambda: p.run_static([bz, bt], outs))
        expect(good, lambda: f.prog.run_static(f.ins, f.outs))
        expect(True, lambda: g.prog.run_static(g.ins, g.outs))
    for x in (f.prog, g.prog, p):
        x.close()


@pytest.mark.parametrize("more", [0, 7])
def test_concurrent_runs_report_their_own(ctx, more):
    """Four threads on one program, two of them with tokens out of bounds: runs on different leases."""
    f = Flagging(ctx, "embed", more)
    errors = []

    def work(good):
        try:
            ins = list(f.ins)
            ins[f.at] = ctx.upload(f.good if good else f.bad)
            outs = [ctx.buffer(b.nbytes) for b in f.outs]
            for _ in range(20):
                expect(good, lambda: f.prog.run(ins, outs))
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k % 2 == 0,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    f.prog.close()


@pytest.mark.parametrize("N,D", [(0, 5), (3, 0)])
def test_programs_whose_steps_launch_nothing(ctx, N, D):
    pb = ProgramBuilder()
    pb.embed(pb.input(max(1, 7 * D)), pb.input(max(1, N), "i32"), pb.output(max(1, N * D)), N, 7, D)
    prog = HipProgram(ctx, pb.image())
    ins, outs = [ctx.buffer(4 * max(1, 7 * D)), ctx.upload(np.full(max(1, N), 99, np.int32))], [ctx.buffer(4 * max(1, N * D))]
    for _ in range(3):
        prog.run(ins, outs)
        prog.run_static(ins, outs)
    prog.close()


@pytest.mark.parametrize("bad", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("concurrent", [False, True])
def test_two_steps_of_one_program(ctx, bad, concurrent):
    """Either step's flag is reported, also where the two run beside each other; it is gone in the next run."""
    R, C = 50, 3000
    pb = ProgramBuilder()
    ins, outs = [], []
    for _ in range(2):
        ins += [pb.input(R * C), pb.input(R, "i32"), pb.input(R)]
        outs += [pb.output(1), pb.output(R * C)]
        pb.distill(*ins[-3:], outs[-2], R, C, 1, grad=outs[-1])
    prog = HipProgram(ctx, pb.image())
    prog.set_concurrent(concurrent)
    good, wrong = (ctx.upload(np.full(R, v, np.int32)) for v in (C - 1, C))
    z, t = ctx.upload(np.zeros(R * C, np.float32)), ctx.upload(np.zeros(R, np.float32))
    bo = [ctx.buffer(s.nbytes) for s in outs]
    for _ in range(10):
        expect(not any(bad), lambda: prog.run([z, wrong if bad[0] else good, t, z, wrong if bad[1] else good, t], bo))
        prog.run([z, good, t, z, good, t], bo)
    prog.close()
