"""The steps for models of tokens run together, as a training step and as a server use them: programs on
one and two streams, replayed graphs, concurrent and asynchronous runs, the no-allocation run."""
import threading

import numpy as np
import pytest

from synaptik_amd.native import HipBackendError, HipContext, HipProgram
from synaptik_amd.program import ProgramBuilder
from tests import token_oracle as o

pytestmark = pytest.mark.gpu


class Model:
    """Tokens -> embedding -> layer norm -> gates and inputs -> recurrence -> logits on the table (tied) ->
    divergence from a teacher, and the way back; `sizes`: sequences, positions, width, vocabulary, entries."""

    def __init__(self, sizes, seed=0, scale=4.0, T=2.0):
        self.B, self.T, self.D, self.V, self.K = B, T_, D, V, K = sizes
        self.scale, self.temperature = scale, T
        rng = np.random.default_rng(seed)
        f = lambda *s, by=1.0: (rng.standard_normal(s) * by).astype(np.float32)  # noqa: E731
        N = B * T_
        self.inputs = dict(
            E=f(V, D, by=0.3), gamma=1 + f(D, by=0.1), beta=f(D, by=0.1), Wz=f(D, D, by=D ** -0.5),
            Wu=f(D, D, by=D ** -0.5), bz=1 + f(D, by=0.3), h0=f(B, D, by=0.5),
            tokens=rng.integers(0, V, N).astype(np.int32), lengths=rng.integers(1, T_ + 1, B).astype(np.int32),
            index=np.stack([rng.permutation(V)[:K] for _ in range(N)]).astype(np.int32), teacher=f(N, K, by=2.0))
        inside = (np.arange(T_)[None] < self.inputs["lengths"][:, None]).reshape(-1)
        self.inputs["tokens"][~inside] = -1
        self.inputs["index"][~inside] = -1

    def build(self, pb):
        """The program's step; returns (input slots in order, output slots by name)."""
        B, T, D, V, K, N = self.B, self.T, self.D, self.V, self.K, self.B * self.T
        kinds = {"tokens": "i32", "lengths": "i32", "index": "i32"}
        s = {k: pb.input(v.size, kinds.get(k, "f32")) for k, v in self.inputs.items()}
        i = lambda n=N * D: pb.internal(n)  # noqa: E731
        out = {k: pb.output(n) for k, n in (("loss", 1), ("last", B * D), ("dE", V * D), ("dgamma", D), ("dbeta", D),
                                            ("dWz", D * D), ("dWu", D * D), ("dbz", D), ("dh0", B * D), ("h", N * D))}
        x, y, z, u, logits, dl = i(), i(), i(), i(), i(N * V), i(N * V)
        dh, dz, du, dy = i(), i(), i(), i()
        pb.embed(s["E"], s["tokens"], x, N, V, D, scale=self.scale, pad=-1)
        pb.layer_norm(x, y, N, D, gamma=s["gamma"], beta=s["beta"])
        pb.gemm(y, s["Wz"], z, N, D, D, trans_b=True, bias=s["bz"])
        pb.gemm(y, s["Wu"], u, N, D, D, trans_b=True)
        pb.gated_scan(z, u, out["h"], B, T, D, h0=s["h0"], last=out["last"], lengths=s["lengths"])
        pb.gemm(out["h"], s["E"], logits, N, V, D, trans_b=True)
        pb.distill(logits, s["index"], s["teacher"], out["loss"], N, V, K, grad=dl, temperature=self.temperature)
        pb.gemm(dl, s["E"], dh, N, D, V)
        pb.gemm(dl, out["h"], out["dE"], V, D, N, trans_a=True)
        pb.gated_scan_grad(dh, z, u, out["h"], dz, du, B, T, D, h0=s["h0"], dh0=out["dh0"], lengths=s["lengths"])
        pb.colsum(dz, out["dbz"], N, D)
        pb.gemm(dz, y, out["dWz"], D, D, N, trans_a=True)
        pb.gemm(du, y, out["dWu"], D, D, N, trans_a=True)
        pb.gemm(dz, s["Wz"], dy, N, D, D)
        pb.gemm(du, s["Wu"], dy, N, D, D, accumulate=True)
        pb.layer_norm_grad(dy, x, dy, N, D, gamma=s["gamma"], dgamma=out["dgamma"], dbeta=out["dbeta"])
        pb.embed_grad(dy, s["tokens"], out["dE"], N, V, D, scale=self.scale, pad=-1, accumulate=True)
        return list(s.values()), out

    def expected(self):
        """The same in 64 bits."""
        B, T, D, V, N = self.B, self.T, self.D, self.V, self.B * self.T
        p = {k: v.astype(np.float64) if v.dtype == np.float32 else v for k, v in self.inputs.items()}
        x = p["E"][np.maximum(p["tokens"], 0)] * self.scale * (p["tokens"] >= 0)[:, None]
        xh, rstd = o.normalised(x, 1e-5)
        y = xh * p["gamma"] + p["beta"]
        z, u = (y @ p["Wz"].T + p["bz"]).reshape(B, T, D), (y @ p["Wu"].T).reshape(B, T, D)
        h, last, _, _ = o.gated_scan(z, u, p["h0"], p["lengths"])
        logits = h.reshape(N, D) @ p["E"].T
        loss, dl, _, _ = o.distill(logits, p["index"], p["teacher"], self.temperature)
        dh = (dl @ p["E"]).reshape(B, T, D)
        (dz, du, dh0), _ = o.gated_scan_grad(dh, z, u, h, p["h0"], None, p["lengths"])
        dz, du = dz.reshape(N, D), du.reshape(N, D)
        dy = dz @ p["Wz"] + du @ p["Wu"]
        g = dy * p["gamma"]
        dx = rstd * (g - g.mean(1, keepdims=True) - xh * (g * xh).mean(1, keepdims=True))
        dE = dl.T @ h.reshape(N, D) + o.embed_grad(dx, p["tokens"], V, self.scale, -1)[0]
        return dict(loss=np.array([loss]), last=last, dE=dE, dgamma=(dy * xh).sum(0), dbeta=dy.sum(0), dWz=dz.T @ y,
                    dWu=du.T @ y, dbz=dz.sum(0), dh0=dh0, h=h)


SMALL, LARGE = (3, 21, 40, 97, 5), (4, 300, 192, 1021, 16)


def check(got, want):
    """A binary32 step is off by some 2^-24 of its terms and a chain of seventeen by the square root of
    their number more: 2e-5 of the result's norm leaves ten times that."""
    for k, w in want.items():
        off = np.linalg.norm(got[k].astype(np.float64) - w.reshape(-1)) / np.linalg.norm(w)
        assert off < 2e-5, (k, off)


@pytest.fixture(scope="module")
def large():
    m = Model(LARGE)
    return m, m.expected()


def bind(ctx, model):
    pb = ProgramBuilder()
    ins, outs = model.build(pb)
    prog = HipProgram(ctx, pb.image())
    return prog, [ctx.upload(v) for v in model.inputs.values()], {k: ctx.buffer(s.nbytes) for k, s in outs.items()}


def test_a_training_step(ctx, large):
    for model, want in ((Model(SMALL, 1), None), large):
        prog, ins, outs = bind(ctx, model)
        prog.run(ins, list(outs.values()))
        check({k: b.download() for k, b in outs.items()}, want or model.expected())
        prog.close()


def test_gradients_follow_differences():
    """The 64-bit form above against differences of its own loss: the chain is put together rightly."""
    m = Model((2, 5, 6, 11, 3), 4)
    for k in m.inputs:
        if m.inputs[k].dtype == np.float32:
            m.inputs[k] = m.inputs[k].astype(np.float64)
    want = m.expected()
    rng = np.random.default_rng(0)
    for name, grad in (("E", "dE"), ("gamma", "dgamma"), ("beta", "dbeta"), ("Wz", "dWz"), ("Wu", "dWu"), ("bz", "dbz"),
                       ("h0", "dh0")):
        base = m.inputs[name]
        for i in rng.permutation(base.size)[:6]:
            side = []
            for h in (1e-6, -1e-6):
                m.inputs[name] = base.copy()
                m.inputs[name].reshape(-1)[i] += h
                side.append(m.expected()["loss"][0])
            m.inputs[name] = base
            assert np.isclose((side[0] - side[1]) / 2e-6, want[grad].reshape(-1)[i], atol=1e-7), (name, i)


def test_one_and_two_streams_and_graphs_give_the_same_bits(ctx, large):
    model, want = large
    prog, ins, outs = bind(ctx, model)
    seen = []
    for graphs in (False, True):
        for streams in (False, True):
            prog.set_graph_mode(graphs)
            prog.set_concurrent(streams)
            for _ in range(4 if graphs else 2):
                for b in outs.values():
                    b.upload(np.full(b.nbytes // 4, np.nan, np.float32))
                prog.run(ins, list(outs.values()))
                seen.append({k: b.download() for k, b in outs.items()})
    assert prog.side_steps() > 0
    for s in seen[1:]:
        for k in s:
            assert np.array_equal(s[k], seen[0][k]), k
    check(seen[0], want)
    prog.close()


def test_replayed_graphs_see_new_inputs(ctx):
    """A captured step replayed over changed inputs, with other work between the replays."""
    model = Model(SMALL, 2)
    prog, ins, outs = bind(ctx, model)
    prog.set_graph_mode(True)
    for seed in (2, 3, 4, 2):
        other = Model(SMALL, seed)
        for b, v in zip(ins, other.inputs.values()):
            b.upload(v)
        prog.run(ins, list(outs.values()))
        check({k: b.download() for k, b in outs.items()}, other.expected())
        ctx.upload(np.zeros(100, np.float32)).download()
    prog.close()


def test_concurrent_and_asynchronous_runs(ctx, large):
    """Threads that run one program at once on buffers of their own; and asynchronous runs in a row."""
    model, want = large
    prog, ins, outs = bind(ctx, model)
    prog.run(ins, list(outs.values()))
    first = {k: b.download() for k, b in outs.items()}
    errors = []

    def work():
        try:
            mine = {k: ctx.buffer(b.nbytes) for k, b in outs.items()}
            for _ in range(3):
                prog.run(ins, list(mine.values()))
                for k, b in mine.items():
                    assert np.array_equal(b.download(), first[k]), k
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for _ in range(3):
        prog.run_async(ins, list(outs.values()))
        prog.wait()
        for k, b in outs.items():
            assert np.array_equal(b.download(), first[k]), k
    prog.close()


def test_the_run_that_allocates_nothing(ctx):
    model = Model(SMALL, 5)
    prog, ins, outs = bind(ctx, model)
    prog.run_static(ins, list(outs.values()))
    got = {k: b.download() for k, b in outs.items()}
    check(got, model.expected())
    prog.run(ins, list(outs.values()))
    for k, b in outs.items():
        assert np.array_equal(b.download(), got[k]), k
    prog.close()


def test_two_contexts(ctx):
    """The same step in another context, beside this one's."""
    model = Model(SMALL, 6)
    prog, ins, outs = bind(ctx, model)
    prog.run(ins, list(outs.values()))
    first = {k: b.download() for k, b in outs.items()}
    with HipContext(0) as other:
        p2, i2, o2 = bind(other, model)
        p2.run(i2, list(o2.values()))
        for k, b in o2.items():
            assert np.array_equal(b.download(), first[k]), k
        p2.close()
        del i2, o2
    prog.close()


def test_a_failing_token_leaves_the_optimizer_step_undone(ctx):
    """A training step with a staged update: a token out of bounds fails the run, and the step counter
    does not advance."""
    N, V, D = 6, 9, 8
    rng = np.random.default_rng(0)
    pb = ProgramBuilder()
    W, tokens, y = pb.input(V * D), pb.input(N, "i32"), pb.internal(N * D)
    counter, nxt = pb.input(1, "i64", inout=True), pb.output(V * D)
    dW = pb.internal(V * D)
    pb.embed(W, tokens, y, N, V, D)
    pb.embed_grad(y, tokens, dW, N, V, D)
    pb.optimizer(counter, [(W, dW, None, None, nxt, None, None, V * D)], kind="sgd", phase=2, lr=0.5)
    pb.step_commit(counter)
    prog = HipProgram(ctx, pb.image())
    w = rng.standard_normal((V, D)).astype(np.float32)
    bw, bt, bc, bn = ctx.upload(w), ctx.upload(np.array([0, 1, 1, 2, 9, 8], np.int32)), ctx.upload(np.zeros(1, np.int64)), ctx.buffer(4 * V * D)
    with pytest.raises(HipBackendError, match="out of bounds"):
        prog.run([bw, bt, bc], [bn])
    assert bc.download(np.int64)[0] == 0
    good = np.array([0, 1, 1, 2, 7, 8], np.int32)
    bt.upload(good)
    prog.run([bw, bt, bc], [bn])
    assert bc.download(np.int64)[0] == 1
    dw, _ = o.embed_grad(w[good], good, V, 1.0)
    assert np.allclose(bn.download().reshape(V, D), w - 0.5 * dw, atol=1e-5)
    prog.close()


def test_a_server_moves_its_requests_on(ctx):
    """Token by token with states in place: the same hidden states as the whole sequences at once."""
    B, T, D, V = 5, 9, 70, 31
    rng = np.random.default_rng(1)
    E, W, b = (rng.standard_normal(s).astype(np.float32) for s in ((V, D), (2 * D, D), (2 * D,)))
    tokens = rng.integers(0, V, (B, T)).astype(np.int32)
    x = o.normalised(E[tokens.reshape(-1)], 1e-5)[0]
    zu = (x @ W.T.astype(np.float64) + b).reshape(B, T, 2 * D)
    want, last, _, _ = o.gated_scan(zu[..., :D], zu[..., D:])
    pb = ProgramBuilder()
    sE, sWz, sWu, sbz, sbu, st = (pb.input(V * D), pb.input(D * D), pb.input(D * D), pb.input(D), pb.input(D),
                                  pb.input(B, "i32"))
    state, h = pb.input(B * D, inout=True), pb.output(B * D)
    x1, z, u = pb.internal(B * D), pb.internal(B * D), pb.internal(B * D)
    pb.embed(sE, st, x1, B, V, D)
    pb.layer_norm(x1, x1, B, D)
    pb.gemm(x1, sWz, z, B, D, D, trans_b=True, bias=sbz)
    pb.gemm(x1, sWu, u, B, D, D, trans_b=True, bias=sbu)
    pb.gated_scan(z, u, h, B, 1, D, h0=state, last=state)
    prog = HipProgram(ctx, pb.image())
    bt, bs, bh = ctx.upload(tokens[:, 0].copy()), ctx.upload(np.zeros(B * D, np.float32)), ctx.buffer(4 * B * D)
    ins = [ctx.upload(a) for a in (E, W[:D], W[D:], b[:D], b[D:])] + [bt, bs]
    for t in range(T):
        bt.upload(tokens[:, t].copy())
        prog.run(ins, [bh])
        got = bh.download().reshape(B, D)
        assert np.linalg.norm(got - want[:, t]) < 2e-5 * np.linalg.norm(want[:, t])
    assert np.linalg.norm(bs.download().reshape(B, D) - last) < 2e-5 * np.linalg.norm(last)
    prog.close()


@pytest.mark.parametrize("name", ["embed_grad", "norm_grad", "scan", "scan_grad", "distill"])
def test_repeated_runs_give_the_same_bits(ctx, name):
    """At sizes where a step takes several launches."""
    rng = np.random.default_rng(7)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    pb = ProgramBuilder()
    if name == "embed_grad":
        N, V, D = 30000, 5000, 300
        t = np.minimum(rng.geometric(0.01, N), V - 1).astype(np.int32)
        arrays = [f(N, D), t]
        ins, outs = [pb.input(N * D), pb.input(N, "i32")], [pb.output(V * D)]
        pb.embed_grad(*ins, outs[0], N, V, D)
    elif name == "norm_grad":
        R, C = 5000, 1100
        arrays = [f(R, C), f(R, C), f(C)]
        ins, outs = [pb.input(R * C), pb.input(R * C), pb.input(C)], [pb.output(R * C), pb.output(C), pb.output(C)]
        pb.layer_norm_grad(ins[0], ins[1], outs[0], R, C, gamma=ins[2], dgamma=outs[1], dbeta=outs[2])
    elif name.startswith("scan"):
        B, T, D = 2, 3000, 130
        n = B * T * D
        arrays = [f(n) for _ in range(4 if name == "scan_grad" else 2)]
        ins = [pb.input(n) for _ in arrays]
        outs = [pb.output(n), pb.output(n)] if name == "scan_grad" else [pb.output(n), pb.output(B * D)]
        if name == "scan":
            pb.gated_scan(*ins, outs[0], B, T, D, last=outs[1])
        else:
            pb.gated_scan_grad(*ins, *outs, B, T, D)
    else:
        R, C, K = 3000, 5000, 20
        arrays = [f(R, C), rng.integers(-1, C, (R, K)), f(R, K)]
        ins = [pb.input(R * C), pb.input(R * K, "i64"), pb.input(R * K)]
        outs = [pb.output(1), pb.output(R * C)]
        pb.distill(*ins, outs[0], R, C, K, grad=outs[1])
    prog = HipProgram(ctx, pb.image())
    bi, bo = [ctx.upload(a) for a in arrays], [ctx.buffer(s.nbytes) for s in outs]
    seen = None
    for _ in range(5):
        prog.run(bi, bo)
        got = [b.download() for b in bo]
        assert seen is None or all(np.array_equal(a, b) for a, b in zip(got, seen))
        seen = got
    prog.close()
