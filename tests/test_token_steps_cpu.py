"""Embeddings, layer norm, gated recurrences and distillation without a device: argument checks, the
arena they ask for, their place in the two-stream schedule, and the 64-bit forms that the GPU tests
compare with, against differences."""
import struct

import numpy as np
import pytest

from synaptik_amd.native import HipBackendError, HipInvalidArgument, program_plan, validate_program_image
from synaptik_amd.program import ProgramBuilder
from tests import token_oracle as o


def embed(pb, N=5, V=9, D=7, **kw):
    pb.embed(pb.input(V * D), pb.input(N, "i32"), pb.output(N * D), N, V, D, **kw)


def embed_grad(pb, N=5, V=9, D=7, **kw):
    pb.embed_grad(pb.input(N * D), pb.input(N, "i64"), pb.output(V * D), N, V, D, **kw)


def layer_norm(pb, R=5, C=7, **kw):
    pb.layer_norm(pb.input(R * C), pb.output(R * C), R, C, gamma=pb.input(C), beta=pb.input(C), **kw)


def layer_norm_grad(pb, R=5, C=7, **kw):
    pb.layer_norm_grad(pb.input(R * C), pb.input(R * C), pb.output(R * C), R, C, gamma=pb.input(C),
                       dgamma=pb.output(C), dbeta=pb.output(C), **kw)


def gated_scan(pb, B=3, T=5, D=7):
    n = B * T * D
    pb.gated_scan(pb.input(n), pb.input(n), pb.output(n), B, T, D, h0=pb.input(B * D), last=pb.output(B * D),
                  lengths=pb.input(B, "i32"))


def gated_scan_grad(pb, B=3, T=5, D=7):
    n = B * T * D
    pb.gated_scan_grad(pb.input(n), pb.input(n), pb.input(n), pb.input(n), pb.output(n), pb.output(n), B, T, D,
                       h0=pb.input(B * D), dlast=pb.input(B * D), dh0=pb.output(B * D), lengths=pb.input(B, "i64"))


def distill(pb, R=5, C=11, K=3, **kw):
    pb.distill(pb.input(R * C), pb.input(R * K, "i32"), pb.input(R * K), pb.output(1), R, C, K,
               grad=pb.output(R * C), **kw)


STEPS = dict(embed=embed, embed_grad=embed_grad, layer_norm=layer_norm, layer_norm_grad=layer_norm_grad,
             gated_scan=gated_scan, gated_scan_grad=gated_scan_grad, distill=distill)
NAMES = sorted(STEPS)
OPTIONAL = {"layer_norm": {1, 2}, "layer_norm_grad": {2, 4, 5}, "gated_scan": {2, 3, 5}, "gated_scan_grad": {4, 5},
            "distill": {4}}
EXTENTS = {"embed": 3, "embed_grad": 3, "layer_norm": 2, "layer_norm_grad": 2}


def built(name, **kw):
    pb = ProgramBuilder()
    STEPS[name](pb, **kw)
    return pb


def refused(pb, match=None):
    with pytest.raises(HipBackendError, match=match):
        validate_program_image(pb.image())


@pytest.mark.parametrize("name", NAMES)
def test_valid_steps_are_accepted(name):
    assert validate_program_image(built(name).image()) > 0


@pytest.mark.parametrize("name", NAMES)
def test_every_slot_is_checked(name):
    """A slot one element short, of another type, out of range, missing, or read-only where written."""
    for i in (i for i in range(8) if built(name).steps[0].slots[i] >= 0):
        pb = built(name)
        pb.steps[0].slots[i] = -1
        if i in OPTIONAL.get(name, ()):
            validate_program_image(pb.image())
        else:
            refused(pb, "missing")
        pb = built(name)
        pb.steps[0].slots[i] = 99
        refused(pb, "out of range")
        pb = built(name)
        pb.slots[pb.steps[0].slots[i]].count -= 1
        refused(pb, "bytes")
        for other in ("u8", "f64"):
            pb = built(name)
            pb.slots[pb.steps[0].slots[i]].dtype = other
            refused(pb, "dtype")
        pb = built(name)
        slot = pb.slots[pb.steps[0].slots[i]]
        if slot.kind == 2:  # an output becomes an input
            slot.kind, slot.ext_index = 1, pb.n_inputs
            for s in pb.slots:
                if s.kind == 2 and s.index > slot.index:
                    s.ext_index -= 1
            refused(pb, "read-only")


def test_the_slots_of_a_payload_are_checked():
    def with_entry(dh0, lengths, short=False):
        pb = built("gated_scan_grad")
        pb.steps[0].payload = struct.pack("<ii", dh0, lengths)[:4 if short else 8]
        return pb

    dh0, lengths = struct.unpack("<ii", built("gated_scan_grad").steps[0].payload)
    validate_program_image(with_entry(dh0, lengths).image())
    validate_program_image(with_entry(-1, -1).image())
    for bad in (with_entry(99, lengths), with_entry(dh0, 99), with_entry(lengths, lengths), with_entry(dh0, dh0),
                with_entry(dh0, lengths, True), with_entry(0, lengths), with_entry(6, lengths)):
        refused(bad)
    pb = built("gated_scan_grad")
    pb.slots[dh0].count -= 1
    refused(pb, "bytes")
    pb = built("gated_scan_grad")
    pb.slots[lengths].dtype = "i32"
    refused(pb, "dtype")
    for name in NAMES:
        if name != "gated_scan_grad":
            pb = built(name)
            pb.steps[0].payload = b"\0" * 8
            refused(pb, "payload")


@pytest.mark.parametrize("name", NAMES)
def test_extents_and_attributes_are_checked(name):
    used = {"embed": [0, 1, 2, 3, 4, 5], "embed_grad": [0, 1, 2, 3, 4, 5, 7], "layer_norm": range(4),
            "layer_norm_grad": range(5)}.get(name, range(4))
    for i in used:
        for bad in (-1, -2 ** 62, 2 ** 31 + 5, 2 ** 62, -2 ** 63, 2 ** 63 - 1):
            pb = built(name)
            pb.steps[0].iargs[i] = bad
            refused(pb)
    for i in range(EXTENTS.get(name, 3)):  # one larger than the slots hold
        pb = built(name)
        pb.steps[0].iargs[i] += 1
        refused(pb)


@pytest.mark.parametrize("eps", [-1e-9, float("nan"), float("inf")])
def test_epsilons_that_are_no_epsilons(eps):
    for name in ("layer_norm", "layer_norm_grad"):
        with pytest.raises(HipInvalidArgument, match="norm"):
            validate_program_image(built(name, eps=eps).image())


@pytest.mark.parametrize("T", [0.0, -1.0, float("nan"), float("inf"), 1e-45])
def test_temperatures_that_are_none(T):
    with pytest.raises(HipInvalidArgument, match="distill"):
        validate_program_image(built("distill", temperature=T).image())


def test_more_entries_than_a_row_may_have():
    validate_program_image(built("distill", C=2000, K=1024).image())
    with pytest.raises(HipInvalidArgument, match="entries"):
        validate_program_image(built("distill", C=2000, K=1025).image())


def test_shared_slots():
    """Written slots are no other operand's, but where a row or a state may be replaced."""
    def norm(ldx, ldy):
        pb = ProgramBuilder()
        s = pb.input(100, inout=True)
        pb.layer_norm(s, s, 5, 7, ldx=ldx, ldy=ldy)
        return pb

    validate_program_image(norm(9, 9).image())
    refused(norm(9, 10), "aliases")

    def norm_grad(lddy, lddx):
        pb = ProgramBuilder()
        s = pb.input(100, inout=True)
        pb.layer_norm_grad(s, pb.input(35), s, 5, 7, lddy=lddy, lddx=lddx)
        return pb

    validate_program_image(norm_grad(9, 9).image())
    refused(norm_grad(9, 10), "aliases")
    # the pairs of slots that may be one
    allowed = {("layer_norm", 0, 3), ("layer_norm_grad", 0, 3), ("gated_scan", 2, 5)}
    for name in NAMES:
        pb = built(name)
        slots = [i for i in range(8) if pb.steps[0].slots[i] >= 0]
        for w in (i for i in slots if pb.slots[pb.steps[0].slots[i]].kind == 2):
            for r in (i for i in slots if i != w):
                pb = ProgramBuilder()
                STEPS[name](pb)
                for s in pb.slots:  # large enough for any operand, all writable
                    s.kind, s.ext_index, s.count = 0, 0, 4096
                a, b = pb.slots[pb.steps[0].slots[r]], pb.slots[pb.steps[0].slots[w]]
                if a.dtype != b.dtype:
                    continue
                pb.steps[0].slots[w] = pb.steps[0].slots[r]
                if (name, *sorted((w, r))) in allowed:
                    validate_program_image(pb.image())
                else:
                    refused(pb, "aliases")
    pb = ProgramBuilder()
    ins = [pb.input(35) for _ in range(4)]
    state = pb.input(7, inout=True)
    pb.gated_scan_grad(*ins, pb.output(35), pb.output(35), 1, 5, 7, dlast=state, dh0=state)
    validate_program_image(pb.image())
    refused_h0 = ProgramBuilder()
    ins = [refused_h0.input(35) for _ in range(4)]
    state = refused_h0.input(7, inout=True)
    refused_h0.gated_scan_grad(*ins, refused_h0.output(35), refused_h0.output(35), 1, 5, 7, h0=state, dh0=state)
    refused(refused_h0, "aliases")


@pytest.mark.parametrize("name,kw", [("embed", dict(N=0)), ("embed", dict(D=0)), ("embed", dict(V=0)), ("embed_grad", dict(N=0)),
                                     ("embed_grad", dict(V=0)), ("embed_grad", dict(D=0)), ("layer_norm", dict(R=0)),
                                     ("layer_norm", dict(C=0)), ("layer_norm_grad", dict(R=0)),
                                     ("layer_norm_grad", dict(C=0)), ("gated_scan", dict(B=0)), ("gated_scan", dict(T=0)),
                                     ("gated_scan", dict(D=0)), ("gated_scan_grad", dict(B=0)),
                                     ("gated_scan_grad", dict(T=0)), ("distill", dict(R=0))], ids=str)
def test_empty_extents_are_accepted(name, kw):
    validate_program_image(built(name, **kw).image())


def test_empty_rows_are_refused():
    for kw in (dict(C=0, K=1), dict(K=0)):
        refused(built("distill", **kw))


def test_extents_whose_products_leave_64_bits():
    for name, at in (("embed", (0, 2)), ("embed_grad", (1, 2)), ("layer_norm", (0, 1)), ("layer_norm_grad", (0, 1)),
                     ("gated_scan", (0, 1, 2)), ("gated_scan_grad", (0, 1, 2)), ("distill", (0, 1))):
        pb = built(name)
        for i in at:
            pb.steps[0].iargs[i] = 2 ** 31 - 1025
        refused(pb)


# ---- the two-stream schedule ----
def effects(step, payload):
    """(slots read, slots written, whether the status word may be flagged), from what the kernels touch."""
    s = step.slots
    if step.opcode == 22:
        return {s[0], s[1]}, {s[2]}, True
    if step.opcode == 23:
        return {s[0], s[1]} | ({s[2]} if step.iargs[7] else set()), {s[2]}, True
    if step.opcode == 24:
        return {s[0], s[1], s[2]}, {s[3]}, False
    if step.opcode == 25:
        return {s[0], s[1], s[2]}, {s[3], s[4], s[5]}, False
    if step.opcode == 26:
        return {s[0], s[1], s[2], s[3]}, {s[4], s[5]}, s[3] >= 0
    if step.opcode == 27:
        dh0, lengths = struct.unpack("<ii", payload)
        return set(s[:6]) | {lengths}, {s[6], s[7], dh0}, lengths >= 0
    if step.opcode == 28:
        return {s[0], s[1], s[2]}, {s[3], s[4]}, True
    assert step.opcode in (1, 12)  # a product, the step commit
    return ({s[0], s[1]}, {s[2]}, False) if step.opcode == 1 else ({s[0]}, {s[0]}, False)


def test_schedule_orders_conflicting_steps():
    """Steps on two streams with one wait each: every pair that conflicts is ordered."""
    rng = np.random.default_rng(0)
    sides = 0
    for _ in range(80):
        pb = ProgramBuilder()
        n = 64
        wide = [pb.input(n * n), pb.internal(n * n), pb.internal(n * n), pb.internal(n * n), pb.output(n * n)]
        rows = [pb.input(n, inout=True), pb.internal(n), pb.internal(n)]
        ids, many, loss = pb.input(n, "i32"), pb.input(n * 4, "i64"), pb.output(1)

        def distinct(pool, k):
            return [pool[i] for i in rng.permutation(len(pool))[:k]]

        for _ in range(14):
            w = distinct(wide[1:], 3)
            src = wide[rng.integers(5)]
            if src in w[:2]:
                src = wide[0]
            r = distinct(rows, 3)
            kind = rng.integers(8)
            if kind == 0:
                pb.embed(src, ids, w[0], n, n, n)
            elif kind == 1:
                pb.embed_grad(src, ids, w[0], n, n, n, accumulate=bool(rng.integers(2)))
            elif kind == 2:
                pb.layer_norm(src, w[0], n, n, gamma=r[0], beta=r[1])
            elif kind == 3:
                pb.layer_norm_grad(src, wide[0], w[0], n, n, gamma=r[0], dgamma=r[1], dbeta=r[2])
            elif kind == 4:
                pb.gated_scan(src, wide[0], w[0], 1, n, n, h0=r[0], last=r[0])
            elif kind == 5:
                pb.gated_scan_grad(src, wide[0], wide[0], src, w[0], w[1], 1, n, n, h0=r[0], dlast=r[1], dh0=r[2])
            elif kind == 6:
                pb.distill(src, many, wide[0], loss, n, n, 4, grad=w[0])
            else:
                pb.gemm(src, wide[0], w[0], n, n, n)
        stream, wait, _ = program_plan(pb.image())
        sides += sum(stream)
        ops = [effects(s, s.payload) for s in pb.steps]
        before, tail = [], [set(), set()]
        for j in range(len(ops)):
            done = set(tail[stream[j]])
            if wait[j] >= 0:
                done |= before[wait[j]] | {wait[j]}
            before.append(done)
            tail[stream[j]] = done | {j}
        for j, (rj, wj, _) in enumerate(ops):
            for i in range(j):
                ri, wi, _ = ops[i]
                if ((wi & (rj | wj)) | (ri & wj)) - {-1}:
                    assert i in before[j], (i, j, stream, wait)
    assert sides > 0


def test_a_step_commit_follows_what_may_flag_the_run():
    """The commit inside a program waits for every step that can flag the status word."""
    for name in NAMES:
        pb = ProgramBuilder()
        pb.fill(pb.output(4), 4)
        STEPS[name](pb)
        counter = pb.input(1, "i64", inout=True)
        pb.step_commit(counter)
        pb.fill(pb.output(4), 4)  # (a trailing commit is part of the run's last launch)
        stream, wait, _ = program_plan(pb.image())
        flags = effects(pb.steps[1], pb.steps[1].payload)[2]
        if flags:
            assert stream[1] == stream[2] or wait[2] >= 1


# ---- the 64-bit forms against differences ----
def differences(f, x, at, h=1e-6):
    out = []
    for i in at:
        a, b = x.copy(), x.copy()
        a.reshape(-1)[i] += h
        b.reshape(-1)[i] -= h
        out.append((f(a) - f(b)) / (2 * h))
    return np.array(out)


def test_layer_norm_grad_is_the_derivative():
    rng = np.random.default_rng(0)
    x, dy, gamma, beta = (rng.standard_normal(s) for s in ((4, 9), (4, 9), 9, 9))
    (dx, dg, db), _ = o.layer_norm_grad(dy, x, gamma, 1e-3)
    f = lambda x, g, b: (o.layer_norm(x, g, b, 1e-3)[0] * dy).sum()  # noqa: E731
    assert np.allclose(differences(lambda v: f(v, gamma, beta), x, range(36)), dx.reshape(-1), atol=1e-7)
    assert np.allclose(differences(lambda v: f(x, v, beta), gamma, range(9)), dg, atol=1e-7)
    assert np.allclose(differences(lambda v: f(x, gamma, v), beta, range(9)), db, atol=1e-7)


@pytest.mark.parametrize("lengths", [None, [6, 0, 3]])
def test_gated_scan_grad_is_the_derivative(lengths):
    rng = np.random.default_rng(1)
    z, u, dh = (rng.standard_normal((3, 6, 4)) for _ in range(3))
    h0, dlast = rng.standard_normal((3, 4)), rng.standard_normal((3, 4))

    def f(z, u, h0):
        h, last, _, _ = o.gated_scan(z, u, h0, lengths)
        return (h * dh).sum() + (last * dlast).sum()

    h = o.gated_scan(z, u, h0, lengths)[0]
    (dz, du, dh0), _ = o.gated_scan_grad(dh, z, u, h, h0, dlast, lengths)
    assert np.allclose(differences(lambda v: f(v, u, h0), z, range(72)), dz.reshape(-1), atol=1e-7)
    assert np.allclose(differences(lambda v: f(z, v, h0), u, range(72)), du.reshape(-1), atol=1e-7)
    assert np.allclose(differences(lambda v: f(z, u, v), h0, range(12)), dh0.reshape(-1), atol=1e-7)


def test_distill_grad_is_the_derivative():
    rng = np.random.default_rng(2)
    z, t = rng.standard_normal((5, 7)), rng.standard_normal((5, 3))
    index = np.array([[0, 1, 2], [6, -1, 6], [-1, -1, -1], [3, 4, -1], [5, 0, 2]])
    t[4, 1] = -np.inf
    loss, grad, _, _ = o.distill(z, index, t, 2.0, 1.5)
    assert np.allclose(1.5 * differences(lambda v: o.distill(v, index, t, 2.0)[0], z, range(35)), grad.reshape(-1), atol=1e-7)
    # a teacher that is the model has no divergence
    full = np.tile(np.arange(7), (5, 1))
    loss, grad, _, _ = o.distill(z, full, z, 2.0)
    assert abs(loss) < 1e-12 and np.abs(grad).max() < 1e-12


def test_embed_grad_is_the_transpose():
    rng = np.random.default_rng(3)
    W, dY = rng.standard_normal((6, 3)).astype(np.float32), rng.standard_normal((10, 3)).astype(np.float32)
    tokens = rng.integers(-1, 6, 10)
    dW, _ = o.embed_grad(dY, tokens, 6, 0.5, pad=2)
    y = o.embed(W, tokens, 0.5, pad=2)
    assert np.isclose((y.astype(np.float64) * dY).sum(), (dW * W).sum())


# ---- hostile images ----
def test_hostile_images_are_refused_or_accepted_without_a_trap():
    """Two hostile extents at once: whatever is accepted asks for an arena that the extents explain."""
    hostile = [-(1 << 63), -1, 0, 1, (1 << 31) - 1, 1 << 31, 1 << 40, (1 << 63) - 1]
    for name in NAMES:
        for i in range(8):
            for j in range(i):
                for a in hostile:
                    for b in hostile:
                        pb = built(name)
                        pb.steps[0].iargs[i], pb.steps[0].iargs[j] = a, b
                        try:
                            assert validate_program_image(pb.image()) < 1 << 24
                        except HipBackendError:
                            pass
