"""Microscaled steps without a device: argument checks, the arena they ask for, their place in the
two-stream schedule, and the 64-bit forms that the GPU tests compare with."""
import struct

import numpy as np
import pytest

from synaptik_amd.native import HipBackendError, HipInvalidArgument, program_plan, validate_program_image
from synaptik_amd.program import (MX_FORMAT, OP_MX_GEMM, ProgramBuilder, mx_code_bytes, mx_groups,
                                  mx_scale_bytes)
from tests import mx_oracle as mx


def steps():
    """name -> (builder of a valid step over fresh slots, its slots in step order)."""
    def encode(pb, R=3, C=130, **kw):
        pb.mx_encode(pb.input(R * C), pb.mx_tensor(R, C, kw.get("format", "e4m3"), "output"), R, C, **kw)

    def decode(pb, R=3, C=130, **kw):
        pb.mx_decode(pb.mx_tensor(R, C, "e4m3", "input"), pb.output(R * C), R, C, **kw)

    def act_grad(pb, R=3, C=130, **kw):
        pb.mx_act_grad(pb.input(R * C), pb.mx_tensor(R, C, "e4m3", "input"), pb.output(R * C), R, C,
                       act="relu", colsum=pb.output(C), **kw)

    def gemm(pb, M=5, N=130, K=7, **kw):
        pb.mx_gemm(pb.input(M * K), pb.mx_tensor(K, N, "e4m3", "input"), pb.output(M * N), M, N, K, **kw)

    def linear(pb, M=5, N=9, K=130, **kw):
        pb.mx_linear(pb.input(M * K), pb.mx_tensor(N, K, "e2m1", "input"), pb.output(M * N), M, N, K,
                     bias=pb.input(N), **kw)

    return dict(encode=encode, decode=decode, act_grad=act_grad, gemm=gemm, linear=linear)


NAMES = sorted(steps())


def built(name, **kw):
    pb = ProgramBuilder()
    steps()[name](pb, **kw)
    return pb


@pytest.mark.parametrize("name", NAMES)
def test_valid_steps_are_accepted(name):
    assert validate_program_image(built(name).image()) > 0


@pytest.mark.parametrize("name", NAMES)
def test_every_slot_is_checked(name):
    """A slot one byte short, of another type, out of range, missing, or read-only where written."""
    pb = built(name)
    used = [i for i in range(8) if pb.steps[0].slots[i] >= 0]
    for i in used:
        q = built(name)
        slot = q.slots[q.steps[0].slots[i]]
        optional = (name, i) in (("act_grad", 4), ("linear", 3))
        q.steps[0].slots[i] = -1
        if optional:
            validate_program_image(q.image())
        else:
            with pytest.raises(HipBackendError):
                validate_program_image(q.image())
        q = built(name)
        q.steps[0].slots[i] = 99
        with pytest.raises(HipBackendError):
            validate_program_image(q.image())
        q = built(name)
        slot = q.slots[q.steps[0].slots[i]]
        slot.count -= 1
        with pytest.raises(HipBackendError, match="bytes"):
            validate_program_image(q.image())
        q = built(name)
        slot = q.slots[q.steps[0].slots[i]]
        slot.dtype = "i32"
        with pytest.raises(HipBackendError):
            validate_program_image(q.image())
        q = built(name)
        slot = q.slots[q.steps[0].slots[i]]
        if slot.kind == 2:  # an output becomes an input
            slot.kind, slot.ext_index = 1, q.n_inputs
            for s in q.slots:
                if s.kind == 2 and s.index > slot.index:
                    s.ext_index -= 1
            with pytest.raises(HipBackendError, match="read-only"):
                validate_program_image(q.image())


@pytest.mark.parametrize("name", NAMES)
def test_extents_and_attributes_are_checked(name):
    extents = {"gemm": 3, "linear": 3}.get(name, 2)
    n_args = {"encode": 5, "decode": 4, "act_grad": 6, "gemm": 7, "linear": 8}[name]
    for i in range(n_args):
        for bad in (-1, -2 ** 62, 2 ** 31 + 5, 2 ** 62):
            q = built(name)
            q.steps[0].iargs[i] = bad
            with pytest.raises(HipBackendError):
                validate_program_image(q.image())
    for i in range(extents):  # an extent one larger than the slots hold
        q = built(name)
        q.steps[0].iargs[i] += 1
        if not ((name, i) in (("linear", 2), ("gemm", 2))):
            with pytest.raises(HipBackendError):
                validate_program_image(q.image())


def test_shared_slots_are_refused():
    pb = ProgramBuilder()
    t = pb.output(4096, "u8")
    pb.mx_encode(pb.input(128), (t, t), 1, 128)
    with pytest.raises(HipBackendError, match="share"):
        validate_program_image(pb.image())
    pb = ProgramBuilder()
    d, Y = pb.input(256, inout=True), pb.mx_tensor(2, 128, "e4m3", "input")
    pb.mx_act_grad(d, Y, d, 1, 128, act="relu", ldy=128, ldz=130)
    with pytest.raises(HipBackendError, match="aliases"):
        validate_program_image(pb.image())
    pb = ProgramBuilder()
    d, Y, z = pb.input(256), pb.mx_tensor(2, 128, "e4m3", "input"), pb.output(256)
    pb.mx_act_grad(d, Y, z, 2, 128, act="relu", colsum=z)
    with pytest.raises(HipBackendError, match="aliases"):
        validate_program_image(pb.image())
    pb = ProgramBuilder()
    a = pb.input(128 * 128, inout=True)
    pb.mx_gemm(a, pb.mx_tensor(128, 128, "e4m3", "input"), a, 128, 128, 128)
    with pytest.raises(HipBackendError, match="aliases"):
        validate_program_image(pb.image())
    pb = ProgramBuilder()
    a = pb.input(128 * 128, inout=True)
    pb.mx_linear(a, pb.mx_tensor(128, 128, "e2m1", "input"), a, 128, 128, 128)
    with pytest.raises(HipBackendError, match="aliases"):
        validate_program_image(pb.image())


def test_four_bits_cannot_keep_every_nonzero_value():
    with pytest.raises(HipInvalidArgument):
        validate_program_image(built("encode", format="e2m1", keep_nonzero=True).image())


def test_unknown_formats_and_kinds_are_refused():
    pb = ProgramBuilder()
    with pytest.raises(ValueError, match="format"):
        pb.mx_tensor(1, 1, "e3m2")
    with pytest.raises(ValueError, match="format"):
        pb.mx_encode(pb.input(1), (pb.input(1, "u8"), pb.input(1, "u8")), 1, 1, format="int8")
    with pytest.raises(KeyError):
        pb.mx_tensor(1, 1, "e4m3", "scratch")


def test_tensors_beyond_32_bit_ordinals_are_refused():
    for R, C in ((2 ** 31, 128), (1, 2 ** 31), (2 ** 20, 2 ** 20)):
        pb = ProgramBuilder()
        pb.mx_decode(pb.mx_tensor(R, C, "e2m1", "input"), pb.output(R * C), R, C)
        with pytest.raises(HipInvalidArgument):
            validate_program_image(pb.image())


def test_sizes_of_a_tensor():
    assert [mx_groups(c) for c in (0, 1, 128, 129, 1021)] == [0, 1, 1, 2, 8]
    assert mx_code_bytes(3, 129, "e4m3") == 3 * 256 and mx_code_bytes(3, 129, "e2m1") == 3 * 128
    assert mx_scale_bytes(3, 129) == 3 * 8


def test_empty_extents_are_accepted():
    for name, kw in (("encode", dict(R=0)), ("encode", dict(C=0)), ("decode", dict(R=0)),
                     ("act_grad", dict(R=0)), ("gemm", dict(K=0)), ("gemm", dict(M=0)),
                     ("gemm", dict(N=0)), ("linear", dict(K=0)), ("linear", dict(M=0)),
                     ("linear", dict(N=0))):
        validate_program_image(built(name, **kw).image())


# ---- the two-stream schedule ----
def mx_effects(opcode, slots):
    """(slots read, slots written) of a microscaled step, from what its kernels touch."""
    s = slots
    return {17: ({s[0]}, {s[1], s[2]}), 18: ({s[0], s[1]}, {s[2]}),
            19: ({s[0], s[1], s[2]}, {s[3], s[4]}), 20: ({s[0], s[1], s[2]}, {s[3]}),
            21: ({s[0], s[1], s[2], s[3]}, {s[4]})}[opcode]


def test_schedule_orders_conflicting_microscaled_steps():
    """Steps on two streams with one wait each: every pair that conflicts is ordered."""
    rng = np.random.default_rng(0)
    for _ in range(60):
        pb = ProgramBuilder()
        n = 64
        wide = [pb.input(n * n), pb.internal(n * n), pb.internal(n * n), pb.output(n * n)]
        narrow = [pb.mx_tensor(n, n, "e4m3", "input"), pb.mx_tensor(n, n, "e4m3"),
                  pb.mx_tensor(n, n, "e4m3")]
        for _ in range(12):
            kind = rng.integers(5)
            src, dst = wide[rng.integers(4)], wide[rng.integers(1, 4)]
            if src is dst:
                continue
            t = narrow[rng.integers(3)]
            if kind == 0:
                pb.mx_encode(src, narrow[rng.integers(1, 3)], n, n)
            elif kind == 1:
                pb.mx_decode(t, dst, n, n)
            elif kind == 2:
                pb.mx_act_grad(src, t, dst, n, n, act="relu")
            elif kind == 3:
                pb.mx_gemm(src, t, dst, n, n, n)
            else:
                pb.mx_linear(src, t, dst, n, n, n, w_format="e4m3")
        stream, wait, _ = program_plan(pb.image())
        ops = [mx_effects(s.opcode, [x if x >= 0 else None for x in s.slots]) for s in pb.steps]
        before = []  # per step, the steps known to be complete when it starts
        tail = [set(), set()]
        for j in range(len(ops)):
            done = set(tail[stream[j]])
            if wait[j] >= 0:
                done |= before[wait[j]] | {wait[j]}
            before.append(done)
            tail[stream[j]] = done | {j}
        for j, (rj, wj) in enumerate(ops):
            for i in range(j):
                ri, wi = ops[i]
                if ((wi & (rj | wj)) | (ri & wj)) - {None}:
                    assert i in before[j], (i, j, stream, wait)


# ---- the oracle ----
@pytest.mark.parametrize("format", mx.FORMATS)
def test_oracle_codes_are_nearest(format):
    """No other code of the block's scale is nearer, the scale is the smallest that holds the
    block, and a tie goes to the even code."""
    rng = np.random.default_rng(2)
    x = (rng.standard_normal((40, 64)) * np.exp2(rng.integers(-30, 30, (40, 1)))).astype(np.float32)
    code, scales = mx.encode(x, format)
    back = mx.values(code, scales, 64, format)
    t = mx.table(format)
    t = np.concatenate([-t[::-1], t])
    for r in range(40):
        for b in range(2):
            f = 2.0 ** (int(scales[r, b]) - 127)
            part = x[r, 32 * b:32 * b + 32].astype(np.float64)
            assert np.abs(part).max() <= t[-1] * f and np.abs(part).max() > t[-1] * f / 2
            near = np.abs(part[:, None] - t[None] * f).min(1)
            assert np.array_equal(np.abs(part - back[r, 32 * b:32 * b + 32]), near)
    assert mx.table("e4m3")[-1] == 448 and mx.table("e5m2")[-1] == 57344
    assert list(mx.table("e2m1")) == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
