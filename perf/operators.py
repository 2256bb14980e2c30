"""Operators of microscaled tensors: what is measured of them, with plain forms beside the
framework's own.

A microscaled tensor holds, for each row, groups of 128 values as codes of 8 or 4 bits (e4m3, e5m2,
e2m1), with one power of two for every 32 consecutive values of the row. A code byte and a scale
byte s stand for value(code) * 2^(s - 127).

Kinds of case (the "kind" entry):
  store       a matrix is encoded and restored: what a training step keeps of an activation between
              its forward and its backward pass, or a server of a weight (ProgramBuilder.mx_encode,
              mx_decode);
  linear      Y = act(X . W^T + b) of microscaled weights and of activations that are encoded on
              the way (ProgramBuilder.mx_linear);
  backward    the backward pass of one trained layer from what was kept in 8 bits: the cotangent
              dZ = act'(dY, Y), its column sums and the weight gradient dW = dZ^T . X
              (ProgramBuilder.mx_act_grad, mx_gemm);
  input_grad  dX = dZ . W through microscaled weights (ProgramBuilder.mx_gemm).

Inputs, weights and outputs are in GPU memory when a pass begins; a pass is the synchronous call
that a program makes.
"""
from __future__ import annotations

import math

import torch

own = False

# format: (exponent of the largest binade, mantissa bits, exponent of the smallest normal value,
# mantissa of the largest value as 23 bits)
_FORMATS = {"e4m3": (8, 3, -6, 0x600000), "e5m2": (15, 2, -14, 0x600000),
            "e2m1": (2, 1, 0, 0x400000)}
_LEAST_SCALE = -110  # exponent: every value a code stands for is then a normal float


def listed():
    return [
        # One position's activations, kept or handed on: latency alone.
        dict(name="store_token", kind="store", rows=1, cols=1024, format="e4m3", nonzero=False),
        # A hidden layer's ReLU outputs at widths that data gave: nothing is a multiple of anything.
        dict(name="store_ragged", kind="store", rows=500, cols=1021, format="e5m2", nonzero=True),
        # A wide layer's weights in 4 bits.
        dict(name="store_weights", kind="store", rows=8192, cols=4096, format="e2m1", nonzero=False),
        # One request at a time through 4-bit weights: the weights' bytes and latency.
        dict(name="linear_token", kind="linear", rows=1, fan_in=4096, fan_out=4096, x="e4m3",
             w="e2m1", act="relu", bias=True),
        # A server's batch through a wide layer, 4 bits on both sides.
        dict(name="linear_batch", kind="linear", rows=64, fan_in=1024, fan_out=4096, x="e2m1",
             w="e2m1", act="none", bias=True),
        # A layer of odd extents, 8 bits on both sides.
        dict(name="linear_ragged", kind="linear", rows=500, fan_in=617, fan_out=1021, x="e4m3",
             w="e4m3", act="tanh", bias=True),
        # A prompt's or a bulk evaluation's rows: the matrix cores' rate.
        dict(name="linear_large", kind="linear", rows=8192, fan_in=4096, fan_out=4096, x="e4m3",
             w="e2m1", act="none", bias=True),
        # The digit classifier's hidden layer, trained from checkpoints in 8 bits.
        dict(name="backward_classifier", kind="backward", rows=1024, fan_in=1024, fan_out=1024,
             format="e4m3", act="relu"),
        # Odd extents, a batch that ends inside every tile, and tanh.
        dict(name="backward_ragged", kind="backward", rows=3001, fan_in=1531, fan_out=2047,
             format="e5m2", act="tanh"),
        # The benchmark's headline layer.
        dict(name="backward_large", kind="backward", rows=4096, fan_in=4096, fan_out=4096,
             format="e4m3", act="relu"),
        # Fine-tuning through frozen 4-bit weights: the gradient that reaches the layer below.
        dict(name="input_grad_ragged", kind="input_grad", rows=500, fan_in=1021, fan_out=1531,
             format="e2m1"),
        # The same through a layer of the headline network's size.
        dict(name="input_grad_large", kind="input_grad", rows=4096, fan_in=4096, fan_out=4096,
             format="e2m1"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _extent(rng, lo, hi):
    """An extent of the range: as drawn (often odd), or rounded to what a person would type."""
    n = _log_int(rng, lo, hi)
    step = rng.choice([1, 1, 4, 16, 64, 128])
    return max(lo, n // step * step)


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        b, f = most.get(c["kind"], (0, 0))
        most[c["kind"]] = (max(b, w["bytes"]), max(f, w["flops"]))
    while True:
        kind = rng.choice(["store", "linear", "linear", "backward", "input_grad"])
        if kind == "store":
            case = dict(kind=kind, rows=_extent(rng, 1, 16384), cols=_extent(rng, 8, 16384),
                        format=rng.choice(["e4m3", "e5m2", "e2m1"]), nonzero=False)
            case["nonzero"] = case["format"] != "e2m1" and rng.random() < 0.5
        elif kind == "linear":
            case = dict(kind=kind, rows=_extent(rng, 1, 8192), fan_in=_extent(rng, 32, 8192),
                        fan_out=_extent(rng, 8, 8192), x=rng.choice(["e4m3", "e4m3", "e2m1", "e5m2"]),
                        w=rng.choice(["e2m1", "e2m1", "e4m3", "e5m2"]),
                        act=rng.choice(["none", "relu", "tanh", "sigmoid"]),
                        bias=rng.random() < 0.8)
        elif kind == "backward":
            case = dict(kind=kind, rows=_extent(rng, 16, 8192), fan_in=_extent(rng, 8, 4096),
                        fan_out=_extent(rng, 8, 4096), format=rng.choice(["e4m3", "e5m2"]),
                        act=rng.choice(["relu", "tanh", "sigmoid"]))
        else:
            case = dict(kind=kind, rows=_extent(rng, 1, 8192), fan_in=_extent(rng, 8, 4096),
                        fan_out=_extent(rng, 8, 4096), format=rng.choice(["e2m1", "e4m3"]))
        w = work(case)
        if w["bytes"] <= most[kind][0] and w["flops"] <= most[kind][1]:
            return case


# ---- the microscaled format, by elementary operations in 32 bits ----
def _groups(cols):
    return -(-cols // 128)


def _power(e):
    """2^e as floats, for integer tensors of exponents of normal numbers."""
    return ((e + 127) << 23).view(torch.float32)


def _blocks(x):
    """The rows of x, zeros to whole groups of 128, as blocks of 32."""
    R, C = x.shape
    if C % 128:
        x = torch.cat([x, x.new_zeros(R, -C % 128)], 1)
    return x.reshape(R, -1, 32)


def _quantise(x, format, nonzero):
    """(the values of x's codes before their scales, [R, 4 G, 32]; the scale bytes, [R, 4 G])."""
    top, bits, least, mantissa = _FORMATS[format]
    v = _blocks(x)
    m = v.abs()
    largest = torch.where(m < math.inf, m, 0.0).amax(2)
    # the smallest power of two under which the block's largest value is within the format
    e = (((largest.view(torch.int32) + (0x7fffff - mantissa)) >> 23) - 127 - top).clamp(min=_LEAST_SCALE)
    m = m * _power(-e)[:, :, None]
    step = ((m.view(torch.int32) >> 23) - 127).clamp(min=least) - bits
    q = torch.round(m * _power(-step)) * _power(step)
    if nonzero:
        q = torch.where((q == 0) & (v != 0), 2.0 ** (least - bits), q)
    return torch.copysign(q, v), (e + 127).to(torch.uint8)


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _codes(q, format):
    """The code bytes of values that the format holds, [R, bytes of a row]."""
    R = q.shape[0]
    q = q.reshape(R, -1)
    if format == "e4m3":
        return q.to(torch.float8_e4m3fn).view(torch.uint8)
    if format == "e5m2":
        return q.to(torch.float8_e5m2).view(torch.uint8)
    place = torch.bucketize(q.abs(), q.new_tensor(_E2M1)) + 8 * torch.signbit(q)
    return (place[:, 0::2] + 16 * place[:, 1::2]).to(torch.uint8)


def _values(codes, scales, cols, format, dtype=torch.float32):
    """The values that codes and scales stand for, [R, cols]."""
    R = codes.shape[0]
    if format == "e2m1":
        table = torch.tensor(_E2M1 + tuple(-t for t in _E2M1), device=codes.device, dtype=dtype)
        v = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], 2)
    else:
        v = codes.view(torch.float8_e4m3fn if format == "e4m3" else torch.float8_e5m2).to(dtype)
    return (v.reshape(R, -1, 32) * _power(scales.int() - 127)[:, :, None].to(dtype)).reshape(R, -1)[:, :cols]


# ---- inputs ----
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)


def _normal(g, shape, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale)


def _encoded(x, format, nonzero=False):
    q, s = _quantise(x, format, nonzero)
    return _codes(q, format), s


def _activate(act, z):
    return {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, 0.0),
            "tanh": lambda: torch.tanh(z), "sigmoid": lambda: 1 / (1 + torch.exp(-z))}[act]()


def _activations(g, rows, cols, act):
    """A hidden layer's outputs: channels of different sizes, some of them far larger."""
    z = _normal(g, (rows, cols)) * torch.exp(_normal(g, (cols,), 0.7))
    return _activate(act, z)


def _weights(g, fan_out, fan_in):
    return _normal(g, (fan_out, fan_in), math.sqrt(2.0 / (fan_in + fan_out)))


def _cotangent(g, rows, cols):
    """Per-sample gradients: their sizes spread over some binades, a tenth of the samples masked."""
    d = _normal(g, (rows, cols), 1.0 / rows) * torch.exp(_normal(g, (rows, 1)))
    return d * (torch.rand((rows, 1), generator=g, device="cuda") >= 0.1)


def _inputs(case, seed):
    g = _generator(seed)
    R = case["rows"]
    if case["kind"] == "store":
        if case["nonzero"]:
            return dict(x=_activations(g, R, case["cols"], "relu"))
        return dict(x=_activations(g, R, case["cols"], "none"))
    I, O = case["fan_in"], case["fan_out"]
    if case["kind"] == "linear":
        return dict(x=_activations(g, R, I, "none"), w=_encoded(_weights(g, O, I), case["w"]),
                    b=_normal(g, (O,), 0.05) if case["bias"] else None)
    if case["kind"] == "backward":
        act, f = case["act"], case["format"]
        return dict(dy=_cotangent(g, R, O), y=_encoded(_activations(g, R, O, act), f, True),
                    x=_encoded(_activations(g, R, I, act), f, True))
    return dict(dz=_cotangent(g, R, O), w=_encoded(_weights(g, O, I), case["format"]))


# ---- the plain forms ----
def _plain_store(case, x):
    q, s = _quantise(x, case["format"], case["nonzero"])
    v = q * _power(s.int() - 127)[:, :, None]
    return dict(values=v.reshape(x.shape[0], -1)[:, :case["cols"]], scales=s)


def _plain_linear(case, x, w, b):
    q, s = _quantise(x, case["x"], False)
    xv = (q * _power(s.int() - 127)[:, :, None]).reshape(x.shape[0], -1)[:, :case["fan_in"]]
    z = xv @ _values(*w, case["fan_in"], case["w"]).t()
    return _activate(case["act"], z if b is None else z + b)


def _slope(act, y):
    return {"relu": lambda: (y > 0).to(y.dtype), "tanh": lambda: 1 - y * y,
            "sigmoid": lambda: y * (1 - y)}[act]()


def _plain_backward(case, dy, y, x):
    dz = dy * _slope(case["act"], _values(*y, case["fan_out"], case["format"]))
    return dict(dz=dz, db=dz.sum(0), dw=dz.t() @ _values(*x, case["fan_in"], case["format"]))


def _plain_input_grad(case, dz, w):
    return dz @ _values(*w, case["fan_in"], case["format"])


_PLAIN = dict(store=_plain_store, linear=_plain_linear, backward=_plain_backward,
              input_grad=_plain_input_grad)


# ---- the framework's operators: a program over the same tensors ----
_backend = None


def _context():
    global _backend
    if _backend is None:
        from synaptik_amd.backend import HipBackendIntegration
        _backend = HipBackendIntegration.open(0)
    return _backend.context


def _empty(*shape, dtype=torch.float32):
    return torch.empty(shape, device="cuda", dtype=dtype)


def _program(case, t):
    """(the program bound to the tensors `t` and to its outputs, the outputs that a pass returns)."""
    from synaptik_amd.native import HipBuffer, HipProgram
    from synaptik_amd.program import ProgramBuilder
    pb, kind, R = ProgramBuilder(), case["kind"], case["rows"]
    ins, outs = [], []

    def take(tensor):
        if tensor is None:
            return None
        if isinstance(tensor, tuple):
            return tuple(take(p) for p in tensor)
        ins.append(tensor)
        return pb.input(tensor.numel(), "u8" if tensor.dtype == torch.uint8 else "f32")

    def give(*shape, dtype=torch.float32):
        outs.append(_empty(*shape, dtype=dtype))
        return pb.output(outs[-1].numel(), "u8" if dtype == torch.uint8 else "f32")

    if kind == "store":
        C, f = case["cols"], case["format"]
        x, values, scales = take(t["x"]), give(R, C), give(R, 4 * _groups(C), dtype=torch.uint8)
        codes = give(R, _groups(C) * (64 if f == "e2m1" else 128), dtype=torch.uint8)
        pb.mx_encode(x, (codes, scales), R, C, format=f, keep_nonzero=case["nonzero"])
        pb.mx_decode((codes, scales), values, R, C, format=f)
        result = dict(values=outs[0], scales=outs[1])
    elif kind == "linear":
        I, O = case["fan_in"], case["fan_out"]
        pb.mx_linear(take(t["x"]), take(t["w"]), give(R, O), R, O, I, x_format=case["x"],
                     w_format=case["w"], bias=take(t["b"]), act=case["act"])
        result = outs[0]
    elif kind == "backward":
        I, O, f = case["fan_in"], case["fan_out"], case["format"]
        dz, db, dw = give(R, O), give(O), give(O, I)
        pb.mx_act_grad(take(t["dy"]), take(t["y"]), dz, R, O, act=case["act"], format=f, colsum=db)
        pb.mx_gemm(dz, take(t["x"]), dw, O, I, R, format=f, trans_a=True)
        result = dict(dz=outs[0], db=outs[1], dw=outs[2])
    else:
        I, O = case["fan_in"], case["fan_out"]
        pb.mx_gemm(take(t["dz"]), take(t["w"]), give(R, I), R, I, O, format=case["format"])
        result = outs[0]
    program = HipProgram(_context(), pb.image())
    wrap = lambda v: HipBuffer(_context(), v.numel() * v.element_size(), v.data_ptr())  # noqa: E731
    return program, program.bind([wrap(v) for v in ins], [wrap(v) for v in outs]), result


def prepare(case, seed):
    state = dict(case=case, inputs=_inputs(case, seed))
    if own:
        state["program"], state["bound"], state["result"] = _program(case, state["inputs"])
    torch.cuda.synchronize()  # the tensors are written before another stream reads them
    return state


def run(state):
    if own:
        state["program"].run_bound(state["bound"])
        return state["result"]
    return _PLAIN[state["case"]["kind"]](state["case"], **state["inputs"])


# ---- the definition in 64 bits ----
def _power64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _stored64(x, format, nonzero):
    """What the codes of x stand for, and their scale bytes, from the definition: scales by
    logarithms, values by the nearest multiple (ties to even) of the format's step."""
    top, bits, least, mantissa = _FORMATS[format]
    limit = (1 + mantissa / 2.0 ** 23) * 2.0 ** top
    v = _blocks(x.double())
    largest = v.abs().amax(2)
    _, e = torch.frexp(largest / limit)  # largest / limit = m 2^e, m in [1/2, 1)
    e = torch.where(largest / limit == _power64(e - 1), e - 1, e)
    e = torch.where(largest > 0, e, torch.full_like(e, _LEAST_SCALE)).clamp(min=_LEAST_SCALE)
    unit = _power64(e)[:, :, None]
    m = v.abs() / unit
    _, k = torch.frexp(m)  # m in [2^(k-1), 2^k)
    step = _power64(torch.clamp(k - 1, min=least) - bits)
    q = torch.round(m / step) * step
    if nonzero:
        q = torch.where((q == 0) & (m > 0), torch.full_like(q, 2.0 ** (least - bits)), q)
    return (torch.sign(v) * q * unit).reshape(x.shape[0], -1)[:, :x.shape[1]], (e + 127).to(torch.uint8)


def exact(case, seed):
    t = _inputs(case, seed)
    kind = case["kind"]
    values = lambda p, cols, f: _values(*p, cols, f, torch.float64)  # noqa: E731
    if kind == "store":
        v, s = _stored64(t["x"], case["format"], case["nonzero"])
        return dict(values=v, scales=s)
    I, O = case["fan_in"], case["fan_out"]
    if kind == "linear":
        z = _stored64(t["x"], case["x"], False)[0] @ values(t["w"], I, case["w"]).t()
        return _activate(case["act"], z if t["b"] is None else z + t["b"].double())
    if kind == "backward":
        f = case["format"]
        dz = t["dy"].double() * _slope(case["act"], values(t["y"], O, f))
        return dict(dz=dz, db=dz.sum(0), dw=dz.t().contiguous() @ values(t["x"], I, f))
    return t["dz"].double() @ values(t["w"], I, case["format"])


def _stored_bytes(rows, cols, format):
    return rows * _groups(cols) * ((64 if format == "e2m1" else 128) + 4.0)


def work(case):
    """Bytes: inputs read once, outputs (codes and scales that are kept among them) written once.
    Operations: two for each multiply-add of the matrix products, a few for each element else."""
    R, kind = case["rows"], case["kind"]
    if kind == "store":
        n = float(R) * case["cols"]
        return {"bytes": 8.0 * n + _stored_bytes(R, case["cols"], case["format"]), "flops": 4.0 * n}
    I, O = case["fan_in"], case["fan_out"]
    product = 2.0 * R * I * O
    if kind == "linear":
        return {"bytes": 4.0 * (R * I + R * O + O * case["bias"]) + _stored_bytes(O, I, case["w"]),
                "flops": product}
    if kind == "backward":
        f = case["format"]
        return {"bytes": 4.0 * (2 * R * O + O + O * I) + _stored_bytes(R, O, f) + _stored_bytes(R, I, f),
                "flops": product + 3.0 * R * O}
    return {"bytes": 4.0 * (R * O + R * I) + _stored_bytes(O, I, case["format"]), "flops": product}
