"""Operators of token models: what is measured of them, with plain forms beside the framework's own.

Kinds of case (the "kind" entry):
  embed       rows of a table by token, scaled; the padding token's row is zero (ProgramBuilder.embed);
  embed_grad  the table's gradient: the sum of each token's rows (ProgramBuilder.embed_grad);
  norm        layer norm with weight and bias (ProgramBuilder.layer_norm);
  norm_grad   its backward pass: the input's, the weight's and the bias' gradients
              (ProgramBuilder.layer_norm_grad);
  scan        the gated linear recurrence h_t = f_t h_{t-1} + (1 - f_t) u_t, f = 1 / (1 + exp(-z)), of
              sequences [B, T, D], from a state and to a state (ProgramBuilder.gated_scan);
  scan_grad   its backward pass: the gates', the inputs' and the first state's gradients
              (ProgramBuilder.gated_scan_grad);
  distill     the divergence of a model's distribution from a teacher's, of which the largest logits are
              known, and its gradient (ProgramBuilder.distill).

Inputs, weights and outputs are in GPU memory when a pass begins; a pass is the synchronous call
that a program makes.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
_INT = {"i32": torch.int32, "i64": torch.int64}


def listed():
    return [
        # One further token for 64 requests, some of which have ended: latency alone.
        dict(name="embed_tokens", kind="embed", rows=64, vocab=32003, width=1024, index="i64", pad=True),
        # A small corpus' vocabulary and a batch padded to its longest text: nothing is a multiple of anything.
        dict(name="embed_grad_ragged", kind="embed_grad", rows=5001, vocab=10007, width=617, index="i32", pad=True),
        # A training batch of 16 texts of 2048 tokens over a large vocabulary.
        dict(name="embed_grad_large", kind="embed_grad", rows=32768, vocab=65536, width=1024, index="i64", pad=False),
        # One position's hidden state while text is generated.
        dict(name="norm_token", kind="norm", rows=1, width=4096),
        # A width and a number of rows that data gave.
        dict(name="norm_grad_ragged", kind="norm_grad", rows=3001, width=1531),
        # A training batch between layers of the headline network's width.
        dict(name="norm_grad_large", kind="norm_grad", rows=16384, width=4096),
        # One further token for 64 requests: each one's state, moved on.
        dict(name="scan_token", kind="scan", batch=64, time=1, width=1024, lengths=False),
        # One very long text: all the work lies along time.
        dict(name="scan_long", kind="scan", batch=1, time=65536, width=512, lengths=False),
        # Texts of different lengths, padded to the longest.
        dict(name="scan_grad_ragged", kind="scan_grad", batch=7, time=1501, width=617, lengths=True),
        # A training batch.
        dict(name="scan_grad_large", kind="scan_grad", batch=16, time=4096, width=1024, lengths=False),
        # A classifier of odd extents against a handful of the teacher's logits.
        dict(name="distill_ragged", kind="distill", rows=500, classes=10007, top=13, index="i32",
             temperature=2.0, grad=True),
        # A training batch of a language model.
        dict(name="distill_large", kind="distill", rows=4096, classes=32003, top=64, index="i64",
             temperature=1.0, grad=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _extent(rng, lo, hi):
    """An extent of the range: as drawn (often odd), or rounded to what a person would type."""
    n = _log_int(rng, lo, hi)
    step = rng.choice([1, 1, 4, 16, 64, 128])
    return max(lo, n // step * step)


def draw(rng):
    most = max(work(c)["bytes"] for c in listed())
    while True:
        kind = rng.choice(["embed", "embed_grad", "norm", "norm_grad", "scan", "scan_grad", "distill"])
        if kind.startswith("embed"):
            case = dict(kind=kind, rows=_extent(rng, 1, 65536), vocab=_extent(rng, 16, 131072),
                        width=_extent(rng, 8, 8192), index=rng.choice(["i32", "i64"]), pad=rng.random() < 0.5)
        elif kind.startswith("norm"):
            case = dict(kind=kind, rows=_extent(rng, 1, 65536), width=_extent(rng, 8, 16384))
        elif kind.startswith("scan"):
            case = dict(kind=kind, batch=_extent(rng, 1, 128), time=_extent(rng, 1, 65536),
                        width=_extent(rng, 8, 4096), lengths=rng.random() < 0.4)
        else:
            classes = _extent(rng, 16, 131072)
            case = dict(kind=kind, rows=_extent(rng, 1, 16384), classes=classes,
                        top=min(classes, _extent(rng, 1, 256)), index=rng.choice(["i32", "i64"]),
                        temperature=rng.choice([1.0, 1.0, 2.0, 4.0]), grad=rng.random() < 0.75)
        if work(case)["bytes"] <= most:
            return case


# ---- inputs ----
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)


def _normal(g, shape, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale)


def _uniform(g, shape):
    return torch.rand(shape, generator=g, device="cuda", dtype=torch.float64)


def _tokens(g, case):
    """Tokens of a text: the k-th most frequent about 1 / k as often as the first; its number says
    nothing of that. A padded batch has a tenth of padding tokens (number 0), here at its end."""
    N, V = case["rows"], case["vocab"]
    rank = torch.exp(_uniform(g, (N,)) * math.log(V)).long().clamp(1, V) - 1
    t = torch.randperm(V, generator=g, device="cuda")[rank]
    if case["pad"]:
        t[N - N // 10:] = 0
    return t.to(_INT[case["index"]])


def _hidden(g, rows, width):
    """Hidden states: rows of different sizes, channels off zero, some of them far larger."""
    x = _normal(g, (rows, width)) * torch.exp(_normal(g, (width,), 0.7))
    return x.mul_(torch.exp(_normal(g, (rows, 1), 0.3))).add_(_normal(g, (width,), 0.5))


def _cotangent(g, rows, width):
    """Per-position gradients: their sizes spread over some binades."""
    return _normal(g, (rows, width), 1.0 / rows) * torch.exp(_normal(g, (rows, 1)))


def _lengths(g, case):
    """Lengths from half of the longest on; the longest is among them."""
    n = (case["time"] * (0.5 + 0.5 * _uniform(g, (case["batch"],)))).long().clamp(min=1)
    n[0] = case["time"]
    return n.to(torch.int32)


def _inputs(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind == "embed":
        V, D = case["vocab"], case["width"]
        return dict(table=_normal(g, (V, D), 0.02), tokens=_tokens(g, case))
    if kind == "embed_grad":
        return dict(dy=_cotangent(g, case["rows"], case["width"]), tokens=_tokens(g, case))
    if kind.startswith("norm"):
        R, C = case["rows"], case["width"]
        t = dict(x=_hidden(g, R, C), gamma=1 + _normal(g, (C,), 0.2))
        if kind == "norm":
            return dict(t, beta=_normal(g, (C,), 0.1))
        return dict(t, dy=_cotangent(g, R, C))
    if kind.startswith("scan"):
        B, T, D = case["batch"], case["time"], case["width"]
        # gates whose memories last from a step or two to some hundreds
        t = dict(z=_normal(g, (B, T, D)).add_(1 + 4 * _uniform(g, (D,)).float()), u=_normal(g, (B, T, D)),
                 h0=_normal(g, (B, D), 0.5), lengths=_lengths(g, case) if case["lengths"] else None)
        if kind == "scan_grad":
            t["h"] = _plain_scan(case, **t)["h"]
            t["dh"] = _normal(g, (B, T, D), 1.0 / (B * T))
            t["dlast"] = _normal(g, (B, D), 1.0 / (B * T))
        return t
    R, C, K = case["rows"], case["classes"], case["top"]
    # distinct classes for each row, the teacher's logits from the largest on
    apart = (_uniform(g, (R, K)) * (C // K)).long() + 1
    index = ((_uniform(g, (R, 1)) * C).long() + apart.clamp(max=C // K).cumsum(1)) % C
    teacher = (_normal(g, (R, K)) - 1.5 * torch.arange(1, K + 1, device="cuda").log()).sort(1, descending=True)[0] + 8
    logits = _normal(g, (R, C), 2.0).scatter_add_(1, index, 0.6 * teacher)
    # a tenth of the rows is masked, a third keeps fewer entries
    kept = torch.where(_uniform(g, (R,)) < 1 / 3, (_uniform(g, (R,)) * K).long() + 1, K)
    kept[1:] *= (_uniform(g, (R - 1,)) >= 0.1).long()
    index = torch.where(torch.arange(K, device="cuda") < kept[:, None], index, -1)
    return dict(logits=logits, index=index.to(_INT[case["index"]]), teacher=teacher)


# ---- the plain forms ----
def _scale(case):
    return math.sqrt(case["width"])


def _plain_embed(case, table, tokens):
    y = table[tokens] * _scale(case)
    return torch.where(tokens[:, None] == 0, 0.0, y) if case["pad"] else y


def _plain_embed_grad(case, dy, tokens):
    if case["pad"]:
        dy = torch.where(tokens[:, None] == 0, 0.0, dy)
    dw = torch.zeros((case["vocab"], case["width"]), device="cuda")
    return dw.index_add_(0, tokens, dy).mul_(_scale(case))


def _normalised(x):
    d = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    return d * rstd, rstd


def _plain_norm(case, x, gamma, beta):
    return _normalised(x)[0] * gamma + beta


def _plain_norm_grad(case, x, gamma, dy):
    xhat, rstd = _normalised(x)
    w, g = dy * xhat, dy * gamma
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return dict(dx=dx, dgamma=w.sum(0), dbeta=dy.sum(0))


def _gates(z):
    e = torch.exp(-z.abs())
    a, b = 1 / (1 + e), e / (1 + e)
    return torch.where(z >= 0, a, b), torch.where(z >= 0, b, a)


def _prefix(f, b):
    """h_t = f_t h_{t-1} + b_t along dimension 1, by doubling."""
    n, step = f.shape[1], 1
    while step < n:
        b = torch.cat([b[:, :step], torch.addcmul(b[:, step:], f[:, step:], b[:, :-step])], 1)
        f = torch.cat([f[:, :step], f[:, step:] * f[:, :-step]], 1)
        step *= 2
    return b


def _within(case, lengths):
    return (torch.arange(case["time"], device="cuda")[None] < lengths[:, None])[:, :, None]


def _plain_scan(case, z, u, h0, lengths):
    f, k = _gates(z)
    b = k * u
    b[:, 0] += f[:, 0] * h0
    h = _prefix(f, b)
    if lengths is None:
        return dict(h=h, last=h[:, -1].contiguous())
    last = h[torch.arange(case["batch"], device="cuda"), lengths.long() - 1]
    return dict(h=torch.where(_within(case, lengths), h, 0.0), last=last)


def _plain_scan_grad(case, z, u, h0, lengths, h, dh, dlast):
    f, k = _gates(z)
    if lengths is None:
        b = dh.clone()
        b[:, -1] += dlast
        carry = f
    else:
        inside = _within(case, lengths)
        b = torch.where(inside, dh, 0.0)
        b[torch.arange(case["batch"], device="cuda"), lengths.long() - 1] += dlast
        carry = torch.where(inside, f, 0.0)
    carry = torch.cat([carry[:, 1:], torch.zeros_like(carry[:, :1])], 1)
    g = _prefix(carry.flip(1), b.flip(1)).flip(1)
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    du, dz = k * g, g * (before - u) * (f * k)
    if lengths is not None:
        du, dz = torch.where(inside, du, 0.0), torch.where(inside, dz, 0.0)
    return dict(dz=dz, du=du, dh0=f[:, 0] * g[:, 0])


def _plain_distill(case, logits, index, teacher):
    T, R = case["temperature"], case["rows"]
    there = index >= 0
    rows = there.any(1)
    n = rows.sum()
    safe = torch.where(there, index, 0).long()
    t = torch.where(there, teacher, -math.inf)
    t = torch.where(rows[:, None], (t - t.amax(1, keepdim=True)) / T, -math.inf)
    e = torch.exp(t)
    sum_t = torch.where(rows, e.sum(1), 1.0)
    p = e / sum_t[:, None]
    zs = (logits - logits.amax(1, keepdim=True)) / T
    ez = torch.exp(zs)
    sum_z = ez.sum(1)
    apart = torch.where(there, t - zs.gather(1, safe), 0.0)
    each = (p * apart).sum(1) - torch.log(sum_t) + torch.log(sum_z)
    loss = T * T * torch.where(rows, each, 0.0).double().sum() / n
    loss = loss.float().reshape(1)
    if not case["grad"]:
        return dict(loss=loss)
    q = ez.div_(sum_z[:, None]).scatter_add_(1, safe, -p)
    return dict(loss=loss, grad=torch.where(rows[:, None], q, 0.0) * (T / n))


_PLAIN = dict(embed=_plain_embed, embed_grad=_plain_embed_grad, norm=_plain_norm, norm_grad=_plain_norm_grad,
              scan=_plain_scan, scan_grad=_plain_scan_grad, distill=_plain_distill)


# ---- the framework's operators: a program over the same tensors ----
_backend = None


def _context():
    global _backend
    if _backend is None:
        from synaptik_amd.backend import HipBackendIntegration
        _backend = HipBackendIntegration.open(0)
    return _backend.context


_SLOT = {torch.float32: "f32", torch.int32: "i32", torch.int64: "i64"}


def _program(case, t):
    """(the program bound to the tensors `t` and to its outputs, the outputs that a pass returns)."""
    from synaptik_amd.native import HipBuffer, HipProgram
    from synaptik_amd.program import ProgramBuilder
    pb, kind = ProgramBuilder(), case["kind"]
    ins, outs = [], []

    def take(name):
        if t[name] is None:
            return None
        ins.append(t[name])
        return pb.input(t[name].numel(), _SLOT[t[name].dtype])

    def give(*shape):
        outs.append(torch.empty(shape, device="cuda"))
        return pb.output(outs[-1].numel())

    if kind.startswith("embed"):
        N, V, D = case["rows"], case["vocab"], case["width"]
        how = dict(scale=_scale(case), pad=0 if case["pad"] else None)
        if kind == "embed":
            pb.embed(take("table"), take("tokens"), give(N, D), N, V, D, **how)
        else:
            pb.embed_grad(take("dy"), take("tokens"), give(V, D), N, V, D, **how)
        result = outs[0]
    elif kind.startswith("norm"):
        R, C = case["rows"], case["width"]
        if kind == "norm":
            pb.layer_norm(take("x"), give(R, C), R, C, gamma=take("gamma"), beta=take("beta"), eps=EPS)
            result = outs[0]
        else:
            pb.layer_norm_grad(take("dy"), take("x"), give(R, C), R, C, gamma=take("gamma"), dgamma=give(C),
                               dbeta=give(C), eps=EPS)
            result = dict(zip(("dx", "dgamma", "dbeta"), outs))
    elif kind.startswith("scan"):
        B, T, D = case["batch"], case["time"], case["width"]
        if kind == "scan":
            pb.gated_scan(take("z"), take("u"), give(B, T, D), B, T, D, h0=take("h0"), last=give(B, D),
                          lengths=take("lengths"))
            result = dict(zip(("h", "last"), outs))
        else:
            pb.gated_scan_grad(take("dh"), take("z"), take("u"), take("h"), give(B, T, D), give(B, T, D), B, T, D,
                               h0=take("h0"), dlast=take("dlast"), dh0=give(B, D), lengths=take("lengths"))
            result = dict(zip(("dz", "du", "dh0"), outs))
    else:
        R, C, K = case["rows"], case["classes"], case["top"]
        pb.distill(take("logits"), take("index"), take("teacher"), give(1), R, C, K,
                   grad=give(R, C) if case["grad"] else None, temperature=case["temperature"])
        result = dict(zip(("loss", "grad"), outs))
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
def _exact_embed_grad(case, dy, tokens):
    """Each token's rows as a difference of running sums over the rows in the tokens' order."""
    t = tokens.long()
    order = torch.argsort(t, stable=True)
    running = torch.cat([dy.new_zeros((1, case["width"]), dtype=torch.float64), dy.double()[order].cumsum(0)])
    ends = torch.bincount(t, minlength=case["vocab"]).cumsum(0)
    dw = running[ends]
    dw[1:] -= running[ends[:-1]]
    if case["pad"]:
        dw[0] = 0
    return dw * _scale(case)


def _exact_norm(x, gamma, beta):
    x = x.double()
    var, mean = torch.var_mean(x, 1, keepdim=True, correction=0)
    return (x - mean) / torch.sqrt(var + EPS) * gamma.double() + beta


def _exact_norm_grad(x, gamma, dy):
    x, gamma = x.double().requires_grad_(), gamma.double().requires_grad_()
    beta = torch.zeros_like(gamma, requires_grad=True)
    y = _exact_norm(x, gamma, beta)
    return dict(zip(("dx", "dgamma", "dbeta"), torch.autograd.grad(y, (x, gamma, beta), dy.double())))


def _steps(case, lengths):
    """1 where a sequence has a position, 0 behind its end, [T, B, 1] in 64 bits."""
    if lengths is None:
        return torch.ones((case["time"], case["batch"], 1), device="cuda", dtype=torch.float64)
    return _within(case, lengths).double().transpose(0, 1).contiguous()


def _exact_scan(case, z, u, h0, lengths):
    """Position by position."""
    inside = _steps(case, lengths)
    f, u = torch.sigmoid(z.double().transpose(0, 1)), u.double().transpose(0, 1)
    state, out = h0.double(), torch.empty_like(f)
    for t in range(case["time"]):
        torch.lerp(u[t], state, f[t], out=out[t])
        state = out[t] if lengths is None else torch.where(inside[t] > 0, out[t], state)
    return dict(h=(out * inside).transpose(0, 1), last=state)


def _exact_scan_grad(case, z, u, h0, lengths, h, dh, dlast):
    inside = _steps(case, lengths)
    f, u = torch.sigmoid(z.double().transpose(0, 1)), u.double().transpose(0, 1)
    before = torch.cat([h0[None], h.transpose(0, 1)[:-1]]).double()
    at_f, at_u = (before - u) * torch.sigmoid(-z.double().transpose(0, 1)) * f, torch.sigmoid(-z.double().transpose(0, 1))
    dh = dh.double().transpose(0, 1) * inside
    carry, g = dlast.double(), torch.empty_like(f)
    for t in reversed(range(case["time"])):
        torch.add(dh[t], carry, out=g[t])
        carry = g[t] * f[t] if lengths is None else torch.where(inside[t] > 0, g[t] * f[t], carry)
    g *= inside
    return dict(dz=(g * at_f).transpose(0, 1), du=(g * at_u).transpose(0, 1), dh0=carry)


def _exact_distill(case, logits, index, teacher):
    T = case["temperature"]
    keep = (index >= 0).any(1)
    z, index, t = logits[keep].double(), index[keep].long(), teacher[keep].double() / T
    log_p = torch.log_softmax(t.masked_fill(index < 0, -math.inf), 1)
    log_q = torch.log_softmax(z / T, 1)
    p = log_p.exp()
    safe, n = index.clamp(min=0), z.shape[0]
    loss = (p * (log_p.masked_fill(index < 0, 0.0) - log_q.gather(1, safe))).sum() * T * T / n
    if not case["grad"]:
        return dict(loss=loss.reshape(1))
    grad = torch.zeros(logits.shape, device="cuda", dtype=torch.float64)
    grad[keep] = (log_q.exp_().scatter_add_(1, safe, -p)) * (T / n)
    return dict(loss=loss.reshape(1), grad=grad)


def exact(case, seed):
    t, kind = _inputs(case, seed), case["kind"]
    if kind == "embed":
        y = t["table"].double()[t["tokens"].long()] * _scale(case)
        if case["pad"]:
            y[t["tokens"] == 0] = 0
        return y
    if kind == "embed_grad":
        return _exact_embed_grad(case, **t)
    if kind == "norm":
        return _exact_norm(**t)
    if kind == "norm_grad":
        return _exact_norm_grad(**t)
    return dict(scan=_exact_scan, scan_grad=_exact_scan_grad, distill=_exact_distill)[kind](case, **t)


def work(case):
    """Bytes: inputs read once, outputs written once; of a table the rows that a batch can touch, of a
    padded batch the positions that there are. Operations: a few for each element."""
    kind = case["kind"]
    if kind.startswith("embed"):
        N, V, D = case["rows"], case["vocab"], case["width"]
        tokens = N * (4.0 if case["index"] == "i32" else 8.0)
        if kind == "embed":
            return {"bytes": 4.0 * D * (min(N, V) + N) + tokens, "flops": 1.0 * N * D}
        return {"bytes": 4.0 * D * (N + V) + tokens, "flops": 2.0 * N * D}
    if kind.startswith("norm"):
        n, C = float(case["rows"]) * case["width"], case["width"]
        return {"bytes": 8.0 * n + 8.0 * C, "flops": 8.0 * n} if kind == "norm" else {"bytes": 12.0 * n + 12.0 * C, "flops": 16.0 * n}
    if kind.startswith("scan"):
        n, state = float(case["batch"]) * case["time"] * case["width"], 4.0 * case["batch"] * case["width"]
        there = 0.75 if case["lengths"] else 1.0
        if kind == "scan":
            return {"bytes": (8.0 * there + 4.0) * n + 2 * state, "flops": 8.0 * n}
        return {"bytes": (16.0 * there + 8.0) * n + 3 * state, "flops": 16.0 * n}
    n = float(case["rows"]) * case["classes"]
    entries = case["rows"] * case["top"] * (8.0 if case["index"] == "i32" else 12.0)
    return {"bytes": (0.9 + case["grad"]) * 4.0 * n + entries, "flops": 6.0 * n}
