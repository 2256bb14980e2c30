"""64-bit forms of the steps for models of tokens, with bounds on what binary32 kernels may be off by.

u = 2^-24 is half a unit in the last place of binary32 relative to the value: what one rounding is off
by at most. Bounds are first order in u; FIRST allows for the rest, and TINY for results below the
normal range."""
import numpy as np

U = 2.0 ** -24
FIRST = 1.001
TINY = 2.0 ** -149


def within(got, want, bound):
    """Equal where the wanted value is not finite, within the bound elsewhere."""
    got, want = np.asarray(got, np.float64).reshape(np.shape(want)), np.asarray(want, np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    rest = ~fine & ~np.isnan(want)
    assert np.array_equal(got[rest], want[rest])
    off = np.abs(got - np.where(fine, want, 0.0))[fine]
    most = (np.broadcast_to(bound, want.shape)[fine]) * FIRST + TINY
    worst = np.argmax(off - most) if off.size else 0
    assert (off <= most).all(), (off[worst], most[worst], want[fine][worst])


# ---- embeddings ----
def embed(W, tokens, scale, pad=None):
    """The product of two binary32 values, rounded once: exact to compare with."""
    y = W[np.clip(tokens, 0, W.shape[0] - 1)] * np.float32(scale)
    y[(tokens < 0) | (tokens >= W.shape[0])] = 0
    if pad is not None:
        y[tokens == pad] = 0
    return y


def embed_grad(dY, tokens, V, scale, pad=None):
    """(dW, a bound): the sums are binary64 (a relative 2^-53 an addition) and rounded once."""
    keep = (tokens >= 0) & (tokens < V)
    if pad is not None:
        keep &= tokens != pad
    dW, mass = np.zeros((V, dY.shape[1])), np.zeros((V, dY.shape[1]))
    scale = float(np.float32(scale))
    np.add.at(dW, tokens[keep], dY[keep].astype(np.float64))
    np.add.at(mass, tokens[keep], np.abs(dY[keep]).astype(np.float64))
    return dW * scale, U * np.abs(dW * scale) + (len(tokens) + 2) * 2.0 ** -52 * mass * abs(scale)


# ---- layer norm ----
def normalised(x, eps):
    x = x.astype(np.float64)
    mean = x.mean(-1, keepdims=True)
    d = x - mean
    rstd = 1.0 / np.sqrt((d * d).mean(-1, keepdims=True) + float(np.float32(eps)))
    return d * rstd, rstd


def layer_norm(x, gamma, beta, eps):
    """(y, a bound): the normalised value is rounded to binary32, then one fused multiply-add; what the
    binary64 statistics are off by shows in values far from the mean alone."""
    xh, rstd = normalised(x, eps)
    g = np.ones(x.shape[1]) if gamma is None else gamma.astype(np.float64)
    b = np.zeros(x.shape[1]) if beta is None else beta.astype(np.float64)
    y = xh * g + b
    with np.errstate(invalid="ignore"):
        inner = (x.shape[1] + 8) * 2.0 ** -52 * (np.abs(x.astype(np.float64)).max(-1, keepdims=True) * rstd + np.abs(xh))
        return y, U * (np.abs(xh * g) + np.abs(y)) + inner * np.abs(g)


def layer_norm_grad(dy, x, gamma, eps):
    """((dx, dgamma, dbeta), their bounds): binary64 throughout, rounded once. n binary64 additions are
    off by n 2^-53 of the terms' sizes."""
    xh, rstd = normalised(x, eps)
    dy, C = dy.astype(np.float64), x.shape[1]
    g = dy if gamma is None else dy * gamma.astype(np.float64)
    mean_g, mean_gx = g.mean(-1, keepdims=True), (g * xh).mean(-1, keepdims=True)
    dx = rstd * (g - mean_g - xh * mean_gx)
    # the mean's own error, which moves every xh of the row alike, and the squares' sum's
    lost = (C + 16) * 2.0 ** -51 * (1 + np.abs(x.astype(np.float64)).max(-1, keepdims=True) * rstd)
    size = np.abs(g) + np.abs(g).mean(-1, keepdims=True) + np.abs(xh) * np.abs(g * xh).mean(-1, keepdims=True)
    deep = lost * rstd * (size + (1 + np.abs(xh)) * np.abs(g).mean(-1, keepdims=True))
    dgamma, dbeta = (dy * xh).sum(0), dy.sum(0)
    far = (x.shape[0] + 8) * 2.0 ** -52
    bounds = (U * np.abs(dx) + deep, U * np.abs(dgamma) + far * np.abs(dy * xh).sum(0) + (lost * (1 + np.abs(xh)) * np.abs(dy)).sum(0),
              U * np.abs(dbeta) + far * np.abs(dy).sum(0))
    return (dx, dgamma, dbeta), bounds


# ---- gated recurrence ----
def gates(z):
    z = z.astype(np.float64)
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-z)), 1.0 / (1.0 + np.exp(z))


def _inside(B, T, lengths):
    n = np.full(B, T) if lengths is None else np.asarray(lengths)
    return np.arange(T)[None, :, None] < n[:, None, None]


def gated_scan(z, u, h0=None, lengths=None):
    """(h, the last states, bounds of both).

    A state is a sum of terms (product of the gates since) k u. A term takes three roundings in its own
    step (k, k u, the sum's), and in every later one at most three: the gate's, the product's with
    it (as part of a run's product, or in the sum) and the sum's. So its error is at most
    (3 (t - s) + 3) u times its size; `mass` sums the sizes and `age` the sizes times t - s."""
    B, T, D = z.shape
    inside = _inside(B, T, lengths)
    f, k = gates(z)
    state = np.zeros((B, D)) if h0 is None else h0.astype(np.float64)
    mass, age = np.abs(state), np.zeros((B, D))
    h, off = np.zeros((B, T, D)), np.zeros((B, T, D))
    for t in range(T):
        live = inside[:, t]
        with np.errstate(invalid="ignore"):
            state = np.where(live, f[:, t] * state + k[:, t] * u[:, t], state)
            age = np.where(live, f[:, t] * (age + mass), age)
            mass = np.where(live, f[:, t] * mass + np.abs(k[:, t] * u[:, t]), mass)
        h[:, t], off[:, t] = np.where(live, state, 0.0), np.where(live, 3 * U * (age + mass), 0.0)
    return h, state, off, 3 * U * (age + mass)


def gated_scan_grad(dh, z, u, h, h0=None, dlast=None, lengths=None):
    """((dz, du, dh0), their bounds), h being the binary32 states that the kernel is given. A term of G
    enters exactly and takes the same three roundings a step; du adds two (k, the product), dz six (f,
    k, their product, h - u, the product with it, the one with G), dh0 two more."""
    B, T, D = z.shape
    inside = _inside(B, T, lengths)
    f, k = gates(z)
    h, u = h.astype(np.float64), u.astype(np.float64)
    before = np.concatenate([(np.zeros((B, D)) if h0 is None else h0.astype(np.float64))[:, None], h[:, :-1]], 1)
    carry = np.zeros((B, D)) if dlast is None else dlast.astype(np.float64)
    mass, age = np.abs(carry), np.zeros((B, D))
    dz, du, bz, bu = (np.zeros((B, T, D)) for _ in range(4))
    for t in reversed(range(T)):
        live = inside[:, t]
        g = np.where(live, dh[:, t], 0.0) + carry
        m = np.where(live, np.abs(dh[:, t]), 0.0) + mass
        off = 3 * U * (age + m)
        w = (before[:, t] - u[:, t]) * f[:, t] * k[:, t]
        dz[:, t], du[:, t] = np.where(live, g * w, 0.0), np.where(live, g * k[:, t], 0.0)
        bz[:, t] = np.where(live, np.abs(w) * (off + 6 * U * np.abs(g)), 0.0)
        bu[:, t] = np.where(live, k[:, t] * (off + 2 * U * np.abs(g)), 0.0)
        age = np.where(live, f[:, t] * (age + m), age)
        mass = np.where(live, f[:, t] * m, mass)
        carry = np.where(live, f[:, t] * g, carry)
    return (dz, du, carry), (bz, bu, 3 * U * (age + mass) + 2 * U * np.abs(carry))


# ---- distillation ----
def distill(z, index, t, T=1.0, g=1.0):
    """(loss, gradient, their bounds).

    A class' weight e = exp((z - m) / T) is off by 3 u a + 2 u of its value, a = (m - z) / T: three
    roundings of the exponent (the difference, 1 / T, the product) and an exponential within one
    unit in the last place; their sum by the mean of that, `mean`. q takes two more roundings
    (1 / sum, the product) and the scale two (its own, the product); a class with an entry takes
    those of the difference and the scale. Weights below 2^-126 count as zero."""
    R, C = z.shape
    T, g = float(np.float32(T)), float(np.float32(g))
    there = (index >= 0) & (index < C) & (t != -np.inf)
    rows = there.any(1)
    n = rows.sum()
    grad, bound, losses, offs = np.zeros((R, C)), np.zeros((R, C)), [], []
    for r in np.flatnonzero(rows):
        with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
            i, tr = index[r][there[r]].astype(np.int64), t[r][there[r]].astype(np.float64) / T
            a = (z[r].astype(np.float64) - z[r].max()) / T
            e = np.exp(a)
            q = e / e.sum()
            log_q = a - np.log(e.sum())
            w = np.exp(tr - tr.max())
            p, log_p = w / w.sum(), tr - tr.max() - np.log(w.sum())
            loss = np.where(p > 0, p * (log_p - log_q[i]), np.where(np.isnan(p), np.nan, 0.0)).sum()
            each = 3 * np.abs(np.where(e > 0, a, 0.0)) + 2
            mean = (each * e).sum() / e.sum()
        whole = np.zeros(C)
        np.add.at(whole, i, p)
        s = g * T / n
        grad[r] = (q - whole) * s
        bound[r] = U * abs(s) * (q * (each + mean + 2) + 3 * np.abs(q - whole)) + abs(s) * 2.0 ** -125
        losses.append(loss)
        # binary64 but for the weights' sum; rounded once
        offs.append(U * (mean + np.abs(loss)) + 2.0 ** -45)
    with np.errstate(invalid="ignore", divide="ignore"):
        loss = T * T * np.float64(np.sum(losses)) / n
        off = T * T * np.sum(offs) / n + U * np.abs(loss)
    return loss, grad, off, bound
