"""Microscaled tensors in 64 bits, from the definition of the formats: the code tables are written
out value by value, scales come from logarithms and codes from the nearest table entry."""
import numpy as np

# (exponent bits, mantissa bits, bias, codes that are numbers)
_LAYOUT = {"e4m3": (4, 3, 7, 0x7f), "e5m2": (5, 2, 15, 0x7c), "e2m1": (2, 1, 1, 0x08)}
LEAST_EXPONENT = -110
FORMATS = tuple(_LAYOUT)


def table(format):
    """The values of the positive codes 0, 1, 2, ... that are finite numbers."""
    e_bits, m_bits, bias, n = _LAYOUT[format]
    out = []
    for c in range(n):
        e, m = c >> m_bits, c & ((1 << m_bits) - 1)
        out.append(m * 2.0 ** (1 - bias - m_bits) if e == 0 else
                   (1 + m / 2.0 ** m_bits) * 2.0 ** (e - bias))
    return np.array(out)


def groups(C):
    return -(-C // 128)


def encode(x, format, keep_nonzero=False):
    """(one code a value [R, 128 G], scale bytes [R, 4 G])."""
    x = np.asarray(x, np.float32).astype(np.float64)
    R, C = x.shape
    v = np.zeros((R, groups(C) * 128))
    v[:, :C] = x
    b = v.reshape(R, -1, 32)
    t = table(format)
    finite = np.isfinite(b)
    largest = np.max(np.where(finite, np.abs(b), 0.0), axis=2, initial=0.0)
    with np.errstate(divide="ignore"):
        e = np.where(largest > 0, np.ceil(np.log2(largest / t[-1])), -1000.0).astype(int)
    # the logarithm may round: settle on the smallest power of two with largest <= t[-1] 2^e
    e = np.where(largest <= np.ldexp(t[-1], e - 1), e - 1, e)
    e = np.where(largest > np.ldexp(t[-1], e), e + 1, e)
    e = np.maximum(e, LEAST_EXPONENT)
    # a finite value stays finite: none rounds to 2^128, above the binary32 range
    m = np.minimum(np.abs(np.where(finite, b, 0.0)), 2.0 ** 128 * (1 - 2.0 ** -(_LAYOUT[format][1] + 1)))
    m = m / np.ldexp(1.0, e)[:, :, None]
    middle = (t[1:] + t[:-1]) / 2
    below = np.searchsorted(middle, m, side="left")   # a value on a middle stays at the code below
    above = np.searchsorted(middle, m, side="right")  # ... or goes to the one above
    code = np.where(below % 2 == 0, below, above)
    if keep_nonzero:
        code = np.where((code == 0) & (b != 0) & finite, 1, code)
    sign = np.signbit(b)
    scales = (e + 127).astype(np.uint8)
    if format == "e2m1":
        code = code + 8 * sign
        lost = ~finite.all(axis=2)
        code[lost] = 0
        scales[lost] = 255
    else:
        code = np.where(np.isnan(b), 0x7f, code)
        code = np.where(np.isinf(b), 0x7c if format == "e5m2" else 0x7f, code)
        code = code + 128 * sign
    return code.reshape(R, -1).astype(np.uint8), scales


def pack(code, format):
    """One code a value as the bytes of a microscaled tensor."""
    if format != "e2m1":
        return code
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)


def values(code, scales, C, format):
    """What codes (one a value) and scales stand for, [R, C] in 64 bits."""
    code = np.asarray(code, np.int64)
    half = 8 if format == "e2m1" else 128
    t = np.full(half, np.nan)
    t[:len(table(format))] = table(format)
    if format == "e5m2":
        t[0x7c] = np.inf
    t = np.concatenate([t, -t])
    s = np.asarray(scales, np.int64)
    f = np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    R = code.shape[0]
    return (t[code].reshape(R, -1, 32) * f[:, :, None]).reshape(R, -1)[:, :C]


def stored(x, format, keep_nonzero=False):
    """(packed codes, scales, the values that they stand for)."""
    code, s = encode(x, format, keep_nonzero)
    return pack(code, format), s, values(code, s, np.asarray(x).shape[1], format)


def activate(act, z):
    with np.errstate(over="ignore"):
        return {None: lambda: z, "none": lambda: z, "relu": lambda: np.where(z > 0, z, 0.0),
                "tanh": lambda: np.tanh(z), "sigmoid": lambda: 1 / (1 + np.exp(-z))}[act]()


def slope(act, y):
    return {None: lambda: np.ones_like(y), "none": lambda: np.ones_like(y),
            "relu": lambda: (y > 0).astype(y.dtype), "tanh": lambda: 1 - y * y,
            "sigmoid": lambda: y * (1 - y)}[act]()
