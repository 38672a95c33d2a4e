"""Float64 oracle of 8-bit rows and weights (fn_fp8_*): e4m3 by its definition (1 sign, 4 exponent and 3 mantissa bits, bias 7, no
infinities, largest number 448, NaN 0x7f), groups of 128, from the formulas."""

import numpy as np

GROUP, TINY = 128, 2.0 ** -116


def value(code):
    """What e4m3 bytes stand for."""
    c = np.asarray(code, np.int64)
    e, f = c >> 3 & 15, c & 7
    v = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >> 7 & 1, -v, v)


def e4m3(x):
    """x rounded to the nearest e4m3 number, ties to even, as float64 (|x| up to 448; NaN stays)."""
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        step = 2.0 ** (np.maximum(np.floor(np.log2(np.abs(x))), -6) - 3)
        return np.where(x == 0, x, np.clip(np.round(x / step) * step, -448, 448))


def groups(y, down, fp32=True):
    """(code values, scales) of y in groups of `down` rows x 128 columns. fp32: quotients and products in that type, as the kernels
    take them (else in 64 bits)."""
    t = np.float32 if fp32 else np.float64
    y = np.asarray(y, t)
    rows, cols = y.shape
    q = np.zeros(y.shape)
    s = np.zeros((-(-rows // down), -(-cols // GROUP)))
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            at = (slice(i * down, (i + 1) * down), slice(j * GROUP, (j + 1) * GROUP))
            a = t(np.maximum(np.abs(y[at]).max(), t(TINY)))
            with np.errstate(invalid="ignore"):
                q[at] = e4m3(y[at] * (t(448) * (t(1) / a)))
            s[i, j] = a * (t(1) / t(448))
    return q, s


def rms(h, weight, eps, fp32=True):
    """The normed rows; fp32: the factor in 64 bits, the products in fp32."""
    h = np.asarray(h, np.float64)
    r = 1 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    with np.errstate(invalid="ignore"):
        if not fp32:
            return h * r * weight
        return h.astype(np.float32) * r.astype(np.float32) * np.asarray(weight, np.float32)


def spread(scale, rows, cols, down):
    return np.repeat(np.repeat(scale, down, 0)[:rows], GROUP, 1)[:, :cols]


def product(xq, xs, wq, ws):
    """From code values and scales, in 64 bits; and the sum of the terms' magnitudes, which errors are relative to."""
    x = xq * spread(xs, *xq.shape, 1)
    w = wq * spread(ws, *wq.shape, GROUP)
    return x @ w.T, np.abs(x) @ np.abs(w).T
