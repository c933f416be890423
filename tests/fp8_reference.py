"""The block-scaled 8-bit operators in float64 (NumPy), for the tests.

Written from the format's definition: a block's scale is the smallest power
of two s with max|x| / s <= 448 (1 for zeros, at least 2^-127), its values
are x / s rounded to the nearest e4m3 value, ties to even."""

import numpy as np

BLOCK = 128


def e4m3(v):
    """Nearest e4m3 value (3 mantissa bits, smallest step 2^-9); |v| <= 448."""
    v = np.asarray(v, np.float64)
    _, p = np.frexp(np.where(v == 0, 1.0, np.abs(v)))  # |v| in [2^(p-1), 2^p)
    step = np.ldexp(1.0, np.maximum(p - 1, -6) - 3)
    return np.rint(v / step) * step


def scale_exponent(amax):
    amax = np.asarray(amax, np.float64)
    e = np.full(amax.shape, -127)
    for k in range(-127, 128):  # the smallest exponent that fits
        e = np.where(amax / np.ldexp(1.0, k) > 448, k + 1, e)
    return np.where(amax == 0, 0, e)


def _block_max(x, rows):
    """Largest finite |x| of each rows x 128 block."""
    m, k = x.shape
    a = np.where(np.isfinite(x), np.abs(x), 0.0)
    mb, kb = -(-m // rows), -(-k // BLOCK)
    p = np.zeros((mb * rows, kb * BLOCK))
    p[:m, :k] = a
    return p.reshape(mb, rows, kb, BLOCK).max(axis=(1, 3))


def spread(s, rows, shape):
    """Block scales as a matrix of `shape`."""
    return np.repeat(np.repeat(s, rows, 0), BLOCK, 1)[:shape[0], :shape[1]]


def quantize(x, rows=1):
    """(values, scales) in float64; NaN where x is not finite."""
    x = np.asarray(x, np.float64)
    s = np.ldexp(1.0, scale_exponent(_block_max(x, rows)))
    with np.errstate(invalid="ignore"):
        v = x / spread(s, rows, x.shape)
    return np.where(np.isfinite(x), e4m3(np.where(np.isfinite(x), v, 0.0)), np.nan), s


def rms_norm(x, weight, eps, residual=None):
    h = np.asarray(x, np.float64) + (0 if residual is None else np.asarray(residual, np.float64))
    y = h / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    return (y if weight is None else y * np.asarray(weight, np.float64)), h


def linear(a, w, bias=None, relu=False, residual=None):
    """float64 values a [m, k], w [n, k]; also sum |a||w|, which bounds the rounding of the sum."""
    y = a @ w.T
    if bias is not None:
        y = y + bias
    if relu:
        y = np.where(np.isnan(y) | (y > 0), y, 0.0)
    if residual is not None:
        y = y + residual
    return y, np.abs(a) @ np.abs(w).T
