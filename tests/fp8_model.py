"""8-bit floats (e4m3) and products on them restated in 64 bits (numpy)."""
import numpy as np

BLOCK = 128


def _values():
    v = np.zeros(256)
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        v[c] = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        if c & 127 == 127:
            v[c] = np.nan
        if c & 128:
            v[c] = -v[c]
    return v


VALUES = _values()


def power(x):
    """The least power of two s with max|x| / s <= 448, 2^-110 at least; NaN
    where a value is not finite."""
    top = np.abs(np.asarray(x, np.float64)).max()
    if not np.isfinite(top):
        return np.nan
    s = 2.0 ** -110
    while top / s > 448:
        s *= 2
    return s


def units(x, s):
    """x / s, at most the last code of 2^120 that f32 holds."""
    u = np.asarray(x, np.float64) / s
    return np.clip(u, -240, 240) if s == 2.0 ** 120 else u


def rounded(x):
    """Values within 448 to the nearest e4m3, ties to even."""
    x = np.asarray(x, np.float64)
    step = np.exp2(np.maximum(np.frexp(x)[1], -5) - 4)
    return np.rint(x / step) * step


def blocks(x):
    """x (rows of a last axis) as the product takes it: each 128 values
    rounded with their power."""
    x = np.asarray(x, np.float64)
    out = np.empty_like(x)
    for at in range(0, x.shape[-1], BLOCK):
        for i in np.ndindex(x.shape[:-1]):
            part = x[i][at:at + BLOCK]
            s = power(part)
            out[i][at:at + BLOCK] = np.nan if np.isnan(s) else rounded(units(part, s)) * s
    return out


def weight(codes, scales):
    """Values of a weight [n][k]."""
    n, k = codes.shape
    s = np.repeat(np.repeat(scales.astype(np.float64), BLOCK, 0)[:n], BLOCK, 1)[:, :k]
    return VALUES[codes] * s


def quantized(w):
    """(codes, scales) of f32 rows [n][k]."""
    n, k = w.shape
    codes = np.zeros((n, k), np.uint8)
    scales = np.zeros((-(-n // BLOCK), -(-k // BLOCK)), np.float32)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            at = np.s_[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK]
            s = power(w[at])
            scales[i, j] = s
            if not np.isnan(s):
                q = rounded(units(w[at], s))
                low = np.abs(q) < 2.0 ** -6
                e = np.where(low, 0, np.frexp(q)[1] + 6)
                m = np.where(low, np.abs(q) * 512, np.abs(q) * np.exp2(10.0 - e) - 8)
                codes[at] = (np.signbit(w[at]).astype(np.int64) << 7 | e << 3 | m.astype(np.int64)).astype(np.uint8)
    return codes, scales


def product(x, codes, scales, add=None):
    """y and, for its rounding, the sum of the products' magnitudes."""
    q, w = blocks(x), weight(codes, scales)
    y, mass = q @ w.T, np.abs(q) @ np.abs(w).T
    return (y, mass) if add is None else (y + add, mass + np.abs(add))
