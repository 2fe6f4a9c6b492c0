"""The paged 8-bit cache and its operators restated in 64 bits (numpy)."""
import numpy as np


def rotated(x, norm, eps, cos, sin, positions):
    """[rows][heads][hd] -> normed and rotated, in 64 bits (not rounded)."""
    x = np.asarray(x, np.float64)
    if norm is not None:
        x = x * norm.astype(np.float64) / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
    if cos is not None:
        half = x.shape[-1] // 2
        c, s = cos[positions].astype(np.float64)[:, None], sin[positions].astype(np.float64)[:, None]
        x = np.concatenate([x[..., :half] * c - x[..., half:] * s, x[..., half:] * c + x[..., :half] * s], -1)
    return x


def block(x):
    """(codes, scale) of one block of f32 values."""
    top = np.abs(x).max()
    if not np.isfinite(top):
        return np.zeros(x.shape, np.int8), np.float32(np.nan)
    if top == 0:
        return np.zeros(x.shape, np.int8), np.float32(0)
    return np.rint(x.astype(np.float64) * 127 / np.float64(top)).astype(np.int8), np.float32(top) / np.float32(127)


def held(x, page):
    """f32 rows [tokens][kv_heads][hd] of one sequence as the cache holds them."""
    out = x.copy()
    for p in range(x.shape[0] // page):
        for h in range(x.shape[1]):
            rows = slice(p * page, (p + 1) * page)
            codes, scale = block(x[rows, h])
            out[rows, h] = codes.astype(np.float32) * scale
    return out


def attention(q, k, v, start, scale, window, absent=()):
    """q [rows][heads][hd] over k, v [tokens][kv_heads][hd] (as held): out and,
    for each row and head, sum p |v| and the largest sums that bound the
    rounding of a score."""
    rows, heads, hd = q.shape
    group = heads // k.shape[1]
    out, mass = np.zeros(q.shape), np.zeros(q.shape)
    slack = np.zeros((rows, heads))
    token = np.arange(k.shape[0])
    gone = np.isin(token, np.asarray(list(absent), np.int64))
    with np.errstate(invalid="ignore"):
        for i in range(rows):
            seen = (token <= start + i) & ~gone
            if window:
                seen &= token > start + i - window
            if not seen.any():
                continue
            for h in range(heads):
                kk, vv = k[seen, h // group].astype(np.float64), v[seen, h // group].astype(np.float64)
                x = q[i, h].astype(np.float64)
                s = kk @ x * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[i, h], mass[i, h] = w @ vv, w @ np.abs(vv)
                slack[i, h] = scale * (2.0 ** -22 * np.abs(x).max() * np.abs(kk).sum(1).max()
                                       + hd * 2.0 ** -24 * (np.abs(kk) @ np.abs(x)).max())
    return out, mass, slack
