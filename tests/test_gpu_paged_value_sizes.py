"""Paged attention: values of one size or of another in each row, broad softmaxes,
in the open page and behind full ones.

Tolerance: as test_gpu_paged's for values of every size: 2^-14 of a weight for the
roundings of V's logarithm with a score, its bound of scores and sums, a least step
of 2^-28 of the largest weight for each token (times its block's largest value),
and a step of the least floats."""
import numpy as np
import pytest

import paged_model as pm
import test_gpu_paged as base
from test_gpu_paged_wide import padded  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

SIZES = [1e-37, 1e-30, 1e-24, 1e-20, 1e20, 1e24, 1e26, 1e30, 1e33, 1e36, 3e38]


def _attend(ctx, group, rows, n, sizes):
    kvh, hd, page = 1, 64, 64
    k, q = base._normal(1, n, hd), base._normal(3, rows, group * hd)
    v = np.clip(base._normal(2, n, hd), -1, 1) * np.resize(np.float32(sizes), n)[:, None]
    c = base.Cache(kvh, hd, page, 1, -(-n // page))
    c.append(ctx, c.seqs([0], [n]), base._up(k), base._up(v))
    got = c.attend(ctx, c.seqs([n - rows], [rows]), base._up(q), group).cpu().numpy().reshape(rows, group, hd)
    hk, hv = (pm.held(x.reshape(n, kvh, hd), page) for x in (k, v))
    ref, mass, slack = pm.attention(q.reshape(rows, group, hd), hk, hv, n - rows, hd ** -0.5, 0)
    tol = mass * (2 * slack[..., None] + 2.0 ** -14 + (n / 64 + 64) * 2.0 ** -24)
    tol += 2.0 ** -28 * np.abs(hv).max(-1).astype(np.float64).sum() + 2.0 ** -148
    assert np.all(np.abs(got - ref) <= tol), float((np.abs(got - ref) / tol).max())


MODES = [(1, 1), (4, 1), (1, 3), (6, 1), (2, 20)]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("n", [30, 60, 120])
@pytest.mark.parametrize("group,rows", MODES)
def test_one_size(ctx, group, rows, n, size):
    _attend(ctx, group, rows, n, [size])


@pytest.mark.parametrize("n", [30, 60, 120])
@pytest.mark.parametrize("group,rows", MODES)
def test_a_size_a_row(ctx, group, rows, n):
    for first in range(len(SIZES)):
        _attend(ctx, group, rows, n, SIZES[first:first + 2] or SIZES)
        _attend(ctx, group, rows, n, SIZES[first:] + [0.0] + SIZES[:first])


@pytest.mark.parametrize("n", [30, 60, 120])
def test_tiles_of_32_columns(ctx, padded, n):
    padded(2)
    for size in SIZES:
        _attend(ctx, 2, 20, n, [size])
    _attend(ctx, 2, 20, n, SIZES)
