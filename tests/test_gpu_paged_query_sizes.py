"""Paged attention of queries of any size over keys of the opposite one: scores as
ordinary ones have them, whose factors lie at either end of float32.  The
tolerances are test_gpu_paged's, with the half steps that least floats are rounded
to: a key or a query of size 1e-37 to 2^-24 of itself, as others."""
import numpy as np
import pytest

import test_gpu_paged as base
from test_gpu_paged_wide import padded  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

SIZES = [3e-38, 1e-37, 1e-36, 1e-33, 1e-30, 1e-15, 1e15, 1e30, 1e33, 1e36, 1e37, 3e37]


def _attend(ctx, group, rows, n, hd, size):
    kvh, page = 1, 32
    k, v = base._normal(1, n, kvh * hd) * np.float32(1 / size), base._normal(2, n, kvh * hd)
    q = base._normal(3, rows, kvh * group * hd) * np.float32(2 * size)
    c = base.Cache(kvh, hd, page, 1, -(-n // page))
    c.append(ctx, c.seqs([0], [n]), base._up(k), base._up(v))
    got = c.attend(ctx, c.seqs([n - rows], [rows]), base._up(q), kvh * group).cpu().numpy()
    held = [base.pm.held(x.reshape(n, kvh, hd), page) for x in (k, v)]
    base._check(got.reshape(rows, -1, hd), q.reshape(rows, -1, hd), *held, n - rows, hd ** -0.5, 0)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("n", [30, 64, 205])
@pytest.mark.parametrize("group,rows,hd", [(1, 1, 64), (4, 1, 128), (1, 3, 128), (6, 1, 64), (2, 20, 128)])
def test_queries_of_any_size(ctx, group, rows, hd, n, size):
    _attend(ctx, group, rows, n, hd, size)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("n", [30, 64, 205])
@pytest.mark.parametrize("hd", [64, 128])
def test_tiles_of_32_columns(ctx, padded, hd, n, size):
    padded(2)
    _attend(ctx, 2, 20, n, hd, size)
