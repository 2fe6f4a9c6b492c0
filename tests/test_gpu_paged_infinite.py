"""Paged attention: infinite queries, and infinite keys in the open page (which
is held in float32).  A query with an Inf or NaN makes its row NaN; a key whose
score is -Inf has no weight."""
import numpy as np
import pytest
import torch

import test_gpu_paged as base
from test_gpu_paged_wide import padded  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

MODES = [(1, 1), (4, 1), (1, 3), (6, 1), (2, 20)]


def _infinite_query(ctx, group, rows, n):
    hd, page = 64, 64
    k = np.abs(base._normal(1, n, hd))
    c = base.Cache(1, hd, page, 1, 4)
    c.append(ctx, c.seqs([0], [n]), base._up(k), base._up(base._normal(2, n, hd)))
    q = base._normal(3, rows, group * hd)
    s = c.seqs([n - rows], [rows])
    ref = c.attend(ctx, s, base._up(q), group)
    for bad in (np.inf, -np.inf, np.nan):
        q[-1, 5] = bad  # the first head of the last row: its scores are all +Inf, -Inf or NaN
        got = c.attend(ctx, s, base._up(q), group)
        assert torch.isnan(got[-1, :hd]).all()
        assert torch.equal(got[-1, hd:], ref[-1, hd:]) and torch.equal(got[:-1], ref[:-1])


@pytest.mark.parametrize("n", [30, 100])  # all in the open page; with a full one
@pytest.mark.parametrize("group,rows", MODES)
def test_infinite_query(ctx, group, rows, n):
    _infinite_query(ctx, group, rows, n)


def _infinite_key(ctx, group, rows, n):
    """As if the token were not there: beside the same call with its score so low
    that nothing is left of it."""
    hd, page = 64, 64
    k, v = base._normal(1, n, hd), base._normal(2, n, hd)
    q = base._normal(3, rows, group * hd)
    q[:, 5::hd] = 1 + np.abs(q[:, 5::hd])
    gone = n - rows - 2  # seen by all rows
    c = base.Cache(1, hd, page, 1, 4)
    s = c.seqs([n - rows], [rows])
    out = []
    for low in (-1e30, -np.inf):
        k[gone, 5] = low
        c.append(ctx, c.seqs([0], [n]), base._up(k), base._up(v))
        out.append(c.attend(ctx, s, base._up(q), group))
    assert torch.isfinite(out[0]).all() and torch.equal(*out)


@pytest.mark.parametrize("n", [30, 100])
@pytest.mark.parametrize("group,rows", MODES)
def test_infinite_key(ctx, group, rows, n):
    _infinite_key(ctx, group, rows, n)


@pytest.mark.parametrize("n", [30, 100])
def test_tiles_of_32_columns(ctx, padded, n):
    padded(2)
    _infinite_query(ctx, 2, 20, n)
    _infinite_key(ctx, 2, 20, n)
