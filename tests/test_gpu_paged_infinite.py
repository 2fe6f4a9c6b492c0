"""Paged attention: infinite queries.  A query with an Inf or NaN makes its row
NaN, in the open page (which is held in float32) as in full ones."""
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


@pytest.mark.parametrize("n", [30, 100])
def test_tiles_of_32_columns(ctx, padded, n):
    padded(2)
    _infinite_query(ctx, 2, 20, n)
