"""Paged attention at scores so large that float32's steps, or even int32's
range, lie between them.  One rounding of a score to float32 is then many units,
so that no softmax of such scores is given by their float32 values but for two
things, which are checked here: a token whose score is above all others' by more
than the roundings has all the weight, and any result lies between the least and
the largest of the values that the row sees."""
import numpy as np
import pytest

import paged_model as pm
import test_gpu_paged as base
from test_gpu_paged_wide import padded  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

KVH, HD, PAGE = 1, 64, 16
# of scores in units of log2, about
SIZES = [2.0 ** 20, 2.0 ** 25, 1.3 * 2.0 ** 27, 1.9 * 2.0 ** 27, 2.0 ** 31, 2.0 ** 33, 1e12, 1e20, 1e30, 1e36]


def _cache(ctx, k, v):
    n = k.shape[0]
    c = base.Cache(KVH, HD, PAGE, 1, -(-n // PAGE))
    c.append(ctx, c.seqs([0], [n]), base._up(k), base._up(v))
    return c, [pm.held(a.reshape(n, KVH, HD), PAGE) for a in (k, v)]


def _one_above(ctx, group, rows, n, order):
    """Scores of every size and sign in `order`.  The weight of the largest is held
    to 22 bits, hi + lo (2^-22), and it and the sum of probabilities to the float32
    steps of an exponential, a logarithm, an inverse, a quotient (less than 12
    steps of 2^-23 with V's exponent below 4): 2^-19 of the largest value that its
    block has is left to them."""
    r = np.random.default_rng(n)
    for i, size in enumerate(SIZES):
        along = r.standard_normal(n)
        if order != "any":
            along = np.sort(along)[::1 if order == "rising" else -1]
        way = r.choice([-1.0, 1.0], HD)
        k = (along[:, None] * way).astype(np.float32)
        v = base._normal(40 + i, n, HD)
        q = np.tile(way * size / HD ** 0.5, (rows, group)).astype(np.float32)
        c, (hk, hv) = _cache(ctx, k, v)
        got = c.attend(ctx, c.seqs([n - rows], [rows]), base._up(q), group).cpu().numpy().reshape(rows, group, HD)
        # float32 roundings of a score: 64 products and the operands' 2^-22
        slack = 2 * size * np.abs(hk).max() * (2.0 ** -22 + 64 * 2.0 ** -24)
        for j in range(rows):
            seen = n - rows + j + 1
            s = hk[:seen, 0].astype(np.float64) @ way * size / HD
            best = np.argmax(s)
            room = 2.0 ** -19 * np.abs(hv[:seen]).max()
            lo, hi = hv[:seen, 0].min(0), hv[:seen, 0].max(0)
            assert np.all((got[j] >= lo - room) & (got[j] <= hi + room)), (size, j)
            if seen == 1 or s[best] - np.delete(s, best).max() > slack + 64:
                assert np.all(np.abs(got[j] - hv[best, 0]) <= room), (size, j)


MODES = [(1, 1), (4, 1), (1, 3), (6, 1), (1, 20), (8, 5)]


@pytest.mark.parametrize("order", ["rising", "falling", "any"])
@pytest.mark.parametrize("n", [9, 48, 300, 2000])
@pytest.mark.parametrize("group,rows", MODES)
def test_one_above_all_others(ctx, group, rows, n, order):
    _one_above(ctx, group, min(rows, n), n, order)


@pytest.mark.parametrize("order", ["rising", "falling", "any"])
@pytest.mark.parametrize("n", [48, 300, 2000])
def test_one_above_all_others_in_tiles_of_32(ctx, padded, n, order):
    padded(2)
    _one_above(ctx, 2, 20, n, order)


def _alike(ctx, group, rows, n, sizes):
    """The same score for every token (a definite one for none)."""
    rows = min(rows, n)
    way = np.random.default_rng(7).choice([-1.0, 1.0], HD)
    k = np.tile(way, (n, 1)).astype(np.float32)
    v = (1 + np.random.default_rng(8).random((n, HD))).astype(np.float32)
    for size in sizes:
        for sign in (1, -1):
            q = np.tile(sign * way * size / HD ** 0.5, (rows, group)).astype(np.float32)
            c, (_, hv) = _cache(ctx, k, v)
            got = c.attend(ctx, c.seqs([n - rows], [rows]), base._up(q), group).cpu().numpy().reshape(rows, group, HD)
            for j in range(rows):
                mine = hv[:n - rows + j + 1, 0]
                room = 2.0 ** -19 * mine.max()
                assert np.all((got[j] >= mine.min(0) - room) & (got[j] <= mine.max(0) + room)), (size, sign, j)


NEAR_SIZES = [2.0 ** 20, 2.0 ** 25, 1.1 * 2.0 ** 26, 1.3 * 2.0 ** 26, 1.1 * 2.0 ** 27, 1.3 * 2.0 ** 27, 2.0 ** 30,
              1.3 * 2.0 ** 31, 1e12, 1.1e20, 1.3e30, 1.7e36]


@pytest.mark.parametrize("n", [9, 300, 2000])
@pytest.mark.parametrize("group,rows", MODES)
def test_all_alike(ctx, group, rows, n):
    _alike(ctx, group, rows, n, NEAR_SIZES)


@pytest.mark.parametrize("n", [300, 2000])
def test_all_alike_in_tiles_of_32(ctx, padded, n):
    padded(2)
    _alike(ctx, 2, 20, n, NEAR_SIZES)


@pytest.mark.parametrize("size", [1e-30, 1e-25, 1e25, 1e38])
@pytest.mark.parametrize("n", [9, 300])
@pytest.mark.parametrize("group,rows", MODES)
def test_all_alike_with_large_and_small_values(ctx, group, rows, n, size):
    """Finite, and between the values, whatever V's size is."""
    rows = min(rows, n)
    way = np.random.default_rng(7).choice([-1.0, 1.0], HD)
    k = np.tile(way, (n, 1)).astype(np.float32)
    v = ((1 + np.random.default_rng(8).random((n, HD))) * size).astype(np.float32)
    c, (_, hv) = _cache(ctx, k, v)
    for score in NEAR_SIZES:
        q = np.tile(way * score / HD ** 0.5, (rows, group)).astype(np.float32)
        got = c.attend(ctx, c.seqs([n - rows], [rows]), base._up(q), group).cpu().numpy().reshape(rows, group, HD)
        room = 2.0 ** -19 * np.float64(hv.max()) + 2.0 ** -148
        assert np.all((got >= hv.min() - room) & (got <= hv.max() + room)), score
