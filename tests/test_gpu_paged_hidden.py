"""Paged attention: what a mask hides beside a page whose V is nothing next to
the others', in one step of tokens.  What is hidden is finite in one call and
NaN in the other: the same values.

Not the same bits: whether probabilities are taken from V's weights or by
themselves is one decision for all columns of a wave, and in the other call some
of them see the NaN.  By themselves they are 2^(t - lg + k), whose terms and sums
are below 256 in size and rounded by half a step there, 2^-17, four of them, and
from the weights 2^t, two: 6 ln 2 2^-17 < 2^-14 of a probability's share."""
import pytest
import torch

import test_gpu_paged as base
from test_gpu_paged_wide import padded  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def _pages(ctx, kvh, hd, page, n, light, size):
    """n tokens; page `light` holds V of that size, zeros or far below the rest."""
    c = base.Cache(kvh, hd, page, 1, -(-n // page))
    k, v = base._normal(1, n, kvh * hd), base._normal(2, n, kvh * hd)
    v[light * page:(light + 1) * page] *= size
    c.append(ctx, c.seqs([0], [n]), base._up(k), base._up(v))
    return c


def _same(ctx, c, s, q, heads, hidden, window, rows):
    ref = c.attend(ctx, s, q, heads, window)[rows].clone()
    assert torch.isfinite(ref).all()
    for scales in ([c.v_scales], [c.k_scales], [c.v_scales, c.k_scales]):
        kept = [b.clone() for b in scales]
        for b in scales:
            b[int(c.table[0, hidden])] = float("nan")
        got = c.attend(ctx, s, q, heads, window)[rows]
        for b, was in zip(scales, kept):
            b.copy_(was)
        assert ((got - ref).abs() <= 2.0 ** -14 * ref.abs().max()).all()


def _before_the_window(ctx, page, hd, group, rows, size):
    """The first row's window begins with the light page, whose neighbour in a step
    of 64 tokens (32 in tiles of 32 columns) lies before it."""
    light = 2 * (64 // page) + 1
    start = (light + 3) * page + 3
    window = start - light * page + 1
    c = _pages(ctx, 2, hd, page, start + rows, light, size)
    q = base._up(base._normal(3, rows, 2 * group * hd))
    _same(ctx, c, c.seqs([start], [rows]), q, 2 * group, light - 1, window, slice(0, rows))


def _behind_the_row(ctx, page, hd, group, rows, size):
    """Rows in the light page, before the next one of their step, which rows of the
    same tile see."""
    light = 64 // page
    start = light * page + 5
    c = _pages(ctx, 2, hd, page, start + rows, light, size)
    assert rows >= 2 * page
    q = base._up(base._normal(3, rows, 2 * group * hd))
    _same(ctx, c, c.seqs([start], [rows]), q, 2 * group, light + 1, 0, slice(0, page - 5))


SIZES = [0.0, 1e-25]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("group,rows", [(1, 1), (4, 1), (1, 3), (6, 1), (2, 5), (1, 20)])
@pytest.mark.parametrize("page,hd", [(16, 64), (16, 128), (32, 64), (32, 128)])
def test_before_the_window(ctx, page, hd, group, rows, size):
    _before_the_window(ctx, page, hd, group, rows, size)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("group,rows", [(1, 80), (3, 70)])
@pytest.mark.parametrize("page,hd", [(16, 64), (16, 128), (32, 64), (32, 128)])
def test_behind_the_row(ctx, page, hd, group, rows, size):
    _behind_the_row(ctx, page, hd, group, rows, size)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("hd", [64, 128])
def test_tiles_of_32_columns(ctx, padded, hd, size):
    padded(2)
    _before_the_window(ctx, 16, hd, 2, 20, size)
    _behind_the_row(ctx, 16, hd, 2, 40, size)
