"""Paged attention: one token with most of the probability and thousands whose
weights lie about the least step that a weight is held to (2^-28 of a reference
on int8 products).  Their share, 1e-4 of the sum here, has to reach the output.

Tolerance, absolute, with probabilities of sum 1 and V about 1.  A lane hands what
a weight's rounding left on to a later one.  So of the weights' sum at most half
a unit of 2^-28 is missing for each of the 64 chains of the wave whose reference
the large weight is, 64 * 2^-29 = 1.2e-7.  And where V differs between the tokens of a
chain, its differences (a spread of 0.43: 0.5 |n| of two) times rests of at most
half a unit add up as their squares do, over 30000 tokens sqrt(30000) * 0.5 * 0.43
* 2^-28 = 1.4e-7, four deviations of which are 5.6e-7.  Then the float32 sums, as
test_gpu_paged counts them, 3e-7: 1e-6 together."""
import numpy as np
import pytest

import paged_model as pm
import test_gpu_paged as base

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("octaves", [26.0, 27.6, 28.05, 28.9, 30.0, 31.3, 33.0])
@pytest.mark.parametrize("group,rows", [(1, 1), (4, 1), (2, 2), (6, 1), (2, 20)])
def test_weights_about_the_least_step(ctx, group, rows, octaves):
    kvh, hd, page, n, pad = 1, 64, 64, 30000, 511
    c = base.Cache(kvh, hd, page, 1, -(-(n + rows) // page))
    q = np.tile(base._normal(1, 1, hd), (rows, group)) + 0.01 * base._normal(2, rows, group * hd)
    k, v = 0.02 * base._normal(3, n + rows, hd), 0.5 + 0.5 * np.abs(base._normal(4, n + rows, hd))
    v[1000] *= 0.01  # so that the others' share shows
    k[1000] = q[0, :hd] * (octaves * np.log(2) * hd ** 0.5 / (q[0, :hd] ** 2).sum())
    c.append(ctx, c.seqs([0], [n + rows]), base._up(k), base._up(v))
    s = c.seqs([0] * pad + [n], [0] * pad + [rows], table=c.table.expand(pad + 1, -1).contiguous(), slots=[0] * (pad + 1))
    got = c.attend(ctx, s, base._up(q), group).cpu().numpy().reshape(rows, group, hd)
    hk, hv = (pm.held(x.reshape(n + rows, kvh, hd), page) for x in (k, v))
    ref, _, _ = pm.attention(q.reshape(rows, group, hd), hk, hv, n, hd ** -0.5, 0)
    assert np.abs(got - ref).max() < 1e-6


@pytest.mark.parametrize("group", [1, 3])
def test_each_weight_by_itself(ctx, group):
    """A dimension where one token alone has a value: its weight, whatever the
    others' roundings handed on to it, is held to 2^-28 of the largest (and to
    test_gpu_paged's float32 roundings of its own)."""
    kvh, hd, page, n = 2, 128, 16, 16
    for seed in range(40):
        c = base.Cache(kvh, hd, page, 1, 1)
        k, v = base._normal(3 * seed, n, kvh * hd), np.zeros((n, kvh * hd), np.float32)
        for t in range(n):
            v[t, t::16] = 1 + 0.01 * t
        q = 4 * base._normal(3 * seed + 1, 1, kvh * group * hd)
        c.append(ctx, c.seqs([0], [n]), base._up(k), base._up(v))
        got = c.attend(ctx, c.seqs([n - 1], [1]), base._up(q), kvh * group).cpu().numpy().reshape(1, -1, hd)
        hk, hv = (pm.held(x.reshape(n, kvh, hd), page) for x in (k, v))
        ref, mass, slack = pm.attention(q.reshape(1, -1, hd), hk, hv, n - 1, hd ** -0.5, 0)
        tol = mass * (2 * slack[..., None] + 64 * 2.0 ** -24) + 2.0 ** -28 * hv.max()
        assert np.all(np.abs(got - ref) <= tol), seed
