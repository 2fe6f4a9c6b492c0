"""Products on 8-bit floats over many blocks of the contraction: the unit that a
tile's sums are held in changes from block to block, and a part that an early
block has brought must not shrink or grow with each.

Where nothing is to be rounded the results are equal: scales that are all c * 2^e
give, to the bit, the sums of scales 2^e, times c.

Where the unit changes, there and back, each change multiplies the sum by a factor.
The factors' product is within 2^-23 of the units' quotient (2^-22 for a part that
comes in on the way; tests/test_fp8_units.py), a multiplication is off by at most half
a step, 2^-24, and so is the last one by the unit: (kb + 4) * 2^-24 of a first block's
part.  No mean is asked of it where nothing is added between: a sum that is the same
number again may be rounded to the same side again.

Where every block adds to the sum, roundings are of ever new digits and to nearest,
and fall to either side: what is left in the mean over all outputs is the factors'
2^-22, and of the others less than 2^-24."""
import numpy as np
import pytest
import torch

import fp8_model as fm
import fp8_shapes as fs
import qtts

pytestmark = pytest.mark.gpu


def _f32(a):
    return np.asarray(a, np.float32)


def _single(count):
    """Values of 1 to 2 with c * (1 / c) below 1 in f32, each quotient rounded."""
    c = _f32(1) + _f32(np.random.default_rng(1).random(20000))
    return c[c * (_f32(1) / c) < 1][:count]


def _pairs(count):
    """Pairs of such values with (a / b) * (b / a), of rounded quotients, furthest
    below 1."""
    r = np.random.default_rng(2)
    a, b = (_f32(1) + _f32(r.random(20000)) for _ in range(2))
    there_and_back = (a / b).astype(np.float64) * (b / a).astype(np.float64)
    best = np.argsort(there_and_back)[:count]
    assert there_and_back[best].max() < 1 - 2.0 ** -24
    return a[best], b[best]


class Product:
    def __init__(self, ctx, shape, k_used, low=0x28, high=0x40):
        self.ctx, (self.rows, self.n, self.k) = ctx, shape
        self.nb, self.kb = -(-self.n // 128), -(-self.k // 128)
        g = torch.Generator(device="cuda").manual_seed(7)
        # positive codes, and x of few bits under one power of two: 8 to 15, a column of 15
        self.codes = torch.randint(low, high, (self.n, self.k), generator=g, device="cuda", dtype=torch.uint8)
        self.x = torch.zeros((self.rows, self.k), device="cuda")
        self.x[:, :k_used] = torch.randint(8, 16, (self.rows, k_used), generator=g, device="cuda").float()
        self.x[:, :k_used:128] = 15
        self.ld = -(-self.n // 4) * 4

    def __call__(self, scales):
        s = torch.from_numpy(np.ascontiguousarray(scales, np.float32)).cuda()
        y = torch.full((self.rows, self.ld), 7.0, device="cuda")
        w = qtts.Fp8Weight(self.codes.data_ptr(), s.data_ptr(), self.n, self.k, self.k)
        torch.cuda.synchronize()
        self.ctx.fp8_gemm_device(w, self.x.data_ptr(), self.k, self.rows, y.data_ptr(), self.ld)
        self.ctx.synchronize()
        return y[:, :self.n]


@pytest.mark.parametrize("shape", [s for s, (_, division) in {**fs.TILES, **fs.DEEP}.items() if division == fs.WHOLE])
def test_equal_scales_are_one_factor(ctx, shape):
    p = Product(ctx, shape, shape[2])
    c = _single(p.nb)
    power = _f32(2.0) ** (np.arange(p.nb) % 7 - 3)
    sums = p(np.repeat(power[:, None], p.kb, 1))
    got = p(np.repeat((c * power)[:, None], p.kb, 1))
    each = torch.from_numpy(np.repeat(c, 128)[:p.n]).cuda()
    assert torch.equal(got, sums * each), float((got / (sums * each) - 1).abs().max())


@pytest.mark.parametrize("shape", [*fs.DEEP])
def test_units_that_alternate(ctx, shape):
    p = Product(ctx, shape, 128)
    a, b = _pairs(p.nb)
    got = p(np.where(np.arange(p.kb) % 2, b[:, None], a[:, None]))
    sums = p(np.ones((p.nb, p.kb)))  # of the first block: whole numbers over 32, exact
    each = torch.from_numpy(np.repeat(a, 128)[:p.n].astype(np.float64)).cuda()
    off = got.double() / (sums.double() * each) - 1
    assert float(off.abs().max()) <= (p.kb + 4) * 2.0 ** -24


@pytest.mark.parametrize("shape", [*fs.DEEP])
@pytest.mark.parametrize("kind", ["equal", "alternating", "any"])
def test_sums_of_one_sign_do_not_drift(ctx, shape, kind):
    p = Product(ctx, shape, shape[2], low=0x20, high=0x48)
    a, b = _pairs(p.nb)
    scales = {"equal": np.repeat(_single(p.nb)[:, None], p.kb, 1),
              "alternating": np.where(np.arange(p.kb) % 2, b[:, None], a[:, None]),
              "any": 1 + np.random.default_rng(3).random((p.nb, p.kb))}[kind].astype(np.float32)
    got = p(scales)
    values = torch.from_numpy(fm.VALUES).cuda()[p.codes.long()]
    each = torch.from_numpy(scales).cuda().double()
    values *= each.repeat_interleave(128, 0)[:p.n].repeat_interleave(128, 1)[:, :p.k]
    ref = p.x.double() @ values.T.contiguous()
    assert abs(float((got.double() / ref - 1).mean())) <= 5 * 2.0 ** -24
