"""Products on 8-bit floats whose blocks' scales lie far apart along k, on every
kernel (tests/fp8_shapes.py), against 64 bits (tests/fp8_model.py).

Tolerance.  Products of two codes under powers of two are exact.  At most k
additions, a multiplication for each block of 128 by the change of unit and one
rounding of that factor, four fused multiply-adds for a block whose scale the codes
do not hold, the last unit, 16 parts and a residual: each is off by at most half a
step of a partial sum, which is within the sum of magnitudes.  (k + 6 kb + 20) *
2^-24 of that; and 2^-140 for sums in f32's subnormals."""
import numpy as np
import pytest

import fp8_model as fm
import fp8_shapes as fs
from test_gpu_fp8 import Weight, _gemm, _rows, _weight

pytestmark = pytest.mark.gpu

LEAST = [2.0 ** -149, 1.0, 1e-40, -3e-5, 2.0 ** -126, 2.0 ** -118, 2.0 ** -117, 0.7]
LARGEST = [2.0 ** 127, 1.0, 3e38, -1e30, 2.0 ** 118, 2.0 ** 117, 1.5 * 2.0 ** 120, 0.7]


def some(rows):
    """Rows that are compared: the first, the last, and those at tiles' borders."""
    at = {r + d for r in range(0, rows + 1, 128) for d in (-1, 0, 1)} | set(range(rows - 9, rows))
    return np.array(sorted(r for r in at if 0 <= r < rows))


def _scales(n, k, pattern):
    """The pattern along k, begun elsewhere in each block of outputs."""
    i, j = np.ogrid[:-(-n // 128), :-(-k // 128)]
    with np.errstate(over="ignore"):
        return np.array(pattern, np.float32)[(i + j) % len(pattern)]


def _compare(got, x, codes, scales, tell):
    at = some(x.shape[0])
    ref, mass = fm.product(x[at], codes, scales)
    k = x.shape[1]
    bound = (k + 6 * -(-k // 128) + 20) * 2.0 ** -24 * mass + 2.0 ** -140
    assert np.all(np.isfinite(got)), tell
    off = np.abs(got[at] - ref)
    assert np.all(off <= bound), (tell, float((off / bound).max()))


@pytest.mark.parametrize("shape", [*fs.TILES, *fs.FEW])
@pytest.mark.parametrize("pattern", [[1e28, *LEAST], [*LEAST, 1e28, 1e-30]])
def test_large_sums_beside_the_least_scales(ctx, shape, pattern):
    rows, n, k = shape
    codes, x = _weight(1, n, k).host[0], _rows(2, rows, k)
    scales = _scales(n, k, pattern)
    _compare(_gemm(ctx, Weight(codes, scales), x), x, codes, scales, shape)


@pytest.mark.parametrize("shape", [*fs.TILES, *fs.FEW])
@pytest.mark.parametrize("pattern,size", [(LEAST, 2.0 ** -40), (LARGEST, 2.0 ** 25)])
def test_terms_of_one_size(ctx, shape, pattern, size):
    """x beside each scale so that every block counts as much as the others."""
    rows, n, k = shape
    codes, x = _weight(3, n, k).host[0], _rows(4, rows, k)
    scales = np.repeat(_scales(128, k, pattern), -(-n // 128), 0)
    power = np.exp2(np.rint(np.log2(size / np.abs(scales[0].astype(np.float64)))))
    x *= np.repeat(power, 128)[:k].astype(np.float32)
    _compare(_gemm(ctx, Weight(codes, scales), x), x, codes, scales, shape)
