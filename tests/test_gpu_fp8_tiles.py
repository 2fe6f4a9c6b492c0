"""Products on 8-bit floats at their edges on every kind of tile, whole, divided and
partly divided, and on every kernel without them (tests/fp8_shapes.py, whose kernels
tests/test_fp8_shapes.py holds against the plan).

Tolerance: (k + 6 kb + 20) * 2^-24 of the sum of magnitudes, as derived in
tests/test_gpu_fp8_scales.py; here no scale is near f32's ends."""
import numpy as np
import pytest
import torch

import fp8_model as fm
import fp8_shapes as fs
from test_gpu_fp8 import Weight, _gemm, _rows, _up, _weight
from test_gpu_fp8_scales import some

pytestmark = pytest.mark.gpu

SHAPES = [*fs.TILES, *fs.FEW]


def _compare(got, x, codes, scales, add=None):
    """Some rows, all of them finite."""
    at = some(x.shape[0])
    at = at[np.isfinite(x[at]).all(1)]
    ref, mass = fm.product(x[at], codes, scales, None if add is None else add[at])
    k = x.shape[1]
    bound = (k + 6 * -(-k // 128) + 20) * 2.0 ** -24 * mass
    off = np.abs(got[at] - ref)
    assert np.all(off <= bound), float((off / bound).max())


def _in_place(ctx, w, x, add):
    rows, k = x.shape
    n, ld = w.w.n, -(-w.w.n // 4) * 4
    dx, y = _up(x), torch.zeros((rows + 1, ld), device="cuda")
    y[:rows, :n] = _up(add)
    torch.cuda.synchronize()
    ctx.fp8_gemm_device(w.w, dx.data_ptr(), k, rows, y.data_ptr(), ld, add=y.data_ptr(), ld_add=ld)
    ctx.synchronize()
    y = y.cpu().numpy()
    assert not y[rows:].any() and not y[:, n:].any()
    return y[:rows, :n]


@pytest.mark.parametrize("shape", SHAPES)
def test_residual(ctx, shape):
    rows, n, k = shape
    w, x, add = _weight(1, n, k), _rows(2, rows, k), 50 * _rows(3, rows, n)
    got = _in_place(ctx, w, x, add)
    _compare(got, x, *w.host, add)
    assert np.array_equal(got, _gemm(ctx, w, x, add=add))


@pytest.mark.parametrize("shape", SHAPES)
def test_rows_that_are_not_finite(ctx, shape):
    """In the first row and the last, in the first block of k and the last."""
    rows, n, k = shape
    w, x, add = _weight(4, n, k), _rows(5, rows, k), _rows(6, rows, n)
    ends = {0: (0, np.nan), rows // 2: (k // 2, np.inf), rows - 1: (k - 1, -np.inf)}
    for row, (at, value) in ends.items():
        x[row, at] = value
    for got in (_gemm(ctx, w, x), _in_place(ctx, w, x, add)):
        bad = np.zeros(rows, bool)
        bad[list(ends)] = True
        assert np.all(np.isnan(got[bad])) and np.all(np.isfinite(got[~bad]))
    _compare(got, x, *w.host, add)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("block", ["first", "middle", "last"])
def test_weights_that_are_not_finite(ctx, shape, block):
    """A code makes its column NaN, a scale those of its block; whichever part of a
    divided tile it lies in."""
    rows, n, k = shape
    kb = -(-k // 128)
    b = {"first": 0, "middle": kb // 2, "last": kb - 1}[block]
    codes, scales = (a.copy() for a in _weight(7, n, k).host)
    x, add = _rows(8, rows, k), _rows(9, rows, n)
    codes[n - 1, min(128 * b + 3, k - 1)] = 0x7f
    codes[3, 128 * b] = 0xff
    bad = np.zeros(n, bool)
    bad[[3, n - 1]] = True
    for nb, value in ((1, np.nan), ((n - 1) // 128 - 1, np.inf)):
        if 0 < nb < n // 128:
            scales[nb, b] = value
            bad[128 * nb:128 * (nb + 1)] = True
    got = _gemm(ctx, Weight(codes, scales), x, add=add)
    assert np.all(np.isnan(got[:, bad])) and np.all(np.isfinite(got[:, ~bad]))
    codes[3, 128 * b] = codes[n - 1, min(128 * b + 3, k - 1)] = 0
    scales[~np.isfinite(scales)] = 0
    at = some(rows)
    ref, mass = fm.product(x[at], codes, scales, add[at])
    bound = (k + 6 * kb + 20) * 2.0 ** -24 * mass
    assert np.all((np.abs(got[at] - ref) <= bound)[:, ~bad])


@pytest.mark.parametrize("shape", SHAPES)
def test_scales_of_zero_and_below(ctx, shape):
    """Codes under 0 are zeros, NaN among them; a column of nothing else is what is
    added."""
    rows, n, k = shape
    codes, scales = (a.copy() for a in _weight(10, n, k).host)
    x, add = _rows(11, rows, k), _rows(12, rows, n)
    i, j = np.ogrid[:scales.shape[0], :scales.shape[1]]
    scales[(i + j) % 3 == 0] = 0
    scales[(i + 2 * j) % 5 == 1] *= -1
    if scales.shape[0] > 1:
        scales[1] = 0
    zero = np.repeat(np.repeat(scales == 0, 128, 0)[:n], 128, 1)[:, :k]
    clean = codes.copy()
    clean[zero] = 0
    codes[zero] = np.where(np.random.default_rng(13).random(codes.shape) < 0.1, 0x7f, codes)[zero]
    got = _gemm(ctx, Weight(codes, scales), x, add=add)
    _compare(got, x, clean, scales, add)
    if scales.shape[0] > 1:
        assert np.array_equal(got[:, 128:256], add[:, 128:256])


@pytest.mark.parametrize("shape", fs.TILES)
def test_graph(ctx, shape):
    """Captured and replayed on other rows and other scales, between calls of another
    size that use the same scratch."""
    rows, n, k = shape
    w, other = _weight(14, n, k), _weight(15, 1300, 1040)
    rng = np.random.default_rng(16)
    inputs = [(_rows(17 + i, rows, k), (w.host[1] * (0.5 + rng.random(w.host[1].shape))).astype(np.float32))
              for i in range(3)]
    x, y = _up(inputs[0][0]), torch.zeros((rows, -(-n // 4) * 4), device="cuda")
    ox, oy = _up(_rows(20, 300, 1040)), torch.zeros((300, 1300), device="cuda")
    stream = torch.cuda.ExternalStream(ctx.stream)

    def call():
        ctx.fp8_gemm_device(w.w, x.data_ptr(), k, rows, y.data_ptr(), y.stride(0))

    def set_to(i):
        x.copy_(_up(inputs[i][0]))
        w.scales.copy_(_up(inputs[i][1]))

    alone = []
    for i in range(3):
        set_to(i)
        torch.cuda.synchronize()
        call()
        ctx.synchronize()
        alone.append(y.clone())
        _compare(y.cpu().numpy()[:, :n], inputs[i][0], w.host[0], inputs[i][1])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        call()
    for i in (1, 2, 0, 2):
        set_to(i)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            ctx.fp8_gemm_device(other.w, ox.data_ptr(), 1040, 300, oy.data_ptr(), 1300)
            g.replay()
            ctx.fp8_gemm_device(other.w, ox.data_ptr(), 1040, 300, oy.data_ptr(), 1300)
        torch.cuda.synchronize()
        assert torch.equal(y, alone[i])
