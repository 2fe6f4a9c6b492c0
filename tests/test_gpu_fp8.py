"""Products on weights in 8-bit floats (qtts_fp8_gemm_device) and the weights'
quantizer, against their restatement in 64 bits (tests/fp8_model.py).

Tolerances.  Codes and scales are equal.  A product of two codes is exact in
f32 and so are the rows' powers of two; a weight's scale takes one rounding with
its block's sum (a fused multiply-add).  A sum of 128 products, one of the
blocks and joining at most 64 parts are f32 additions, each off by at most half
a step of a partial sum, which is within the sum of magnitudes: (128 + blocks +
64 + 2) * 2^-24 of that."""
import numpy as np
import pytest
import torch

import fp8_model as fm
import qtts

pytestmark = pytest.mark.gpu


def _up(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _padded(rows, width, ld, fill, dtype=torch.float32):
    return torch.full((rows, ld), fill, dtype=dtype, device="cuda")


class Weight:
    def __init__(self, codes, scales, ld=None):
        n, k = codes.shape
        self.ld = k if ld is None else ld
        # what lies behind a row's end is NaN
        self.codes = torch.full((n, self.ld), 127, dtype=torch.uint8, device="cuda")
        self.codes[:, :k] = _up(codes)
        self.scales = _up(scales)
        self.host = (codes, scales)
        self.w = qtts.Fp8Weight(self.codes.data_ptr(), self.scales.data_ptr(), n, k, self.ld)


def _weight(seed, n, k, ld=None):
    r = np.random.default_rng(seed)
    codes = r.integers(0, 256, (n, k)).astype(np.uint8)
    codes[codes & 127 == 127] = 0x3a
    scales = (np.exp(r.standard_normal((-(-n // 128), -(-k // 128)))) * 0.01).astype(np.float32)
    return Weight(codes, scales, ld)


def _rows(seed, rows, k):
    r = np.random.default_rng(seed)
    return (r.standard_normal((rows, k)) * np.exp(r.standard_normal(k))).astype(np.float32)


def _gemm(ctx, w, x, add=None, ld_y=None, ld_x=None):
    """y with what lies behind its rows and their ends checked to be as it was."""
    rows, k = x.shape
    n = w.w.n
    ld_x, ld_y = ld_x or -(-k // 4) * 4, ld_y or -(-n // 4) * 4
    dx = _padded(rows + 1, k, ld_x, float("nan"))
    dx[:rows, :k] = _up(x)
    y = _padded(rows + 2, n, ld_y, 7.0)
    more = {}
    if add is not None:
        da = _padded(rows, n, ld_y + 8, float("nan"))
        da[:, :n] = _up(add)
        more = dict(add=da.data_ptr(), ld_add=ld_y + 8)
    torch.cuda.synchronize()
    ctx.fp8_gemm_device(w.w, dx.data_ptr(), ld_x, rows, y.data_ptr(), ld_y, **more)
    ctx.synchronize()
    y = y.cpu().numpy()
    assert np.all(y[rows:] == 7.0) and np.all(y[:, n:] == 7.0)
    return y[:rows, :n]


def _check(got, x, w, add=None, tell=""):
    ref, mass = fm.product(x, *w.host, add)
    kb = -(-x.shape[1] // 128)
    bound = (128 + kb + 66) * 2.0 ** -24 * mass + 2.0 ** -149
    off = np.abs(got - ref)
    assert np.all(off <= bound), (tell, float((off / bound).max()))


@pytest.mark.parametrize("k", [16, 48, 112, 128, 144, 256, 400, 1040])
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 64, 129])
def test_sizes(ctx, rows, k):
    """Odd outputs, blocks cut short on either side."""
    for n in (1, 31, 128, 197, 300):
        w = _weight(n + k, n, k, ld=-(-k // 16) * 16 + 32)
        x = _rows(rows + k, rows, k)
        _check(_gemm(ctx, w, x, ld_x=k + 4, ld_y=-(-n // 4) * 4 + 4), x, w, tell=(rows, n, k))


@pytest.mark.parametrize("rows,n,k", [(1, 4096, 2048), (3, 2048, 6144), (16, 2048, 6144), (40, 1000, 6144),
                                      (200, 640, 2048), (515, 1100, 512), (700, 300, 8192)])
def test_large(ctx, rows, n, k):
    w, x, add = _weight(1, n, k), _rows(2, rows, k), _rows(3, rows, n)
    _check(_gemm(ctx, w, x), x, w)
    _check(_gemm(ctx, w, x, add=add), x, w, add)


@pytest.mark.parametrize("rows", [2, 5, 9, 16, 17, 31, 32, 33, 49, 64, 65])
@pytest.mark.parametrize("n,k", [(4090, 1552), (30, 8208), (9001, 272), (300, 16), (260, 3184)])
def test_few_rows(ctx, rows, n, k):
    """The kernel for them and tiles of 64, on either side of where one gives way to
    the other."""
    w, x, add = _weight(1, n, k), _rows(2, rows, k), _rows(3, rows, n)
    _check(_gemm(ctx, w, x, add=add), x, w, add)


@pytest.mark.parametrize("rows,n,k", [(258, 5737, 16), (321, 5471, 16), (2694, 4369, 16), (400, 6001, 144),
                                      (300, 5737, 272), (2694, 4369, 272), (69, 5737, 1040), (321, 5452, 784),
                                      (72, 5733, 2064), (69, 3267, 4112), (20, 4103, 6160), (132, 5452, 4112)])
def test_tiles(ctx, rows, n, k):
    """Tiles of 64, 128 and 256, whole and divided, cut short on every side."""
    w = _weight(n + k, n, k, ld=-(-k // 16) * 16 + 32)
    x, add = _rows(rows + k, rows, k), _rows(3, rows, n)
    _check(_gemm(ctx, w, x, add=add, ld_x=k + 4, ld_y=-(-n // 4) * 4 + 4), x, w, add)


@pytest.mark.parametrize("rows,n,k", [(646, 5378, 1040), (1051, 2047, 6144), (3337, 4740, 528)])
def test_the_last_round_divided(ctx, rows, n, k):
    """Tiles of 128, 64 and 256 of which 256 or 512 have a block each and the others
    several, and the join of these."""
    w, x, add = _weight(1, n, k), _rows(2, rows, k), _rows(3, rows, n)
    _check(_gemm(ctx, w, x, add=add), x, w, add)


@pytest.mark.parametrize("rows,n", [(5, 260), (40, 260), (130, 260), (300, 5500)])
def test_residual_in_place(ctx, rows, n):
    w, x, add = _weight(4, n, 384), _rows(5, rows, 384), _rows(6, rows, n)
    dx, y = _up(x), _up(add)
    torch.cuda.synchronize()
    ctx.fp8_gemm_device(w.w, dx.data_ptr(), 384, rows, y.data_ptr(), n, add=y.data_ptr(), ld_add=n)
    ctx.synchronize()
    _check(y.cpu().numpy(), x, w, add)


def _edges():
    """Rows of 128 values with every code's value, every border between two and
    their neighbours, at several powers of two; zeros; the ends of f32."""
    v = np.sort(fm.VALUES[~np.isnan(fm.VALUES)])
    mid = (v[1:] + v[:-1]) / 2
    near = [np.nextafter(mid.astype(np.float32), np.float32(s * np.inf)) for s in (1, -1)]
    pool = np.concatenate([v, mid, *near]).astype(np.float32)
    pool = np.concatenate([pool, np.zeros(-pool.size % 127, np.float32)]).reshape(-1, 127)
    rows = [np.concatenate([p, [np.float32(448)]]) * np.float32(2.0 ** s)
            for p in pool for s in (0, -3, 60, 118, -100, -117, -120, -126)]
    for top in (448.0, np.nextafter(np.float32(448), np.float32(1e9)), 3.4028235e38, 1.1754944e-38, 1e-45, 0.0):
        rows.append(np.linspace(-1, 1, 128).astype(np.float32) * np.float32(top))
    return np.stack(rows).astype(np.float32)


@pytest.mark.parametrize("each", [7, 64, 200])
def test_rows_are_rounded_exactly(ctx, each):
    """Through a weight of ones on the diagonal a row comes back as its codes'
    values."""
    w = Weight(np.where(np.eye(128, dtype=bool), 0x38, 0).astype(np.uint8), np.ones((1, 1), np.float32))
    x = _edges()
    for at in range(0, x.shape[0], each):
        part = x[at:at + each]
        assert np.array_equal(_gemm(ctx, w, part), fm.blocks(part).astype(np.float32)), at


@pytest.mark.parametrize("n,k", [(128, 128), (1, 16), (130, 272), (300, 1008)])
def test_weights_are_rounded_exactly(ctx, n, k):
    r = np.random.default_rng(n)
    src = (r.standard_normal((n, k)) * np.exp(3 * r.standard_normal((n, 1)))).astype(np.float32)
    edges = _edges().reshape(-1)
    m = min(edges.size, src.size // 2)
    src.reshape(-1)[:m] = edges[:m]
    src[-1, -16:] = [0.0, -0.0] * 8
    dsrc = _padded(n, k, k + 4, float("nan"))
    dsrc[:, :k] = _up(src)
    codes = torch.full((n + 1, k + 16), 99, dtype=torch.uint8, device="cuda")
    scales = torch.full((-(-n // 128) * -(-k // 128) + 1,), 5.0, device="cuda")
    torch.cuda.synchronize()
    ctx.fp8_quantize_device(dsrc.data_ptr(), k + 4, qtts.Fp8Weight(codes.data_ptr(), scales.data_ptr(), n, k, k + 16))
    ctx.synchronize()
    ref, s = fm.quantized(src)
    codes, scales = codes.cpu().numpy(), scales.cpu().numpy()
    assert np.array_equal(scales[:-1].reshape(s.shape), s) and scales[-1] == 5.0
    assert np.array_equal(codes[:n, :k], ref)
    assert np.all(codes[n:] == 99) and np.all(codes[:, k:] == 99)


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("rows,n", [(3, 300), (30, 300), (90, 300), (300, 5737)])
def test_not_finite(ctx, rows, n, bad):
    """A row with an Inf or NaN is NaN, the others are not; a weight's code or
    scale makes its outputs NaN; a block of a weight that is not finite has
    scale NaN."""
    k = 272
    w, x = _weight(8, n, k), _rows(9, rows, k)
    x[1, 260] = bad
    got = _gemm(ctx, w, x)
    assert np.all(np.isnan(got[1]))
    rest = [i for i in range(rows) if i != 1]
    _check(got[rest], x[rest], w)
    codes, scales = (a.copy() for a in w.host)
    codes[17, 271], scales[1, 0] = 0xff, bad
    x = np.abs(_rows(9, rows, k)) + 1
    got = _gemm(ctx, Weight(codes, scales), x)
    assert np.all(np.isnan(got[:, 17])) and not np.any(np.isfinite(got[:, 128:256]))
    some = np.r_[0:17, 18:128, 256:n]
    ref, mass = fm.product(x, w.host[0], w.host[1])
    assert np.all(np.abs(got[:, some] - ref[:, some]) <= 200 * 2.0 ** -24 * mass[:, some])
    src = _rows(10, n, k)
    src[130, 200] = bad
    dsrc, dc, ds = _up(src), torch.zeros((n, k), dtype=torch.uint8, device="cuda"), torch.zeros((-(-n // 128), 3), device="cuda")
    torch.cuda.synchronize()
    ctx.fp8_quantize_device(dsrc.data_ptr(), k, qtts.Fp8Weight(dc.data_ptr(), ds.data_ptr(), n, k, k))
    ctx.synchronize()
    codes, scales = fm.quantized(src)
    assert np.isnan(scales[1, 1]) and np.array_equal(ds.cpu().numpy(), scales, equal_nan=True)
    assert np.array_equal(dc.cpu().numpy(), codes)


@pytest.mark.parametrize("rows,times", [(2, 1), (10, 1), (40, 1), (300, 1), (128, 11), (330, 11)])
def test_scales_of_any_size(ctx, rows, times):
    """Scales of 0 (whose codes count as 0, NaN among them), negative ones, the least
    and the largest, in any order along k and beside each other along n; x so that
    the results stay f32's."""
    n, k = 512 * times - 112, 1168
    codes = _weight(40, n, k).host[0].copy()
    scales = np.tile(np.array([[0.01, 0.0, -0.02, 0.0, 0.03, -0.5, 1e-3, 0.0, 0.0, 0.7],
                       [0.0] * 10,
                       [1e-40, 3e38, 1e-30, 2.0 ** -149, 1e20, 0.0, 1.0, -3e38, 1e-38, 2e30],
                       [2.0 ** -126, 2.0 ** -118, 2.0 ** -117, 2.0 ** 117, 2.0 ** 118, 2.0 ** 127, 1.5, 1.0, 0.75, 3.0]],
                      np.float32), (times, 1))
    each = 512 * np.arange(times)[:, None]
    columns = lambda a, b: np.sort((each + np.arange(a, b)).reshape(-1))  # of every turn of the scales
    x = _rows(41, rows, k)
    for b in range(10):  # the third and fourth row's products of one size
        x[:, b * 128:(b + 1) * 128] *= np.float32(0.2)
    codes[5, 130], codes[150, 7], codes[395, 300] = 0x7f, 0xff, 0x11
    x2 = x.copy()
    w = Weight(codes, scales)
    got = _gemm(ctx, w, x2)
    assert not np.any(got[:, columns(128, 256)])
    clean = codes.copy()
    clean[5, 130] = clean[150, 7] = 0
    ref, mass = fm.product(x2, clean, scales)
    fine = columns(0, 256)
    off, bound = np.abs(got - ref), (128 + 10 + 66) * 2.0 ** -24 * mass + 2.0 ** -140
    assert np.all(off[:, fine] <= bound[:, fine])
    # sums of up to 3e38 * 448 * 448: f32's where the definition's are, to the same bound
    for cols in (columns(256, 384), columns(384, 400)):
        for b in range(10):
            alone = np.zeros_like(scales)
            alone[:, b] = scales[:, b]
            tiny = (x2 * np.float32(2.0 ** -20)).astype(np.float32)
            got = _gemm(ctx, Weight(clean, alone), tiny)
            ref, mass = fm.product(tiny, clean, alone)
            inside = mass[:, cols] < 1e37
            # a scale below 2^-117 leaves a sum in f32's subnormals
            off = np.abs(got[:, cols] - ref[:, cols])
            assert np.all((off <= 204 * 2.0 ** -24 * mass[:, cols] + 2.0 ** -140)[inside]), b


@pytest.mark.parametrize("rows,n", [(1, 20), (9, 20), (60, 300), (258, 5737), (400, 6001)])
@pytest.mark.parametrize("k", [144, 208])
def test_nan_codes_under_a_scale_of_zero(ctx, rows, n, k):
    """They count as 0 wherever they lie, also where a later block is cut short."""
    codes = _weight(80, n, k).host[0].copy()
    scales = np.full((-(-n // 128), 2), 0.5, np.float32)
    scales[0, 0] = 0
    codes[:16, :128:3] = 0x7f
    x = _rows(81, rows, k)
    clean = codes.copy()
    clean[:16, :128] = 0
    got, (ref, mass) = _gemm(ctx, Weight(codes, scales), x), fm.product(x, clean, scales)
    assert np.all(np.abs(got - ref) <= (128 + 2 + 66) * 2.0 ** -24 * mass + 2.0 ** -149)


@pytest.mark.parametrize("rows,n,k", [(4, 100, 8192), (1, 70, 32768), (3, 40, 11008), (4, 33, 8208), (16, 20, 20000)])
def test_long_rows(ctx, rows, n, k):
    """As much of x in LDS as a few rows may have there, and one block more."""
    w, x = _weight(50, n, k), _rows(51, rows, k)
    _check(_gemm(ctx, w, x), x, w)


def test_more_rows_than_the_scratch_holds(ctx):
    rows, k, n = 524288 + 300, 16, 7
    w = _weight(52, n, k)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((rows, k), generator=g, device="cuda")
    y = torch.full((rows + 1, 8), 7.0, device="cuda")
    torch.cuda.synchronize()
    ctx.fp8_gemm_device(w.w, x.data_ptr(), k, rows, y.data_ptr(), 8)
    ctx.synchronize()
    assert bool(torch.all(y[rows:] == 7)) and bool(torch.all(y[:, 7] == 7))
    some = np.r_[0:20, 524270:524310, rows - 20:rows]
    _check(y.cpu().numpy()[some, :7], x.cpu().numpy()[some], w)


def test_two_contexts_at_once(ctx):
    other = qtts.Context(0)
    try:
        jobs = []
        for c, seed in ((ctx, 60), (other, 70)):
            for rows, n, k in ((40, 640, 2048), (7, 500, 512), (300, 260, 1024), (20, 4103, 6160), (70, 5737, 1040)):
                w, x = _weight(seed, n, k), _up(_rows(seed + 1, rows, k))
                y = torch.zeros((rows, -(-n // 4) * 4), device="cuda")
                jobs.append((c, w, x, rows, k, n, y))
        torch.cuda.synchronize()

        def go():
            for c, w, x, rows, k, n, y in jobs:
                c.fp8_gemm_device(w.w, x.data_ptr(), k, rows, y.data_ptr(), y.stride(0))
        go()
        torch.cuda.synchronize()
        alone = []
        for c, w, x, rows, k, n, y in jobs:
            c.fp8_gemm_device(w.w, x.data_ptr(), k, rows, y.data_ptr(), y.stride(0))
            c.synchronize()
            alone.append(y.clone())
        torch.cuda.synchronize()
        for _ in range(20):
            go()
        torch.cuda.synchronize()
        assert all(torch.equal(job[-1], a) for job, a in zip(jobs, alone))
    finally:
        other.close()


def test_no_rows(ctx):
    w = _weight(1, 32, 64)
    ctx.fp8_gemm_device(w.w, 0, 64, 0, 0, 32)


@pytest.mark.parametrize("rows,n,k", [(40, 640, 2048), (290, 640, 2048), (20, 4104, 6160)])
def test_graph_and_own_stream(ctx, rows, n, k):
    """Captured and replayed on other values, between plain calls that use the
    scratch for other sizes."""
    w, big = _weight(11, n, k), _weight(12, 200, 1024)
    xs = [_rows(20 + i, rows, k) for i in range(3)]
    x, y = _up(xs[0]), torch.zeros((rows, n), device="cuda")
    bx, by = _up(_rows(30, 300, 1024)), torch.zeros((300, 200), device="cuda")
    stream = torch.cuda.ExternalStream(ctx.stream)
    call = lambda: ctx.fp8_gemm_device(w.w, x.data_ptr(), k, rows, y.data_ptr(), n)
    torch.cuda.synchronize()
    alone = []
    for a in xs:
        x.copy_(_up(a))
        torch.cuda.synchronize()
        call()
        ctx.synchronize()
        alone.append(y.clone())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        call()
    for i in (1, 2, 0, 2):
        with torch.cuda.stream(stream):
            x.copy_(_up(xs[i]))
            ctx.fp8_gemm_device(big.w, bx.data_ptr(), 1024, 300, by.data_ptr(), 200)
            g.replay()
            ctx.fp8_gemm_device(big.w, bx.data_ptr(), 1024, 300, by.data_ptr(), 200)
        torch.cuda.synchronize()
        assert torch.equal(y, alone[i])
