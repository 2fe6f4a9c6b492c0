"""The scratch of products on 8-bit floats: a context takes it with the first product
that uses it, in a capture too, and no other."""
import pytest
import torch

import qtts
from test_gpu_fp8 import _check, _rows, _up, _weight

pytestmark = pytest.mark.gpu

MIB = 2 ** 20


def _taken(before):
    return (before - torch.cuda.mem_get_info()[0]) / MIB


def _free():
    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]


def _call(ctx, w, x, y):
    ctx.fp8_gemm_device(w.w, x.data_ptr(), x.shape[1], x.shape[0], y.data_ptr(), y.shape[1])


def test_taken_with_the_first_product_that_uses_it():
    # (90 rows of 512 would be brought over by the product's own blocks)
    w, few, x, large = _weight(1, 260, 2048), _up(_rows(2, 1, 2048)), _up(_rows(3, 90, 2048)), _up(_rows(3, 4000, 2048))
    y = torch.zeros((4000, 260), device="cuda")
    before = _free()
    ctx = qtts.Context(0)
    try:
        _call(ctx, w, few, y)  # brings its rows over itself
        ctx.synchronize()
        assert _taken(before) < 64  # 136 more when contexts were made with it
        before = _free()
        _call(ctx, w, x, y)
        ctx.synchronize()
        assert 128 <= _taken(before) < 160
        _check(y.cpu().numpy()[:90], x.cpu().numpy(), w)
        before = _free()
        _call(ctx, w, large, y)
        ctx.synchronize()
        assert _taken(before) < 2
        before = _free()
    finally:
        ctx.close()
    assert _taken(before) < -128


def test_first_product_in_a_capture():
    w, y = _weight(4, 260, 2048), torch.zeros((90, 260), device="cuda")
    inputs = [_rows(5 + i, 90, 2048) for i in range(3)]
    x = _up(inputs[0])
    ctx = qtts.Context(0)
    try:
        torch.cuda.synchronize()
        stream = torch.cuda.ExternalStream(ctx.stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            _call(ctx, w, x, y)
        for i in (0, 1, 2, 1):
            x.copy_(_up(inputs[i]))
            y.zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                g.replay()
            ctx.synchronize()
            _check(y.cpu().numpy(), inputs[i], w)
            got = y.clone()
            torch.cuda.synchronize()
            _call(ctx, w, x, y)
            ctx.synchronize()
            assert torch.equal(y, got)
        del g
    finally:
        ctx.close()


def test_a_full_card():
    """Refused where the scratch cannot be had, and nothing is left of it: products that
    do without go on, and the others when there is room."""
    w, few, rows = _weight(8, 260, 2048), _rows(9, 1, 2048), _rows(10, 90, 2048)
    x, y, hold = _up(rows), torch.zeros((90, 260), device="cuda"), []
    one = _up(few)
    ctx = qtts.Context(0)
    try:
        _call(ctx, w, one, y)
        ctx.synchronize()
        for _ in range(4):
            room = _free() - 100 * MIB
            if room > 30 * MIB:
                hold.append(torch.empty(room, dtype=torch.uint8, device="cuda"))
        assert _free() < 136 * MIB
        with pytest.raises(qtts.QttsError) as e:
            _call(ctx, w, x, y)
        assert e.value.status == qtts.QTTS_ENOMEM
        _call(ctx, w, one, y)
        ctx.synchronize()
        hold.clear()
        torch.cuda.empty_cache()
        _check(y.cpu().numpy()[:1], few, w)
        _call(ctx, w, x, y)
        ctx.synchronize()
        _check(y.cpu().numpy(), rows, w)
    finally:
        hold.clear()
        torch.cuda.empty_cache()
        ctx.close()
