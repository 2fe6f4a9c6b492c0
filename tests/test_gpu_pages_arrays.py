"""What a reservation lacks in the place of its starts or ends, and a packing whose
arrays are the pool's, which is refused before anything is written."""
import numpy as np
import pytest
import torch

import pages_model as model
import qtts
from test_gpu_pages import SHAPES, Pool, _ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("place", ["starts", "ends"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_lacking_in_place(ctx, shape, place):
    p = Pool(sum(shape) + 1, *shape)
    r = np.random.default_rng(3)
    batch, most = p.pool.batch, p.pool.max_pages * p.page
    starts = r.integers(0, most + 1, batch)
    ends = np.minimum(starts + np.where(r.random(batch) < 0.7, 1, r.integers(0, most + 1, batch)), most)
    starts[r.random(batch) < 0.03] = -1
    before = p.now()
    at = {"starts": _ints(starts), "ends": _ints(ends)}
    torch.cuda.synchronize()
    ctx.paged_reserve_device(p.pool, at["starts"].data_ptr(), at["ends"].data_ptr(), at[place].data_ptr())
    ctx.synchronize()
    table, refs, lacking = model.reserve(*before[:2], starts.tolist(), ends.tolist(), p.page)
    assert list(p.now()) == [table, refs, before[2]] and at[place].tolist() == lacking


def test_the_pools_own_arrays_are_refused(ctx):
    p = Pool(1, 5, 7, 60, 64)
    before = p.now()
    a, b = (torch.zeros(64, device="cuda").int().data_ptr() for _ in range(2))
    tokens = _ints([0] * 5).data_ptr()
    for own in (p.pool.refs, p.pool.page_table, p.pool.slots):
        for call in (lambda: ctx.paged_compact_device(p.pool, own, b), lambda: ctx.paged_compact_device(p.pool, a, own),
                     lambda: ctx.paged_compact_device(p.pool, a, b, own),
                     lambda: ctx.paged_reserve_device(p.pool, tokens, tokens, own),
                     lambda: ctx.paged_remap_device(p.pool, 0, tokens, copied=own)):
            with pytest.raises(qtts.QttsError):
                call()
    with pytest.raises(qtts.QttsError):
        ctx.paged_compact_device(p.pool, a, b, a)
    ctx.synchronize()
    assert p.now() == before
