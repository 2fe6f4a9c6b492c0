"""Attention with sinks where sinks and window hide nothing: the other kernel's tokens,
numbered alike and divided alike, and so the other kernel's bits."""
import pytest
import torch

import test_gpu_paged as paged
from test_gpu_paged_sinks import _attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sinks,window", [(1, 2 ** 31 - 1), (2 ** 31 - 1, 1), (2000, 4000)])
@pytest.mark.parametrize("kvh,group,hd,counts", [(2, 2, 128, [1, 1, 1]), (2, 2, 64, [1, 70, 5]), (1, 6, 128, [3, 2, 1]),
                                                 (8, 2, 64, [100, 99, 100])])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_nothing_hidden(ctx, page, kvh, group, hd, counts, sinks, window):
    starts, heads = [700, 40, 1900], kvh * group
    c, _ = paged._filled(ctx, kvh, hd, page, starts, counts, seed=2)
    q, s = paged._up(paged._normal(3, sum(counts), heads * hd)), c.seqs(starts, counts)
    plain = _attend(ctx, c, s, q, heads, 0, 0)
    assert torch.equal(_attend(ctx, c, s, q, heads, window, sinks), plain)
