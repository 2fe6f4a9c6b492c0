"""Sequences that go back after their window has passed pages: with as many tokens
more in the remaps' window as they go back, every page that attention's window then
sees is still there.  The server, its bounds and its definitions are
tests/test_gpu_long_streams.py's."""
import pytest
import torch

import pages_model
import test_gpu_paged as paged
from test_gpu_long_streams import BATCH, PAGE, SINKS, WIDE, WINDOW, Server

pytestmark = pytest.mark.gpu


class Back(Server):
    def go_on(self, tokens, window):
        ctx, before, own = self.ctx, self.now(), list(range(BATCH))
        dt, copied = paged._ints(tokens), paged._ints([9] * BATCH)
        torch.cuda.synchronize()
        ctx.paged_remap_device(self.pool, 0, dt.data_ptr(), window=window, sinks=SINKS, copied=copied.data_ptr())
        ctx.synchronize()
        assert self.now() == pages_model.remap(*before, own, tokens, PAGE, window, SINKS)[:3]
        assert copied.tolist() == [-1] * BATCH
        self.held = [[(k[:n], v[:n]) for k, v in layers] for layers, n in zip(self.held, tokens)]
        self.lens = list(tokens)


@pytest.mark.parametrize("back", [16, 33, 48])
def test_back_by_as_many_tokens_as_the_window_is_wider(ctx, back):
    sv = Back(ctx)
    sv.step([90, 75, 0, 0, 0])
    for _ in range(50):
        sv.step([1, 1, 0, 0, 0])
        sv.go_on(sv.lens, WINDOW + back)
    assert sv.table[0].tolist()[2] == -1  # the window has passed some
    to = [max(-(-(n - back) // PAGE) * PAGE, 0) for n in sv.lens[:2]] + [0, 0, 0]
    assert all(0 < n - t <= back for n, t in zip(sv.lens, to[:2]))
    sv.go_on(to, WINDOW)
    assert all(row[j] >= 0 for row, t in zip(sv.table.tolist(), to[:2])
               for j in range(WIDE) if j * PAGE < t and ((j + 1) * PAGE > t - WINDOW + 1 or j * PAGE < SINKS))
    for n in (1, 3, 1, 20, 1):
        sv.step([n, 1, 0, 0, 0])
