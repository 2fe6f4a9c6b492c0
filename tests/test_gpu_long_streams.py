"""A server of long streams as it strings the operators together: two decoder
layers on 8-bit weights over one pool of pages, sequences that join, go on, fork,
go back, end and drop what their window has passed, a pool that is packed.  Each
operator is held against its definition in 64 bits on the values that it was given,
with its own tests' bounds; tables, references and slots against lists."""
import numpy as np
import pytest
import torch

import fp8_model as fm
import paged_model as pm
import pages_model
import qtts
import test_gpu_fp8 as fp8
import test_gpu_paged as paged
import test_gpu_paged_sinks as sinks_test

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KVH, HD, PAGE, LAYERS = 256, 4, 2, 64, 16, 2
QKV, WINDOW, SINKS = (HEADS + 2 * KVH) * HD, 40, 20
BATCH, WIDE, PAGES, SLOTS = 5, 12, 34, 7


def _weight(seed, n, k):
    w = (np.random.default_rng(seed).standard_normal((n, k)) * k ** -0.5).astype(np.float32)
    return fp8.Weight(*fm.quantized(w))


class Server:
    def __init__(self, ctx):
        self.ctx, self.stream = ctx, torch.cuda.ExternalStream(ctx.stream)
        self.rng = np.random.default_rng(3)
        self.layers = [dict(qkv=_weight(10 + i, QKV, HIDDEN), o=_weight(20 + i, HIDDEN, HEADS * HD),
                            cache=paged.Cache(KVH, HD, PAGE, SLOTS, 1, spare=PAGES - SLOTS)) for i in range(LAYERS)]
        self.table, self.refs = (torch.full(s, v, dtype=torch.int32, device="cuda")
                                 for s, v in (((BATCH, WIDE), -1), ((PAGES,), 0)))
        self.slots = paged._ints([6, 0, 3, 1, 5])
        self.pool = qtts.PagedPool(self.refs.data_ptr(), self.table.data_ptr(), self.slots.data_ptr(), PAGES, PAGE,
                                   BATCH, WIDE)
        self.cos, self.sin = paged._rope(HD)
        self.d_cos, self.d_sin = paged._up(self.cos), paged._up(self.sin)
        empty = np.zeros((0, KVH, HD), np.float32)
        # what each sequence of each layer holds
        self.held = [[(empty, empty) for _ in range(LAYERS)] for _ in range(BATCH)]
        self.lens = [0] * BATCH

    def now(self):
        return self.table.tolist(), self.refs.tolist(), self.slots.tolist()

    def turn(self, source, tokens, pack=False):
        """Between two steps: rows become others, layers copy open rows, the pool
        is packed."""
        ctx, before = self.ctx, self.now()
        ds, dt, copied = paged._ints(source), paged._ints(tokens), paged._ints([9] * BATCH)
        moves, live = paged._ints([[9] * (PAGES // 2)] * 2), paged._ints([9])
        torch.cuda.synchronize()
        ctx.paged_remap_device(self.pool, ds.data_ptr(), dt.data_ptr(), window=WINDOW, sinks=SINKS,
                               copied=copied.data_ptr())
        if pack:
            ctx.paged_compact_device(self.pool, moves[0].data_ptr(), moves[1].data_ptr(), live.data_ptr())
        for layer in self.layers:
            kv = layer["cache"].kv
            ctx.paged_copy_open_device(kv, BATCH, copied.data_ptr(), self.slots.data_ptr(), dt.data_ptr())
            if pack:
                ctx.paged_copy_pages_device(kv, kv, PAGES // 2, moves[0].data_ptr(), moves[1].data_ptr())
        ctx.synchronize()
        table, refs, slots, ref_copied = pages_model.remap(*before, source, tokens, PAGE, WINDOW, SINKS)
        assert copied.tolist() == ref_copied
        if pack:
            table, refs, frm, to, n = pages_model.compact(table, refs)
            assert moves.tolist() == [frm, to] and live.tolist() == [n]
        assert self.now() == (table, refs, slots)
        self.held = [[(k[:n], v[:n]) for k, v in self.held[s]] if s >= 0 else [(np.zeros((0, KVH, HD), np.float32),) * 2]
                     * LAYERS for s, n in zip(source, tokens)]
        self.lens = list(tokens)

    def step(self, counts):
        """Each row's next tokens through both layers."""
        ctx, rows, before = self.ctx, sum(counts), self.now()
        ends = [a + n for a, n in zip(self.lens, counts)]
        starts, d_ends, lacking = paged._ints(self.lens), paged._ints(ends), paged._ints([9] * BATCH)
        offsets = paged._ints(np.concatenate([[0], np.cumsum(counts)]))
        x = paged._up(self.rng.standard_normal((rows, HIDDEN)).astype(np.float32))
        seqs = qtts.PagedSeqs(BATCH, WIDE, rows, max(counts), self.table.data_ptr(), self.slots.data_ptr(),
                              starts.data_ptr(), offsets.data_ptr(), paged.ROPE_ROWS)
        torch.cuda.synchronize()
        ctx.paged_reserve_device(self.pool, starts.data_ptr(), d_ends.data_ptr(), lacking.data_ptr())
        kept = []
        with torch.cuda.stream(self.stream):
            for layer in self.layers:
                qkv = torch.empty((rows, QKV), device="cuda")
                q, out = (torch.empty((rows, HEADS * HD), device="cuda") for _ in range(2))
                y = torch.empty((rows, HIDDEN), device="cuda")
                at = qkv.data_ptr()
                ctx.fp8_gemm_device(layer["qkv"].w, x.data_ptr(), HIDDEN, rows, at, QKV)
                ctx.paged_append_device(layer["cache"].kv, seqs, at + 4 * HEADS * HD, QKV, at + 4 * (HEADS + KVH) * HD,
                                        QKV, heads=HEADS, q=at, ld_q=QKV, q_out=q.data_ptr(), ld_q_out=HEADS * HD,
                                        rope_cos=self.d_cos.data_ptr(), rope_sin=self.d_sin.data_ptr(),
                                        rope_rows=paged.ROPE_ROWS)
                ctx.paged_attention_device(layer["cache"].kv, seqs, HEADS, q.data_ptr(), HEADS * HD, out.data_ptr(),
                                           HEADS * HD, scale=HD ** -0.5, window=WINDOW, sinks=SINKS)
                ctx.fp8_gemm_device(layer["o"].w, out.data_ptr(), HEADS * HD, rows, y.data_ptr(), HIDDEN,
                                    add=x.data_ptr(), ld_add=HIDDEN)
                kept.append((x, qkv, q, out, y))
                x = y
        ctx.synchronize()
        table, refs, ref_lacking = pages_model.reserve(*before[:2], self.lens, ends, PAGE)
        assert self.now() == (table, refs, before[2]) and lacking.tolist() == ref_lacking == [0] * BATCH
        for l, (layer, tensors) in enumerate(zip(self.layers, kept)):
            x, qkv, q, out, y = (t.cpu().numpy() for t in tensors)
            fp8._check(qkv, x, layer["qkv"])
            fp8._check(y, out, layer["o"], add=x)
            parts, at = qkv.reshape(rows, -1, HD), 0
            for b, n in enumerate(counts):
                r, pos = slice(at, at + n), self.lens[b] + np.arange(n)
                at += n
                if n == 0:
                    continue
                turned = lambda a: pm.rotated(a, None, 0.0, self.cos, self.sin, pos)
                ref, mine = turned(parts[r, :HEADS]), q[r].reshape(n, HEADS, HD)
                assert np.all(np.abs(mine - ref) <= 2.0 ** -24 * np.abs(ref) + 2.0 ** -45 * np.abs(ref).max())
                k, v = self.held[b][l]
                k = np.concatenate([k, turned(parts[r, HEADS:HEADS + KVH]).astype(np.float32)])
                v = np.concatenate([v, parts[r, HEADS + KVH:]])
                self.held[b][l] = (k, v)
                sinks_test._check(out[r].reshape(n, HEADS, HD), mine, pm.held(k, PAGE), pm.held(v, PAGE), self.lens[b],
                                  HD ** -0.5, WINDOW, SINKS, columns=max(counts) * (HEADS // KVH))
        self.lens = ends


def test_streams(ctx):
    sv = Server(ctx)
    sv.step([37, 20, 0, 0, 0])  # two prompts
    for _ in range(3):
        sv.step([1, 1, 0, 0, 0])
    sv.turn([0, 1, 0, 0, 1], [40, 23, 40, 40, 23])  # candidates of both
    sv.step([1, 1, 1, 1, 1])
    for _ in range(9):  # past a page's end, each its own
        sv.step([1, 1, 1, 1, 1])
    sv.turn([2, 1, 2, -1, 2], [50, 33, 50, 0, 50])  # one is best, another goes on, the rest end
    sv.step([1, 1, 1, 25, 1])  # a prompt beside them
    for _ in range(20):
        sv.step([1, 1, 1, 1, 1])
    assert min(sv.lens) > 40
    sv.turn([0, 1, 2, 3, 4], sv.lens, pack=True)  # what the window has passed goes back
    used = sum(r > 0 for r in sv.refs.tolist())
    assert used < sum(-(-n // PAGE) for n in sv.lens) - 4
    for _ in range(30):
        sv.step([1, 1, 1, 1, 1])
        sv.turn([0, 1, 2, 3, 4], sv.lens)
    assert sum(r > 0 for r in sv.refs.tolist()) <= BATCH * (2 + 4)  # sinks, window, the page being filled
    sv.turn([4, 0, -1, 0, 1], [sv.lens[4], 96, 0, 96, sv.lens[1]], pack=True)  # in another order, one back to a page's end
    sv.step([1, 16, 33, 2, 1])
    for _ in range(8):
        sv.step([1, 1, 1, 1, 1])


def test_streams_in_a_graph(ctx):
    """A step and the turn before it captured once; replayed with the server's own
    eager work between, each replay gives what the same calls give by themselves."""
    results = []
    for captured in (False, True):
        sv = Server(ctx)
        sv.step([60, 33, 47, 5, 70])
        starts, ends, source = (paged._ints(a) for a in (sv.lens, [n + 1 for n in sv.lens], range(BATCH)))
        offsets, copied = paged._ints(range(BATCH + 1)), paged._ints([0] * BATCH)
        xs = [paged._up(np.random.default_rng(50 + i).standard_normal((BATCH, HIDDEN)).astype(np.float32))
              for i in range(10)]
        x, y = torch.zeros_like(xs[0]), torch.zeros_like(xs[0])
        qkv, q, out = (torch.zeros((BATCH, w), device="cuda") for w in (QKV, HEADS * HD, HEADS * HD))
        seqs = qtts.PagedSeqs(BATCH, WIDE, BATCH, 1, sv.table.data_ptr(), sv.slots.data_ptr(), starts.data_ptr(),
                              offsets.data_ptr(), paged.ROPE_ROWS)
        layer = sv.layers[0]

        def call():
            at, kv = qkv.data_ptr(), layer["cache"].kv
            ctx.paged_remap_device(sv.pool, source.data_ptr(), starts.data_ptr(), window=WINDOW, sinks=SINKS,
                                   copied=copied.data_ptr())
            ctx.paged_copy_open_device(kv, BATCH, copied.data_ptr(), sv.slots.data_ptr(), starts.data_ptr())
            ctx.paged_reserve_device(sv.pool, starts.data_ptr(), ends.data_ptr())
            ctx.fp8_gemm_device(layer["qkv"].w, x.data_ptr(), HIDDEN, BATCH, at, QKV)
            ctx.paged_append_device(kv, seqs, at + 4 * HEADS * HD, QKV, at + 4 * (HEADS + KVH) * HD, QKV, heads=HEADS,
                                    q=at, ld_q=QKV, q_out=q.data_ptr(), ld_q_out=HEADS * HD,
                                    rope_cos=sv.d_cos.data_ptr(), rope_sin=sv.d_sin.data_ptr(), rope_rows=paged.ROPE_ROWS)
            ctx.paged_attention_device(kv, seqs, HEADS, q.data_ptr(), HEADS * HD, out.data_ptr(), HEADS * HD,
                                       scale=HD ** -0.5, window=WINDOW, sinks=SINKS)
            ctx.fp8_gemm_device(layer["o"].w, out.data_ptr(), HEADS * HD, BATCH, y.data_ptr(), HIDDEN, add=x.data_ptr(),
                                ld_add=HIDDEN)

        torch.cuda.synchronize()
        if captured:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=sv.stream):
                call()
        got = []
        for i, new in enumerate(xs):
            torch.cuda.synchronize()
            with torch.cuda.stream(sv.stream):
                x.copy_(new)
                if i == 4:  # a fork: row 1 goes on from row 4
                    source.copy_(paged._ints([0, 4, 2, 3, 4]))
                    starts[1], ends[1] = starts[4].clone(), ends[4].clone()
                else:
                    source.copy_(paged._ints(range(BATCH)))
                (g.replay if captured else call)()
                starts += 1
                ends += 1
            torch.cuda.synchronize()
            got.append([t.clone() for t in (y, out, sv.table, sv.refs, sv.slots, copied)])
        results.append(got)
    for eager, replayed in zip(*results):
        assert all(torch.equal(a, b) for a, b in zip(eager, replayed))
    assert any(bool((step[5] >= 0).any()) for step in results[0])
