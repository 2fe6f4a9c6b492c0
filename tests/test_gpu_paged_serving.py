"""The paged cache and the row sampler as a server uses them: one decoder layer
with sequences that join while others go on, leave, and hand their pages and
slot to the next.  Products in between are the framework's; each operator is
held against its definition in 64 bits on the values that it was given."""
import numpy as np
import pytest
import torch

import paged_model as pm
import qtts
import test_gpu_paged as paged
import test_gpu_sample_rows as sampling

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KVH, HD, PAGE, VOCAB = 256, 8, 2, 64, 16, 12320  # a vocabulary of the sampler's long rows
QKV = (HEADS + 2 * KVH) * HD


class Server:
    def __init__(self, ctx, slots, pages_each):
        self.ctx = ctx
        rng = np.random.default_rng(1)
        weight = lambda k, n, s: qtts.DeviceQ4(ctx, qtts.Q4Weight.quantize(
            (rng.standard_normal((k, n)) * s).astype(np.float32)))
        self.embed = paged._up(rng.standard_normal((VOCAB, HIDDEN)).astype(np.float32))
        self.qkv, self.o = weight(HIDDEN, QKV, 0.06), weight(HEADS * HD, HIDDEN, 0.06)
        self.head = weight(HIDDEN, VOCAB, 0.1)
        cos, sin = paged._rope(HD)
        self.cos, self.sin = cos, sin
        self.d_cos, self.d_sin = paged._up(cos), paged._up(sin)
        self.norms = [(1 + 0.1 * rng.standard_normal(HD)).astype(np.float16) for _ in range(2)]
        self.d_norms = [paged._up(n) for n in self.norms]
        self.cache = paged.Cache(KVH, HD, PAGE, slots, pages_each, spare=0)
        self.free_pages = list(range(slots * pages_each))
        self.free_slots = list(range(slots))
        self.max_pages = pages_each
        self.stream = torch.cuda.ExternalStream(ctx.stream)
        self.rng = np.random.default_rng(2)

    def join(self, prompt):
        return dict(slot=self.free_slots.pop(0), pages=[], n=0, next=list(prompt), k=np.zeros((0, KVH, HD), np.float32),
                    v=np.zeros((0, KVH, HD), np.float32), drawn=[])

    def leave(self, s):
        self.free_slots.append(s["slot"])
        self.free_pages += s["pages"]

    def step(self, live):
        """One call over every live sequence: prompts whole, others their last
        token; a token drawn for each."""
        counts = [len(s["next"]) for s in live]
        starts = [s["n"] for s in live]
        table = np.full((len(live), self.max_pages), -1, np.int32)
        for b, s in enumerate(live):
            while len(s["pages"]) * PAGE < s["n"] + counts[b]:
                s["pages"].append(self.free_pages.pop(0))
            table[b, :len(s["pages"])] = s["pages"]
        seqs = self.cache.seqs(starts, counts, table=paged._ints(table), slots=[s["slot"] for s in live])
        rows, ctx = sum(counts), self.ctx
        tokens = torch.tensor([t for s in live for t in s["next"]], device="cuda")
        u = self.rng.random(len(live)).astype(np.float32)
        par = dict(temperature=np.full(len(live), 0.9, np.float32), top_k=np.full(len(live), 60, np.int32),
                   top_p=np.full(len(live), 0.95, np.float32))
        d_par = {n: paged._up(a) for n, a in par.items()}
        d_u = paged._up(u)
        last = torch.tensor(np.cumsum(counts) - 1, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(self.stream):
            x = self.embed[tokens]
            qkv = torch.empty((rows, QKV), device="cuda")
            q, out = (torch.empty((rows, HEADS * HD), device="cuda") for _ in range(2))
            y = torch.empty((rows, HIDDEN), device="cuda")
            logits = torch.empty((len(live), VOCAB), device="cuda")
            token = torch.empty(len(live), dtype=torch.int32, device="cuda")
            at = qkv.data_ptr()
            self.qkv.gemm_device(x.data_ptr(), rows, at)
            ctx.paged_append_device(self.cache.kv, seqs, at + 4 * HEADS * HD, QKV, at + 4 * (HEADS + KVH) * HD, QKV,
                                    heads=HEADS, q=at, ld_q=QKV, q_out=q.data_ptr(), ld_q_out=HEADS * HD,
                                    q_norm=self.d_norms[0].data_ptr(), k_norm=self.d_norms[1].data_ptr(),
                                    rope_cos=self.d_cos.data_ptr(), rope_sin=self.d_sin.data_ptr(),
                                    rope_rows=paged.ROPE_ROWS)
            ctx.paged_attention_device(self.cache.kv, seqs, HEADS, q.data_ptr(), HEADS * HD, out.data_ptr(), HEADS * HD,
                                       scale=HD ** -0.5)
            self.o.gemm_device(out.data_ptr(), rows, y.data_ptr())
            h = (x + y)[last].contiguous()
            self.head.gemm_device(h.data_ptr(), len(live), logits.data_ptr())
            ctx.sample_rows_device(logits.data_ptr(), VOCAB, len(live), VOCAB, d_u.data_ptr(), token.data_ptr(),
                                   **{n: a.data_ptr() for n, a in d_par.items()})
        ctx.synchronize()
        qkv, q, out, logits, token = (t.cpu().numpy() for t in (qkv, q, out, logits, token))
        parts = qkv.reshape(rows, -1, HD)
        at = 0
        for b, s in enumerate(live):
            r = slice(at, at + counts[b])
            at += counts[b]
            pos = s["n"] + np.arange(counts[b])
            turn = lambda a, norm: pm.rotated(a, norm, 1e-6, self.cos, self.sin, pos)
            ref = turn(parts[r, :HEADS], self.norms[0])
            mine = q[r].reshape(ref.shape)
            assert np.all(np.abs(mine - ref) <= 2.0 ** -24 * np.abs(ref) + 2.0 ** -45 * np.abs(ref).max())
            s["k"] = np.concatenate([s["k"], turn(parts[r, HEADS:HEADS + KVH], self.norms[1]).astype(np.float32)])
            s["v"] = np.concatenate([s["v"], parts[r, HEADS + KVH:]])
            paged._check(out[r].reshape(ref.shape), mine, pm.held(s["k"], PAGE), pm.held(s["v"], PAGE), s["n"],
                         HD ** -0.5, 0)
            ref, _, kept = sampling.definition(logits[b], 0.9, 60, float(par["top_p"][b]), 0.0, float(u[b]))
            assert token[b] == ref and len(kept) > 1
            s["n"] += counts[b]
            s["next"] = [int(token[b])]
            s["drawn"].append(int(token[b]))


def test_serving(ctx):
    sv = Server(ctx, slots=3, pages_each=6)
    prompt = lambda n: sv.rng.integers(0, VOCAB, n)
    a, b = sv.join(prompt(40)), sv.join(prompt(17))
    sv.step([a, b])
    for _ in range(9):  # a fills its third page, b goes into its second
        sv.step([a, b])
    c = sv.join(prompt(33))
    sv.step([c, a, b])  # a prompt beside single tokens
    for _ in range(3):
        sv.step([b, c, a])  # in another order
    sv.leave(a)
    d = sv.join(prompt(70))  # a's slot and pages
    sv.step([b, c, d])
    for _ in range(20):
        sv.step([b, d])  # c waits
    sv.step([c, b, d])
    assert [len(s["drawn"]) for s in (a, b, c, d)] == [14, 36, 6, 22]


def _work(ctx, seed):
    """Calls that use the context's scratch in every way: tokens shared among
    blocks, in few columns and in many; long rows drawn from."""
    c, _ = paged._filled(ctx, KVH, HD, PAGE, [3000, 900], [40, 40], seed=seed)
    few, many = c.seqs([3039, 939], [1, 1]), c.seqs([3000, 900], [40, 40])
    q = paged._up(paged._normal(seed + 1, 80, HEADS * HD))
    outs = [torch.zeros_like(q) for _ in range(2)]
    x = paged._up(paged._normal(seed + 2, 7, VOCAB) * 3)
    u = paged._up(np.random.default_rng(seed).random(7).astype(np.float32))
    k, p = paged._ints([50, 0, 300, 0, 7, 0, 2000]), paged._up(np.full(7, 0.9, np.float32))
    token, share = torch.zeros(7, dtype=torch.int32, device="cuda"), torch.zeros(7, device="cuda")

    def call():
        for s, out in ((few, outs[0]), (many, outs[1])):
            ctx.paged_attention_device(c.kv, s, HEADS, q.data_ptr(), HEADS * HD, out.data_ptr(), HEADS * HD,
                                       scale=HD ** -0.5)
        ctx.sample_rows_device(x.data_ptr(), VOCAB, 7, VOCAB, u.data_ptr(), token.data_ptr(), probs=share.data_ptr(),
                               top_k=k.data_ptr(), top_p=p.data_ptr())

    def results():
        return [t.clone() for t in (*outs, token, share)]
    call.keep = (c, few, many, x, u, k, p)
    return call, results


def test_two_contexts_at_once(ctx):
    """Each has its scratch: what they give on their own."""
    other = qtts.Context(0)
    try:
        both = [_work(ctx, 20), _work(other, 30)]
        torch.cuda.synchronize()
        alone = []
        for (call, results), x in zip(both, (ctx, other)):
            call()
            x.synchronize()
            alone.append(results())
        for _ in range(30):
            for call, _ in both:
                call()
        ctx.synchronize(), other.synchronize()
        for (_, results), ref in zip(both, alone):
            assert all(torch.equal(a, b) for a, b in zip(results(), ref))
    finally:
        other.close()


def test_two_graphs_in_turn(ctx):
    """Captured from one context they share its scratch, and replayed on its
    stream, with plain calls between, they leave it to each other in order."""
    jobs = [_work(ctx, 40), _work(ctx, 50)]
    torch.cuda.synchronize()
    alone, graphs = [], []
    for call, results in jobs:
        call()
        ctx.synchronize()
        alone.append(results())
    stream = torch.cuda.ExternalStream(ctx.stream)
    for call, _ in jobs:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            call()
        graphs.append(g)
    for i in range(6):
        with torch.cuda.stream(stream):
            for g in graphs[::1 if i % 2 else -1]:
                g.replay()
            jobs[i % 2][0]()
            graphs[0].replay()
        torch.cuda.synchronize()
        for (_, results), ref in zip(jobs, alone):
            assert all(torch.equal(a, b) for a, b in zip(results(), ref))
