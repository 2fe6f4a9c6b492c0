"""Operators of a server whose streams are long, many and share beginnings.

Attention over the paged cache with a window and first tokens that stay
visible, so that a stream of any length keeps a fixed number of pages; the
pages themselves, forked, given back, handed out, packed and copied on the
device; and the products between them on weights in 8-bit floats with a scale
for each block of 128 by 128.  Each is here in its plain form, elementary torch
operations, and as the calls of the Python binding (`qtts.py`, one C entry point
each).

The cache's layout: pages of P tokens; int8 codes with one f32 scale for each
page and kv head, K as [pages][kv_heads][P][head_dim], V as
[pages][kv_heads][head_dim][P].  The page that a sequence is filling is held
in f32, [slots][kv_heads][P][head_dim].

8-bit floats are e4m3 (4 bits of exponent, 3 of mantissa, largest 448).  Rows of
a product's input take a power of two for each 128 values, the least with which
they stay within 448; a weight's scales are any f32.
"""
import functools
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "qora-tts-12hz-1.7b_amd")

# The talker's heads: 16 over 8 kv heads of 128 (the 1.7B shapes).
TALKER = {"heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64}
POOL = {"kv_heads": 8, "head_dim": 128, "page": 64}
BLOCK = 128
MOST_WORK = 8192 * 2048 * 12288


def listed():
    return [
        # One stream's step far into a long reading, over the last 2048 tokens
        # and the first 4 (latency).
        dict(TALKER, name="sinks_one", kind="sinks", batch=1, rows=1, context=30000, window=2048, sinks=4),
        # A full server of such streams, with a prompt's first page held.
        dict(TALKER, name="sinks_64", kind="sinks", batch=64, rows=1, context=8000, window=1000, sinks=64),
        # A text chunk of four streams behind what they have said.
        dict(TALKER, name="sinks_chunk", kind="sinks", batch=4, rows=500, context=5000, window=1500, sinks=30),
        # One prompt becomes eight candidates.
        dict(POOL, name="fork_best", kind="fork", batch=8, context=1064, best=True, window=0, sinks=0),
        # A full server between two steps: streams end, begin, fork, are cut
        # back, and drop what their window has passed.
        dict(POOL, name="fork_64", kind="fork", batch=64, context=8000, best=False, window=1000, sinks=64),
        # A few streams ended; the pool is packed.
        dict(POOL, name="compact_8", kind="compact", batch=8, context=1064),
        # A full server's, half of it given back: 0.3 GB of a layer moved.
        dict(POOL, name="compact_64", kind="compact", batch=64, context=8000),
        # One token through the talker's gate and up projections.
        {"name": "fp8_one", "kind": "fp8", "rows": 1, "k": 2048, "n": 12288, "add": False},
        # Sixteen streams through its down projection, onto the residual.
        {"name": "fp8_16", "kind": "fp8", "rows": 16, "k": 6144, "n": 2048, "add": True},
        # Odd sizes: what a pruned projection's may be.
        {"name": "fp8_odd", "kind": "fp8", "rows": 333, "k": 1552, "n": 1001, "add": False},
        # A prompt through its q, k and v.
        {"name": "fp8_prompt", "kind": "fp8", "rows": 1064, "k": 2048, "n": 4096, "add": False},
        # A server's prompts in one product.
        {"name": "fp8_large", "kind": "fp8", "rows": 8192, "k": 2048, "n": 12288, "add": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["sinks", "sinks", "fork", "compact", "fp8", "fp8", "fp8"])
    if kind == "fp8":
        k, n = 16 * _log(rng, 4, 384), _log(rng, 64, 12288)
        rows = _log(rng, 1, min(8192, MOST_WORK // (k * n)))
        return {"kind": kind, "rows": rows, "k": k, "n": n, "add": rng.random() < 0.3}
    heads, kv_heads, head_dim = rng.choice([(16, 8, 128), (16, 8, 128), (16, 16, 64), (12, 4, 128), (8, 1, 128),
                                            (6, 2, 64), (32, 2, 128)])
    case = {"kind": kind, "kv_heads": kv_heads, "head_dim": head_dim, "page": rng.choice([16, 32, 64, 128])}
    if kind == "sinks":
        case["heads"] = heads
        shape = rng.choice(["one", "one", "few", "many"])
        if shape == "many":  # at most the work of the listed chunk
            most = 4 * 500 * 5500 * 2048 // (heads * head_dim)
            rows = _log(rng, 10, 1064)
            batch = _log(rng, 1, max(1, min(6, most // (rows * (rows + 50)))))
            context = _log(rng, 1, max(1, min(6000, most // (batch * rows) - rows)))
        else:
            rows = 1 if shape == "one" else _log(rng, 2, 9)
            batch = _log(rng, 1, 64)
            context = _log(rng, 1, min(30000, 64 * 8000 // batch))
        case.update(batch=batch, rows=rows, context=context, window=_log(rng, 1, 4000), sinks=_log(rng, 1, 300))
        return case
    case["batch"] = _log(rng, 1, 64)
    case["context"] = _log(rng, 1, 64 * 8000 * 1024 // (case["batch"] * kv_heads * head_dim) // 4)
    if kind == "fork":
        case.update(best=rng.random() < 0.3, window=rng.choice([0, _log(rng, 1, 4000)]), sinks=_log(rng, 1, 300))
    return case


# ---------------------------------------------------------------------------
# Plans: lengths go by the case alone
# ---------------------------------------------------------------------------
def _lengths(case):
    """(tokens cached before the call, new rows) of each sequence: ragged, the
    first at the case's own sizes."""
    rng = random.Random("%(batch)d %(rows)d %(context)d %(page)d" % case)
    starts, news = [case["context"]], [case["rows"]]
    for _ in range(case["batch"] - 1):
        starts.append(rng.randint(case["context"] // 2, case["context"]))
        news.append(rng.randint((case["rows"] + 1) // 2, case["rows"]))
    return starts, news


def _turn(case):
    """What a server does with its sequences between two steps: lengths before,
    each row's source and length after, and the length to make room for."""
    rng = random.Random("%(kind)s %(batch)d %(context)d %(page)d" % case)
    batch, most, p = case["batch"], case["context"], case["page"]
    if case["kind"] == "fork" and case["best"]:
        before, source = [most] + [0] * (batch - 1), [0] * batch
    else:
        before = [most] + [rng.randint(most // 2, most) for _ in range(batch - 1)]
        ends = 0.5 if case["kind"] == "compact" else 0.2
        source = [-1 if rng.random() < ends else rng.randrange(batch) if case["kind"] == "fork" and rng.random() < 0.3
                  else b for b in range(batch)]
    after, room = [], []
    for b, s in enumerate(source):
        n = before[s] if s >= 0 else 0
        if case["kind"] == "fork" and s == b and not case["best"] and rng.random() < 0.1:
            n = int(0.7 * n) // p * p  # gone back, to a page's first token
        after.append(n)
        room.append(n + 1 if s >= 0 else rng.randint(1, max(1, most // 4)))
    return before, source, after, room


def _offsets(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------
# Inputs, from the seed alone
# ---------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _pool(gen, pool, kvh, p, hd):
    """A pool of pages.  Codes as full blocks of normal values have them (max at
    3.5 to 4.5 deviations), scales of unequal heads and pages."""
    codes = torch.empty((2, pool, kvh, p * hd), dtype=torch.int8, device="cuda")
    for half in range(2):
        for i in range(0, pool, 1024):
            part = codes[half, i:i + 1024]
            part.copy_((_normal(gen, *part.shape) * 31).round_().clamp_(-127, 127))
    scales = torch.exp(0.3 * _normal(gen, 2, pool, kvh)) / 31
    return {"k_codes": codes[0].view(pool, kvh, p, hd), "v_codes": codes[1].view(pool, kvh, hd, p),
            "k_scales": scales[0], "v_scales": scales[1]}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "fp8":
        return _prepare_fp8(case, gen)
    if case["kind"] == "sinks":
        return _prepare_sinks(case, gen)
    return _prepare_pages(case, gen)


def _prepare_sinks(case, gen):
    starts, news = _lengths(case)
    p, kvh, hd, batch = case["page"], case["kv_heads"], case["head_dim"], case["batch"]
    window, sinks = case["window"], case["sinks"]
    # pages that the window has passed and that hold no sink have gone back
    held = [[j for j in range(-(-(s + n) // p)) if j * p < sinks or (j + 1) * p > s - window + 1]
            for s, n in zip(starts, news)]
    wide, pool = max(-(-(s + n) // p) for s, n in zip(starts, news)), sum(map(len, held)) + 3
    order = torch.randperm(pool, generator=gen, device="cuda").int()
    table = torch.full((batch, wide), -1, dtype=torch.int32, device="cuda")
    at = torch.tensor([b * wide + j for b, js in enumerate(held) for j in js], device="cuda")
    table.view(-1)[at] = order[:at.numel()]
    s = {"case": case, "table": table, "starts": _int(starts), "offsets": _int(_offsets(news)), "rows": sum(news),
         "max_rows": max(news), "slots": torch.randperm(batch + 2, generator=gen, device="cuda")[:batch].int()}
    s.update(_pool(gen, pool, kvh, p, hd))
    opened = _normal(gen, 2, batch + 2, kvh, p, hd)
    s["k_open"], s["v_open"] = opened[0], opened[1]
    s["q"] = _normal(gen, s["rows"], case["heads"] * hd)
    return s


def _prepare_pages(case, gen):
    before, source, after, room = _turn(case)
    p, batch = case["page"], case["batch"]
    # every sequence's own pages (the one that it fills among them), and the
    # beginning of some shared with the one before
    rng = random.Random("shared %(batch)d %(context)d" % case)
    need = [-(-n // p) for n in before]
    wide = max(max(need), max(-(-n // p) for n in room)) + 1
    shared = [0] + [min(need[b - 1], need[b] - 1) // 2 if need[b] > 1 and rng.random() < 0.3 else 0
                    for b in range(1, batch)]
    used = sum(need) - sum(shared)
    pool = 2 * used + sum(-(-n // p) for n in room) // 2 + 8
    order = torch.randperm(pool, generator=gen, device="cuda").int()
    table = torch.full((batch, wide), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, (n, k) in enumerate(zip(need, shared)):
        table[b, :k] = table[b - 1, :k]
        table[b, k:n] = order[at:at + n - k]
        at += n - k
    refs = torch.bincount(table[table >= 0].long(), minlength=pool).int()
    slots = torch.randperm(batch + 2, generator=gen, device="cuda")[:batch].int()
    # refs, table and slots in one buffer: a pass puts them back as they were
    # first, so that it can be made again
    parts = [refs, table.view(-1), slots]
    sizes = [-(-x.numel() // 4) * 4 for x in parts]
    meta = torch.zeros(sum(sizes), dtype=torch.int32, device="cuda")
    views = [v[:x.numel()] for v, x in zip(meta.split(sizes), parts)]
    for v, x in zip(views, parts):
        v.copy_(x)
    s = {"case": case, "meta": meta, "meta_before": meta.clone(), "refs": views[0], "table": views[1].view(batch, wide),
         "slots": views[2], "source": _int(source), "tokens": _int(after), "room": _int(room), "pages": pool}
    kvh, hd = case["kv_heads"], case["head_dim"]
    if case["kind"] == "compact":
        s.update(_pool(gen, pool, kvh, p, hd))
    opened = _normal(gen, 2, batch + 2, kvh, p, hd) if case["kind"] == "fork" else torch.zeros((2, 1, kvh, p, hd),
                                                                                            device="cuda")
    s["k_open"], s["v_open"] = opened[0], opened[1]
    return s


def _prepare_fp8(case, gen):
    rows, k, n = case["rows"], case["k"], case["n"]
    # channels of unequal size on both sides, a few of them far above the rest
    x = _normal(gen, rows, k) * torch.exp(0.7 * _normal(gen, k))
    w = _normal(gen, n, k) * torch.exp(0.5 * _normal(gen, n, 1)) * k ** -0.5
    blocks = torch.zeros((-(-n // BLOCK) * BLOCK, -(-k // BLOCK) * BLOCK), device="cuda")
    blocks[:n, :k] = w
    blocks = blocks.view(-(-n // BLOCK), BLOCK, -(-k // BLOCK), BLOCK)
    scales = blocks.abs().amax((1, 3)) / 448
    codes = (blocks / scales[:, None, :, None]).clamp_(-448, 448).to(torch.float8_e4m3fn)
    codes = codes.view(torch.uint8).view(-1, -(-k // BLOCK) * BLOCK)[:n, :k].contiguous()
    return {"case": case, "x": x, "codes": codes, "scales": scales.contiguous(),
            "add": _normal(gen, rows, -(-n // 4) * 4) if case["add"] else None}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"sinks": _own_sinks, "fork": _own_fork, "compact": _own_compact, "fp8": _own_fp8}[kind](s)
    return {"sinks": _plain_sinks, "fork": _plain_fork, "compact": _plain_compact, "fp8": _plain_fp8}[kind](s)


def _places(offsets, starts, rows):
    """(sequence, position) of each row."""
    r = torch.arange(rows, device="cuda")
    b = torch.searchsorted(offsets[1:].long(), r, right=True)
    return b, starts.long()[b] + r - offsets.long()[b]


def _plain_sinks(s):
    case, rows, most = s["case"], s["rows"], s["max_rows"]
    heads, kvh, hd, p, batch = (case[n] for n in ("heads", "kv_heads", "head_dim", "page", "batch"))
    group = heads // kvh
    pages = s["table"].long()
    wide = pages.shape[1] * p
    there = (pages >= 0).repeat_interleave(p, 1)
    pages = pages.clamp(min=0)
    k = (s["k_codes"][pages].float() * s["k_scales"][pages][..., None, None]).transpose(1, 2)
    v = (s["v_codes"][pages].float() * s["v_scales"][pages][..., None, None]).permute(0, 2, 1, 4, 3)
    k, v = k.reshape(batch, kvh, wide, hd), v.reshape(batch, kvh, wide, hd)
    j = torch.arange(wide, device="cuda")
    end = s["starts"].long() + (s["offsets"][1:] - s["offsets"][:-1]).long()
    opened = (j >= (end // p * p)[:, None])
    slots = s["slots"].long()
    k = torch.where(opened[:, None, :, None], s["k_open"][slots].repeat(1, 1, wide // p, 1), k)
    v = torch.where(opened[:, None, :, None], s["v_open"][slots].repeat(1, 1, wide // p, 1), v)
    # rows padded to the longest, [batch][kv_heads][head_dim][group * rows]
    i = torch.arange(most, device="cuda")
    q = s["q"].view(rows, kvh, group, hd)[(s["offsets"].long()[:-1, None] + i).clamp(max=rows - 1)]
    q = q.permute(0, 2, 4, 3, 1).reshape(batch, kvh, hd, group * most)
    scores = (k @ q).view(batch, kvh, wide, group, most) * hd ** -0.5
    pos = (s["starts"].long()[:, None] + i)[:, None, :]
    at = j[:, None]
    seen = (at <= pos) & ((at > pos - case["window"]) | (at < case["sinks"])) & (there | opened)[:, :, None]
    scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    scores = torch.exp(scores - scores.amax(2, keepdim=True))
    scores = scores / scores.sum(2, keepdim=True)
    out = scores.view(batch, kvh, wide, group * most).transpose(2, 3).contiguous() @ v
    out = out.view(batch, kvh, group, most, hd).permute(0, 3, 1, 2, 4)
    b, pos = _places(s["offsets"], s["starts"], rows)
    return out[b, pos - s["starts"].long()[b]].reshape(rows, heads * hd)


def _plain_remap(s, window, sinks):
    """New table rows from the old ones, references counted, and the slots: one
    heir of a sequence keeps its slot, itself if it goes on."""
    case, table, refs = s["case"], s["table"], s["refs"]
    p, batch, wide = case["page"], case["batch"], s["table"].shape[1]
    b, j = torch.arange(batch, device="cuda"), torch.arange(wide, device="cuda")
    source, tokens = s["source"].long(), s["tokens"].long()
    goes, kept = source >= 0, source == b
    old, src = table.long(), source.clamp(min=0)
    entries = torch.where(kept, -(-tokens // p), tokens // p)
    hold = goes[:, None] & (j < entries[:, None])
    if window:
        hold &= ((j + 1) * p > (tokens - window + 1)[:, None]) | (j * p < sinks)
    new = torch.where(hold, old[src], -1)
    one = torch.ones_like(new, dtype=torch.int32)
    refs.index_add_(0, old.clamp(min=0).view(-1), torch.where(old >= 0, -one, 0 * one).view(-1))
    refs.index_add_(0, new.clamp(min=0).view(-1), torch.where(new >= 0, one, 0 * one).view(-1))
    table.copy_(new)
    slots = s["slots"].clone()
    heir = torch.full((batch + 1,), batch, device="cuda")
    heir.scatter_reduce_(0, torch.where(goes, source, batch), torch.where(kept, -1, b), "amin")
    heir = torch.where(heir[:batch] == -1, b, heir[:batch])
    first = goes & (heir[src] == b)
    # the others take the slots of those that ended, in order
    ended = torch.argsort((heir < batch).int(), stable=True)
    order = (~first).long().cumsum(0) - 1
    s["slots"].copy_(slots[torch.where(first, src, ended[order.clamp(min=0)])])
    return torch.where(goes & ~first & (tokens % p > 0), slots[src], -1)


def _plain_fork(s):
    case, p, batch = s["case"], s["case"]["page"], s["case"]["batch"]
    s["meta"].copy_(s["meta_before"])
    copied = _plain_remap(s, case["window"], case["sinks"])
    # pages for what comes next, the lowest free ones, in order
    table, refs = s["table"], s["refs"]
    j = torch.arange(table.shape[1], device="cuda")
    want = (table < 0) & (j >= (s["tokens"].long() // p)[:, None]) & (j < (-(-s["room"].long() // p))[:, None])
    need = want.sum(1)
    free = (refs <= 0).sum()
    served = need.cumsum(0) <= free
    want &= served[:, None]
    rank = (want.view(-1).long().cumsum(0) - 1).view_as(want)
    lowest = torch.argsort((refs > 0).int(), stable=True)
    table.copy_(torch.where(want, lowest[rank.clamp(0, refs.numel() - 1)].int(), table))
    taken = torch.zeros_like(refs).index_add_(0, table.clamp(min=0).long().view(-1), want.int().view(-1))
    refs.copy_(torch.where(taken > 0, 1, refs))
    # open rows of those that have no slot of their own yet
    r = torch.arange(p, device="cuda")
    take = ((copied >= 0)[:, None] & (r < (s["tokens"].long() % p)[:, None]))[:, None, :, None]
    to, frm = s["slots"].long(), copied.clamp(min=0)
    k, v = s["k_open"], s["v_open"]
    k[to] = torch.where(take, k[frm], k[to])
    v[to] = torch.where(take, v[frm], v[to])
    return {"table": table, "refs": refs, "slots": s["slots"], "copied": copied.int(),
            "lacking": torch.where(served, 0, need).int(), "k_open": k, "v_open": v}


def _plain_compact(s):
    s["meta"].copy_(s["meta_before"])
    _plain_remap(s, 0, 0)
    refs, table, n = s["refs"], s["table"], s["pages"]
    ids = torch.arange(n, device="cuda")
    live = refs > 0
    count = live.sum()
    movers, holes = live & (ids >= count), ~live & (ids < count)
    moves = int(movers.sum())
    frm = torch.full((n // 2,), -1, dtype=torch.int32, device="cuda")
    to = frm.clone()
    frm[:moves], to[:moves] = ids[movers].int(), ids[holes].int()
    a, b = frm[:moves].long(), to[:moves].long()
    name = ids.clone()
    name[a] = b
    table.copy_(torch.where(table >= 0, name[table.clamp(min=0).long()].int(), table))
    refs[b] = refs[a]
    refs[a] = 0
    s["k_codes"][b], s["v_codes"][b] = s["k_codes"][a], s["v_codes"][a]
    s["k_scales"][b], s["v_scales"][b] = s["k_scales"][a], s["v_scales"][a]
    return {"table": table, "refs": refs, "from": frm, "to": to, "live": count.int().view(1), "k_codes": s["k_codes"],
            "v_codes": s["v_codes"], "k_scales": s["k_scales"], "v_scales": s["v_scales"]}


def _plain_fp8(s):
    case, x = s["case"], s["x"]
    rows, k, n = case["rows"], case["k"], case["n"]
    blocks = -(-k // BLOCK)
    x = torch.nn.functional.pad(x, (0, blocks * BLOCK - k)).view(rows, blocks, BLOCK)
    top = x.abs().amax(2, keepdim=True)
    part, e = torch.frexp(top)  # 448 = 0.875 * 2^9
    e = (e - 9 + (part > 0.875)).clamp(min=-126)
    e = torch.where(top > 0, e, -126)
    step = ((e.int() + 127) << 23).view(torch.float32)
    x = ((x / step).to(torch.float8_e4m3fn).float() * step).view(rows, -1)[:, :k]
    scales = s["scales"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    w = s["codes"].view(torch.float8_e4m3fn).float() * scales
    y = x @ w.t()
    return y if s["add"] is None else y + s["add"][:, :n]


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _ctx():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    import qtts

    ctx = qtts.Context(0)
    return qtts, ctx, torch.cuda.ExternalStream(ctx.stream)


def _own_sinks(s):
    qtts, ctx, stream = _ctx()
    case = s["case"]
    width = case["heads"] * case["head_dim"]
    kv = qtts.PagedKv(s["k_codes"].data_ptr(), s["v_codes"].data_ptr(), s["k_scales"].data_ptr(),
                      s["v_scales"].data_ptr(), s["k_open"].data_ptr(), s["v_open"].data_ptr(),
                      s["k_codes"].shape[0], case["kv_heads"], case["head_dim"], case["page"], s["k_open"].shape[0])
    seqs = qtts.PagedSeqs(case["batch"], s["table"].shape[1], s["rows"], s["max_rows"], s["table"].data_ptr(),
                          s["slots"].data_ptr(), s["starts"].data_ptr(), s["offsets"].data_ptr())
    with torch.cuda.stream(stream):
        out = torch.empty((s["rows"], width), device="cuda")
    ctx.paged_attention_device(kv, seqs, case["heads"], s["q"].data_ptr(), width, out.data_ptr(), width,
                               scale=case["head_dim"] ** -0.5, window=case["window"], sinks=case["sinks"])
    return out


def _own_pool(qtts, s):
    return qtts.PagedPool(s["refs"].data_ptr(), s["table"].data_ptr(), s["slots"].data_ptr(), s["pages"],
                          s["case"]["page"], s["case"]["batch"], s["table"].shape[1])


def _own_fork(s):
    qtts, ctx, stream = _ctx()
    case = s["case"]
    batch, pool = case["batch"], _own_pool(qtts, s)
    with torch.cuda.stream(stream):
        s["meta"].copy_(s["meta_before"])
        copied = torch.empty(batch, dtype=torch.int32, device="cuda")
        lacking = torch.empty(batch, dtype=torch.int32, device="cuda")
    tokens = s["tokens"].data_ptr()
    ctx.paged_remap_device(pool, s["source"].data_ptr(), tokens, window=case["window"], sinks=case["sinks"],
                           copied=copied.data_ptr())
    ctx.paged_reserve_device(pool, tokens, s["room"].data_ptr(), lacking.data_ptr())
    kv = qtts.PagedKv(0, 0, 0, 0, s["k_open"].data_ptr(), s["v_open"].data_ptr(), s["pages"], case["kv_heads"],
                      case["head_dim"], case["page"], s["k_open"].shape[0])
    ctx.paged_copy_open_device(kv, batch, copied.data_ptr(), s["slots"].data_ptr(), tokens)
    return {"table": s["table"], "refs": s["refs"], "slots": s["slots"], "copied": copied, "lacking": lacking,
            "k_open": s["k_open"], "v_open": s["v_open"]}


def _own_compact(s):
    qtts, ctx, stream = _ctx()
    case = s["case"]
    pool, most = _own_pool(qtts, s), s["pages"] // 2
    with torch.cuda.stream(stream):
        s["meta"].copy_(s["meta_before"])
        moves = torch.empty((2, most), dtype=torch.int32, device="cuda")
        live = torch.empty(1, dtype=torch.int32, device="cuda")
    frm, to = moves[0].data_ptr(), moves[1].data_ptr()
    ctx.paged_remap_device(pool, s["source"].data_ptr(), s["tokens"].data_ptr())
    ctx.paged_compact_device(pool, frm, to, live.data_ptr())
    kv = qtts.PagedKv(s["k_codes"].data_ptr(), s["v_codes"].data_ptr(), s["k_scales"].data_ptr(),
                      s["v_scales"].data_ptr(), 0, 0, s["pages"], case["kv_heads"], case["head_dim"], case["page"], 0)
    ctx.paged_copy_pages_device(kv, kv, most, frm, to)
    return {"table": s["table"], "refs": s["refs"], "from": moves[0], "to": moves[1], "live": live,
            "k_codes": s["k_codes"], "v_codes": s["v_codes"], "k_scales": s["k_scales"], "v_scales": s["v_scales"]}


def _own_fp8(s):
    qtts, ctx, stream = _ctx()
    case, add = s["case"], s["add"]
    rows, k, n = case["rows"], case["k"], case["n"]
    ld = -(-n // 4) * 4
    with torch.cuda.stream(stream):
        y = torch.empty((rows, ld), device="cuda")
    w = qtts.Fp8Weight(s["codes"].data_ptr(), s["scales"].data_ptr(), n, k, k)
    more = {} if add is None else {"add": add.data_ptr(), "ld_add": ld}
    ctx.fp8_gemm_device(w, s["x"].data_ptr(), k, rows, y.data_ptr(), ld, **more)
    return y[:, :n]


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["kind"] == "fp8":
        rows, k, n = case["rows"], case["k"], case["n"]
        scales = -(-n // BLOCK) * -(-k // BLOCK)
        move = float(n) * k + 4.0 * scales + 4.0 * rows * (k + n) + (4.0 * rows * n if case["add"] else 0.0)
        return {"bytes": move, "flops": 2.0 * rows * k * n}
    kvh, hd, p = case["kv_heads"], case["head_dim"], case["page"]
    if case["kind"] == "sinks":
        heads, window, sinks = case["heads"], case["window"], case["sinks"]
        codes = opened = rows = pairs = 0
        for s, n in zip(*_lengths(case)):
            e = s + n
            low, full = max(0, s - window + 1), e // p * p
            first = min(sinks, low)
            codes += min(first, full) + max(0, full - low)
            opened += max(0, first - full) + e - max(full, low)
            rows += n
            pairs += sum(min(t + 1, window + min(sinks, max(0, t + 1 - window))) for t in range(s, e))
        move = 2.0 * kvh * hd * (codes + 4 * opened) + 8.0 * kvh * codes / p + 8.0 * rows * heads * hd
        return {"bytes": move, "flops": 4.0 * heads * hd * pairs}
    before, source, after, room = _turn(case)
    held = sum(-(-n // p) for n in before)
    entries = held + sum(n // p for n in after)
    move = 8.0 * entries + 16.0 * case["batch"]
    if case["kind"] == "fork":
        again = [s >= 0 and s != b for b, s in enumerate(source)]
        move += 16.0 * kvh * hd * sum(n % p for n, a in zip(after, again) if a) + 4.0 * sum(-(-n // p) for n in room)
        return {"bytes": move, "flops": float(entries)}
    # of pages spread evenly over the pool, those that lie behind the live ones
    pool = 2 * held + sum(-(-n // p) for n in room) // 2 + 8
    live = sum(-(-n // p) for n in after)
    moved = live * (1.0 - live / pool)
    return {"bytes": move + 4.0 * moved * kvh * (p * hd + 4), "flops": float(entries)}


# ---------------------------------------------------------------------------
# From the definitions, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"sinks": _exact_sinks, "fork": _exact_fork, "compact": _exact_compact, "fp8": _exact_fp8}[case["kind"]](s)


def _exact_sinks(s):
    case = s["case"]
    heads, kvh, hd, p = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    out, at = [], 0
    for b, (start, n) in enumerate(zip(*_lengths(case))):
        end = start + n
        full = end // p
        ids, slot = s["table"][b, :full].long(), int(s["slots"][b])
        gone = ids < 0
        ids = ids.clamp(min=0)
        rows = s["q"][at:at + n].view(n, heads, hd).double()
        at += n
        pos = start + torch.arange(n, device="cuda")
        key = torch.arange(end, device="cuda")
        hidden = (key > pos[:, None]) | ((key <= pos[:, None] - case["window"]) & (key >= case["sinks"]))
        hidden[:, :full * p] |= gone.repeat_interleave(p)
        result = torch.empty((n, heads, hd), dtype=torch.float64, device="cuda")
        for g in range(kvh):
            k = s["k_codes"][ids, g].double() * s["k_scales"][ids, g].double()[:, None, None]
            v = (s["v_codes"][ids, g].double() * s["v_scales"][ids, g].double()[:, None, None]).transpose(1, 2)
            k = torch.cat([k.reshape(-1, hd), s["k_open"][slot, g, :end - full * p].double()])
            v = torch.cat([v.reshape(-1, hd), s["v_open"][slot, g, :end - full * p].double()])
            for h in range(g * heads // kvh, (g + 1) * heads // kvh):
                score = rows[:, h] @ k.t().contiguous() / math.sqrt(hd)
                result[:, h] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ v
        out.append(result.reshape(n, -1))
    return torch.cat(out)


def _exact_rows(s):
    """Tables, slots and copies after the turn, by lists."""
    case, p = s["case"], s["case"]["page"]
    _, source, after, _ = _turn(case)
    old, slots = s["table"].tolist(), s["slots"].tolist()
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    table, heirs = [], {}
    for b, (src, n) in enumerate(zip(source, after)):
        row = [-1] * len(old[b])
        if src >= 0:
            if src not in heirs or src == b:
                heirs[src] = b
            for j in range(-(-n // p) if src == b else n // p):
                if not window or (j + 1) * p > n - window + 1 or j * p < sinks:
                    row[j] = old[src][j]
        table.append(row)
    ended = [slots[b] for b in range(len(source)) if b not in heirs]
    taken, copied = [], []
    for b, (src, n) in enumerate(zip(source, after)):
        if src >= 0 and heirs[src] == b:
            taken.append(slots[src])
            copied.append(-1)
        else:
            taken.append(ended.pop(0))
            copied.append(slots[src] if src >= 0 and n % p else -1)
    return table, taken, copied, after


def _counted(table, pages):
    refs = [0] * pages
    for row in table:
        for i in row:
            if i >= 0:
                refs[i] += 1
    return refs


def _exact_fork(s):
    case, p = s["case"], s["case"]["page"]
    table, slots, copied, after = _exact_rows(s)
    refs = _counted(table, s["pages"])
    room = _turn(case)[3]
    free = [i for i, r in enumerate(refs) if r == 0]
    lacking, stuck = [], False
    for row, n, m in zip(table, after, room):
        want = [j for j in range(n // p, -(-m // p)) if row[j] < 0]
        stuck |= len(want) > len(free)
        lacking.append(len(want) if stuck else 0)
        if not stuck:
            for j in want:
                row[j] = free.pop(0)
                refs[row[j]] = 1
    k, v = s["k_open"].double().clone(), s["v_open"].double().clone()
    for frm, to, n in zip(copied, slots, after):
        if frm >= 0:
            k[to, :, :n % p], v[to, :, :n % p] = s["k_open"][frm, :, :n % p], s["v_open"][frm, :, :n % p]
    return {"table": _int(table), "refs": _int(refs), "slots": _int(slots), "copied": _int(copied),
            "lacking": _int(lacking), "k_open": k, "v_open": v}


def _exact_compact(s):
    table = _exact_rows(s)[0]
    refs = _counted(table, s["pages"])
    live = sum(r > 0 for r in refs)
    frm = [i for i in range(live, len(refs)) if refs[i] > 0]
    to = [i for i in range(live) if refs[i] == 0]
    name = dict(zip(frm, to))
    table = [[name.get(i, i) for i in row] for row in table]
    for a, b in name.items():
        refs[b], refs[a] = refs[a], 0
    rest = [-1] * (s["pages"] // 2 - len(frm))
    out = {"table": _int(table), "refs": _int(refs), "from": _int(frm + rest), "to": _int(to + rest),
           "live": _int([live])}
    a, b = torch.tensor(frm, device="cuda").long(), torch.tensor(to, device="cuda").long()
    for part in ("k_codes", "v_codes", "k_scales", "v_scales"):
        out[part] = s[part].clone() if "codes" in part else s[part].double()
        out[part][b] = out[part][a]
    return out


def _power(e):
    """2^e to the last bit, which a power function need not give."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_fp8(s):
    case, x = s["case"], s["x"].double()
    rows, k, n = case["rows"], case["k"], case["n"]
    w = s["codes"].view(torch.float8_e4m3fn).double()
    y = torch.zeros((rows, n), dtype=torch.float64, device="cuda")
    for j, at in enumerate(range(0, k, BLOCK)):
        part = x[:, at:at + BLOCK]
        top = part.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -140) / 448) - 1e-9).clamp(min=-126)
        e = torch.where(448 * _power(e) < top, e + 1, e)
        units = part / _power(e)
        # steps of e4m3: 2^-3 of the value's power of two, 2^-9 at least
        step = _power(torch.frexp(units).exponent.clamp(min=-5) - 4)
        code = (units / step).round() * step
        scale = s["scales"][:, j].double().repeat_interleave(BLOCK)[:n]
        y += _power(e) * (code @ w[:, at:at + BLOCK].t().contiguous()) * scale
    return y if s["add"] is None else y + s["add"][:, :n].double()
