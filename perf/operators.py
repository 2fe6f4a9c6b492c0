"""Serving operators over a paged 8-bit cache, as measurable cases.

Four operators that a server of many streams runs between its products: the
rotated append of keys and values to a paged cache (with the cached rows read
back as f32), attention over that cache, and sampling of many rows from given
random numbers.  Each is here in its plain form, elementary torch operations,
and as the calls of the Python binding (`qtts.py`, one C entry point each).

The cache's layout: pages of P tokens; int8 codes with one f32 scale for each
page and kv head, K as [pages][kv_heads][P][head_dim], V as
[pages][kv_heads][head_dim][P].  The page that a sequence is filling is held
in f32, [slots][kv_heads][P][head_dim], and rounded once, when it is full:
scale = max|x| / 127, code = 127 x / max|x| to the nearest, ties to even.
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

# The talker's heads: 16 over 8 kv heads of 128 (the 1.7B shapes); the speech
# decoder's: 16 of 64, each with its own keys, over a window of 72.
TALKER = {"heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64}
DECODER = {"heads": 16, "kv_heads": 16, "head_dim": 64, "page": 32}
ROPE_ROWS, ROPE_THETA, EPS = 32768, 1.0e6, 1.0e-6
TEXT_VOCAB, CODE_VOCAB = 151936, 2048


def listed():
    return [
        # One token of one stream: what a single user's step adds to one
        # layer's cache.
        dict(TALKER, name="append_one", kind="append", batch=1, rows=1, context=1064, norm=True),
        # One token of each of 64 streams at ragged lengths; some fill a page.
        dict(TALKER, name="append_64", kind="append", batch=64, rows=1, context=4000, norm=True),
        # Prompts of four requests, the second parts of them: pages that were
        # begun before, whole ones, and ones left open.
        dict(TALKER, name="append_prompts", kind="append", batch=4, rows=2000, context=1500, norm=True),
        # One stream's step over the cache of a 1064-row prompt (latency).
        dict(TALKER, name="attend_one", kind="attend", batch=1, rows=1, context=1064, window=0),
        # Sixteen streams past their prompts.
        dict(TALKER, name="attend_16", kind="attend", batch=16, rows=1, context=2064, window=0),
        # Four streams at the end of the talker's position table.
        dict(TALKER, name="attend_far", kind="attend", batch=4, rows=1, context=32760, window=0),
        # A full server: 64 streams of up to 8000 tokens.
        dict(TALKER, name="attend_64", kind="attend", batch=64, rows=1, context=8000, window=0),
        # The second part of a long prompt, over the first.
        dict(TALKER, name="attend_chunk", kind="attend", batch=1, rows=1064, context=2000, window=0),
        # Frames of eight codes' streams under the decoder's sliding window.
        dict(DECODER, name="attend_window", kind="attend", batch=8, rows=500, context=300, window=72),
        # One row over the text vocabulary (latency).
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": TEXT_VOCAB, "mix": False},
        # A full server's rows over it, every request with its own settings.
        {"name": "sample_64", "kind": "sample", "rows": 64, "vocab": TEXT_VOCAB, "mix": True},
        # 64 streams' codes of one group.
        {"name": "sample_codes", "kind": "sample", "rows": 64, "vocab": CODE_VOCAB, "mix": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "sample"])
    if kind == "sample":
        rows = _log(rng, 1, 64)
        return {"kind": kind, "rows": rows, "vocab": _log(rng, 100, TEXT_VOCAB), "mix": rng.random() < 0.7}
    heads, kv_heads, head_dim = rng.choice([(16, 8, 128), (16, 8, 128), (16, 16, 64), (12, 4, 128), (8, 1, 128),
                                            (6, 2, 64), (32, 2, 128)])
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": rng.choice([16, 32, 64, 128])}
    shape = rng.choice(["one", "one", "few", "many"])
    if shape == "many":  # at most the work of the listed part of a prompt
        most = 1064 * 2500 * 2048 // (heads * head_dim)
        rows = _log(rng, 10, 1064)
        batch = _log(rng, 1, max(1, min(6, most // (rows * (rows + 50)))))
        context = _log(rng, 1, max(1, min(4000, most // (batch * rows) - rows)))
    else:
        rows = 1 if shape == "one" else _log(rng, 2, 9)
        batch = _log(rng, 1, 64)
        context = _log(rng, 1, min(30000, 64 * 8000 // batch))
    case.update(batch=batch, rows=rows, context=context)
    if kind == "append":
        case["norm"] = rng.random() < 0.5
    else:
        case["window"] = rng.choice([0, 0, 0, _log(rng, 1, 2000)])
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


def _read_starts(case):
    """The first position of each sequence that an append changes: its first
    new row, or the beginning of the page that it fills."""
    p = case["page"]
    return [s // p * p if (s + n) // p > s // p else s for s, n in zip(*_lengths(case))]


def _offsets(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@functools.lru_cache(maxsize=None)
def _rope(head_dim):
    half = head_dim // 2
    freq = ROPE_THETA ** (-torch.arange(half, dtype=torch.float64, device="cuda") * 2 / head_dim)
    angle = torch.arange(ROPE_ROWS, dtype=torch.float64, device="cuda")[:, None] * freq
    return angle.cos().float().contiguous(), angle.sin().float().contiguous()


# ---------------------------------------------------------------------------
# Inputs, from the seed alone
# ---------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _paged(case, seed):
    """Page pool, open rows and plan of one layer of `batch` sequences."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    starts, news = _lengths(case)
    p, kvh, hd, batch = case["page"], case["kv_heads"], case["head_dim"], case["batch"]
    need = [-(-(s + n) // p) for s, n in zip(starts, news)]
    wide, pool = max(need), sum(need) + 3
    order = torch.randperm(pool, generator=gen, device="cuda").int()
    table = torch.zeros((batch, wide), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    s = {"case": case, "table": table, "starts": _int(starts), "offsets": _int(_offsets(news)),
         "rows": sum(news), "max_rows": max(news), "longest": max(a + n for a, n in zip(starts, news)),
         "slots": torch.randperm(batch + 2, generator=gen, device="cuda")[:batch].int()}
    # codes as full blocks of normal values have them (max at 3.5 to 4.5
    # deviations), scales of unequal heads and pages
    codes = torch.empty((2, pool, kvh, p * hd), dtype=torch.int8, device="cuda")
    for half in range(2):
        for i in range(0, pool, 1024):
            part = codes[half, i:i + 1024]
            part.copy_((_normal(gen, *part.shape) * 31).round_().clamp_(-127, 127))
    s["k_codes"], s["v_codes"] = codes[0].view(pool, kvh, p, hd), codes[1].view(pool, kvh, hd, p)
    scales = torch.exp(0.3 * _normal(gen, 2, pool, kvh)) / 31
    s["k_scales"], s["v_scales"] = scales[0], scales[1]
    opened = _normal(gen, 2, batch + 2, kvh, p, hd)
    s["opened"], s["k_open"], s["v_open"] = opened, opened[0], opened[1]
    return s, gen


def prepare(case, seed):
    if case["kind"] == "sample":
        return _prepare_sample(case, seed)
    s, gen = _paged(case, seed)
    heads, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "attend":
        s["q"] = _normal(gen, s["rows"], heads * hd)
        return s
    # rows as a fused q|k|v product leaves them, channels of unequal size
    width = (heads + 2 * kvh) * hd
    s["qkv"] = _normal(gen, s["rows"], width) * torch.exp(0.5 * _normal(gen, width))
    s["cos"], s["sin"] = _rope(hd)
    s["q_norm"] = (1 + 0.1 * _normal(gen, hd)).half() if case["norm"] else None
    s["k_norm"] = (1 + 0.1 * _normal(gen, hd)).half() if case["norm"] else None
    starts, news = _lengths(case)
    ends, firsts = [a + n for a, n in zip(starts, news)], _read_starts(case)
    s["ends"], s["read_starts"] = _int(ends), _int(firsts)
    counts = [e - f for e, f in zip(ends, firsts)]
    s["read_offsets"], s["read_rows"], s["read_max"] = _int(_offsets(counts)), sum(counts), max(counts)
    p = case["page"]
    s["touched"] = max((e + p - 1) // p - a // p for a, e in zip(starts, ends))
    # A pass over a page begun before leaves the next page's rows in its
    # place: the rows that were there are put back first, so that a pass can
    # be made again.
    again = any(a % p and e % p and e // p > a // p for a, e in zip(starts, ends))
    s["opened_before"] = s["opened"].clone() if again else None
    return s


def _prepare_sample(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    # a bulk, and a few tokens well above it, as a trained head has them
    logits = 2.0 * _normal(gen, rows, vocab)
    few = min(vocab, 40)
    places = torch.rand((rows, vocab), generator=gen, device="cuda").topk(few, 1).indices  # no place twice
    logits.scatter_(1, places, 8 + 2.5 * _normal(gen, rows, few))
    logits[:, vocab - vocab // 16:] = -math.inf  # control tokens that a request may not draw
    u = torch.rand(rows, generator=gen, device="cuda")

    def pick(values):
        i = torch.randint(0, len(values), (rows,), generator=gen, device="cuda")
        return torch.tensor(values, device="cuda")[i].contiguous()

    if case["mix"]:
        t, k = pick([0.0, 0.6, 0.8, 1.0, 1.3]), pick([0, 20, 50, 200, 2000]).int()
        p, m = pick([1.0, 0.95, 0.9, 0.8, 0.5]), pick([0.0, 0.0, 0.02, 0.1])
    else:
        t, k = torch.full((rows,), 0.8, device="cuda"), torch.full((rows,), 50, dtype=torch.int32, device="cuda")
        p, m = torch.full((rows,), 0.95, device="cuda"), torch.zeros(rows, device="cuda")
    return {"case": case, "logits": logits, "u": u, "temperature": t, "top_k": k, "top_p": p, "min_p": m}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "sample": _own_sample}[kind](s)
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[kind](s)


def _places(offsets, starts, rows):
    """(sequence, position) of each row."""
    r = torch.arange(rows, device="cuda")
    b = torch.searchsorted(offsets[1:].long(), r, right=True)
    return b, starts.long()[b] + r - offsets.long()[b]


def _rotated(x, norm, cos, sin):
    """RMSNorm and rotation of [rows][heads][head_dim] in 64 bits, rounded once."""
    x = x.double()
    if norm is not None:
        x = x * norm.double() / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    a, b = x.chunk(2, -1)
    cos, sin = cos.double()[:, None], sin.double()[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).float()


def _plain_append(s):
    case, rows = s["case"], s["rows"]
    heads, kvh, hd, p = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    qkv = s["qkv"].view(rows, heads + 2 * kvh, hd)
    _, pos = _places(s["offsets"], s["starts"], rows)
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rotated(qkv[:, :heads], s["q_norm"], cos, sin)
    new = torch.stack([_rotated(qkv[:, heads:heads + kvh], s["k_norm"], cos, sin), qkv[:, heads + kvh:]])
    # every page that the rows touch, [2][batch][pages][P][kv_heads][head_dim]
    first, start, end = (s["starts"].long() // p)[:, None], s["starts"].long()[:, None], s["ends"].long()[:, None]
    at = first * p + torch.arange(s["touched"] * p, device="cuda")
    source = (s["offsets"].long()[:-1, None] + at - start).clamp(0, rows - 1)
    opened = s["opened"] if s["opened_before"] is None else s["opened_before"]
    before = opened[:, s["slots"].long()].transpose(2, 3).repeat(1, 1, s["touched"], 1, 1)
    x = torch.where((at >= start)[..., None, None], new[:, source], before)
    x = x.view(2, case["batch"], s["touched"], p, kvh, hd)
    full = (first + torch.arange(s["touched"], device="cuda") + 1) * p <= end
    top = x.abs().amax((3, 5), keepdim=True)
    codes = (x.double() * 127 / top.double()).round_().float()
    held = torch.where(full[:, :, None, None, None], codes * (top / 127), x)
    held = held.view(2, case["batch"], s["touched"] * p, kvh * hd)
    b, pos = _places(s["read_offsets"], s["read_starts"], s["read_rows"])
    held = held[:, b, pos - first[b, 0] * p]
    return {"q": q.view(rows, -1), "k": held[0], "v": held[1]}


def _plain_attend(s):
    case, rows, longest, most = s["case"], s["rows"], s["longest"], s["max_rows"]
    heads, kvh, hd, p, batch = (case[n] for n in ("heads", "kv_heads", "head_dim", "page", "batch"))
    group = heads // kvh
    pages = s["table"].long()
    wide = pages.shape[1] * p
    k = (s["k_codes"][pages].float() * s["k_scales"][pages][..., None, None]).transpose(1, 2)
    v = (s["v_codes"][pages].float() * s["v_scales"][pages][..., None, None]).permute(0, 2, 1, 4, 3)
    k, v = k.reshape(batch, kvh, wide, hd), v.reshape(batch, kvh, wide, hd)
    j = torch.arange(wide, device="cuda")
    news = (s["offsets"][1:] - s["offsets"][:-1]).long()
    end = s["starts"].long() + news
    opened = (j >= (end // p * p)[:, None])[:, None, :, None]
    slots = s["slots"].long()
    k = torch.where(opened, s["k_open"][slots].repeat(1, 1, wide // p, 1), k)
    v = torch.where(opened, s["v_open"][slots].repeat(1, 1, wide // p, 1), v)
    # rows padded to the longest, [batch][kv_heads][head_dim][group * rows]
    i = torch.arange(most, device="cuda")
    q = s["q"].view(rows, kvh, group, hd)[(s["offsets"].long()[:-1, None] + i).clamp(max=rows - 1)]
    q = q.permute(0, 2, 4, 3, 1).reshape(batch, kvh, hd, group * most)
    scores = (k @ q).view(batch, kvh, wide, group, most) * hd ** -0.5
    pos = (s["starts"].long()[:, None] + i)[:, None, :]
    seen = j[:, None] <= pos
    if case["window"]:
        seen &= j[:, None] > pos - case["window"]
    scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    scores = torch.exp(scores - scores.amax(2, keepdim=True))
    scores = scores / scores.sum(2, keepdim=True)
    out = scores.view(batch, kvh, wide, group * most).transpose(2, 3).contiguous() @ v
    out = out.view(batch, kvh, group, most, hd).permute(0, 3, 1, 2, 4)
    b, pos = _places(s["offsets"], s["starts"], rows)
    return out[b, pos - s["starts"].long()[b]].reshape(rows, heads * hd)


def _plain_sample(s):
    logits, rows, vocab = s["logits"], s["case"]["rows"], s["case"]["vocab"]
    greedy = (s["temperature"] <= 0)[:, None]
    x, order = torch.sort(logits, dim=1, descending=True, stable=True)
    t = torch.where(greedy, 1.0, s["temperature"][:, None].double())
    w = torch.exp((x.double() - x[:, :1].double()) / t)
    rank = torch.arange(vocab, device="cuda")
    k = torch.where((s["top_k"] > 0) & (s["top_k"] < vocab), s["top_k"].long(), vocab)[:, None]
    w = torch.where(rank < torch.where(greedy, 1, k), w, 0.0)
    before = w.cumsum(1) - w
    p = s["top_p"][:, None].double()
    keep = (p >= 1) | (before < p * w.sum(1, keepdim=True)) | (rank == 0)
    keep &= w >= s["min_p"][:, None].double()
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    run_sum = kept.cumsum(1)
    target = s["u"][:, None].double() * run_sum[:, -1:]
    token = (run_sum <= target).sum(1)
    prob = kept.gather(1, token[:, None])[:, 0] / run_sum[:, -1]
    return {"token": token.int(), "prob": prob.float()}


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


def _own_views(qtts, s):
    case = s["case"]
    kv = qtts.PagedKv(s["k_codes"].data_ptr(), s["v_codes"].data_ptr(), s["k_scales"].data_ptr(),
                      s["v_scales"].data_ptr(), s["k_open"].data_ptr(), s["v_open"].data_ptr(),
                      s["k_codes"].shape[0], case["kv_heads"], case["head_dim"], case["page"], s["k_open"].shape[0])
    seqs = qtts.PagedSeqs(case["batch"], s["table"].shape[1], s["rows"], s["max_rows"], s["table"].data_ptr(),
                          s["slots"].data_ptr(), s["starts"].data_ptr(), s["offsets"].data_ptr())
    return kv, seqs


def _own_append(s):
    qtts, ctx, stream = _ctx()
    case, rows = s["case"], s["rows"]
    heads, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    kv, seqs = _own_views(qtts, s)
    with torch.cuda.stream(stream):
        if s["opened_before"] is not None:
            s["opened"].copy_(s["opened_before"])
        q = torch.empty((rows, heads * hd), device="cuda")
        k = torch.empty((s["read_rows"], kvh * hd), device="cuda")
        v = torch.empty((s["read_rows"], kvh * hd), device="cuda")
    at, ld = s["qkv"].data_ptr(), s["qkv"].shape[1]
    norms = {} if s["q_norm"] is None else {"q_norm": s["q_norm"].data_ptr(), "k_norm": s["k_norm"].data_ptr(),
                                            "eps": EPS}
    ctx.paged_append_device(kv, seqs, at + 4 * heads * hd, ld, at + 4 * (heads + kvh) * hd, ld, heads=heads, q=at,
                            ld_q=ld, q_out=q.data_ptr(), ld_q_out=heads * hd, rope_cos=s["cos"].data_ptr(),
                            rope_sin=s["sin"].data_ptr(), rope_rows=ROPE_ROWS, **norms)
    read = qtts.PagedSeqs(case["batch"], s["table"].shape[1], s["read_rows"], s["read_max"], s["table"].data_ptr(),
                          s["slots"].data_ptr(), s["read_starts"].data_ptr(), s["read_offsets"].data_ptr())
    ctx.paged_read_device(kv, read, s["ends"].data_ptr(), k.data_ptr(), kvh * hd, v.data_ptr(), kvh * hd)
    return {"q": q, "k": k, "v": v}


def _own_attend(s):
    qtts, ctx, stream = _ctx()
    case = s["case"]
    width = case["heads"] * case["head_dim"]
    kv, seqs = _own_views(qtts, s)
    with torch.cuda.stream(stream):
        out = torch.empty((s["rows"], width), device="cuda")
    ctx.paged_attention_device(kv, seqs, case["heads"], s["q"].data_ptr(), width, out.data_ptr(), width,
                               scale=case["head_dim"] ** -0.5, window=case["window"])
    return out


def _own_sample(s):
    _, ctx, stream = _ctx()
    case = s["case"]
    with torch.cuda.stream(stream):
        token = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
        prob = torch.empty(case["rows"], device="cuda")
    ctx.sample_rows_device(s["logits"].data_ptr(), case["vocab"], case["rows"], case["vocab"], s["u"].data_ptr(),
                           token.data_ptr(), probs=prob.data_ptr(), temperature=s["temperature"].data_ptr(),
                           top_k=s["top_k"].data_ptr(), top_p=s["top_p"].data_ptr(), min_p=s["min_p"].data_ptr())
    return {"token": token, "prob": prob}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["kind"] == "sample":
        n = float(case["rows"]) * case["vocab"]
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 3 * n}
    heads, kvh, hd, p = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    starts, news = _lengths(case)
    ends = [s + n for s, n in zip(starts, news)]
    rows = sum(news)
    if case["kind"] == "append":
        move = 4.0 * rows * (2 * heads + 2 * kvh) * hd + 4.0 * min(rows, ROPE_ROWS) * hd
        changed = sum(e - f for e, f in zip(ends, _read_starts(case)))
        closed = sum(e // p * p - f for e, f in zip(ends, _read_starts(case)) if e // p * p > f)
        begun = sum(s % p for s, e in zip(starts, ends) if e // p > s // p)
        # codes of full pages and f32 rows of open ones are written, and the
        # changed positions come back as f32
        move += 2.0 * kvh * hd * (closed + 4 * (changed - closed) + 4 * begun + 4 * changed)
        return {"bytes": move, "flops": 6.0 * rows * (heads + kvh) * hd + 4.0 * closed * kvh * hd}
    seen, pairs = 0, 0
    codes, opened = 0, 0
    for s, e in zip(starts, ends):
        w = case["window"] or e
        low = max(0, s - w + 1)
        full = e // p * p
        codes += max(0, full - low)
        opened += e - max(full, low)
        pairs += sum(min(t + 1, w) for t in range(s, e))
    move = 2.0 * kvh * hd * (codes + 4 * opened) + 8.0 * kvh * codes / p + 8.0 * rows * heads * hd
    return {"bytes": move, "flops": 4.0 * heads * hd * pairs}


# ---------------------------------------------------------------------------
# From the definitions, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](s)


def _exact_append(s):
    case = s["case"]
    heads, kvh, hd, p = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    cos, sin = s["cos"].double(), s["sin"].double()
    q_all, k_all, v_all = [], [], []

    def turn(x, norm, start):
        x = x.reshape(x.shape[0], -1, hd).double()
        if norm is not None:
            x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / hd + EPS) * norm.double()
        c = cos[start:start + x.shape[0], None].repeat(1, 1, 2)
        n = sin[start:start + x.shape[0], None].repeat(1, 1, 2)
        other = torch.cat([-x[..., hd // 2:], x[..., :hd // 2]], -1)
        return x * c + other * n

    at = 0
    for b, (start, n, low) in enumerate(zip(*_lengths(case), _read_starts(case))):
        rows = s["qkv"][at:at + n]
        at += n
        q_all.append(turn(rows[:, :heads * hd], s["q_norm"], start).reshape(n, -1))
        k = turn(rows[:, heads * hd:(heads + kvh) * hd], s["k_norm"], start)
        # a row is held in f32 until its page is full
        k = k.float().double()
        v = rows[:, (heads + kvh) * hd:].reshape(n, kvh, hd).double()
        slot = int(s["slots"][b])
        head = start % p
        for new, opened, out in ((k, s["k_open"], k_all), (v, s["v_open"], v_all)):
            x = torch.cat([opened[slot, :, :head].transpose(0, 1).double(), new])
            whole = x.shape[0] // p * p
            blocks = x[:whole].reshape(-1, p, kvh, hd)
            step = blocks.abs().amax((1, 3), keepdim=True) / 127
            held = torch.cat([((blocks / step).round() * step).reshape(-1, kvh, hd), x[whole:]])
            out.append(held[low - start // p * p:].reshape(-1, kvh * hd))
    return {"q": torch.cat(q_all), "k": torch.cat(k_all), "v": torch.cat(v_all)}


def _exact_attend(s):
    case = s["case"]
    heads, kvh, hd, p = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    out, at = [], 0
    for b, (start, n) in enumerate(zip(*_lengths(case))):
        end = start + n
        full = end // p
        ids, slot = s["table"][b, :full].long(), int(s["slots"][b])
        rows = s["q"][at:at + n].view(n, heads, hd).double()
        at += n
        pos = start + torch.arange(n, device="cuda")
        key = torch.arange(end, device="cuda")
        hidden = key > pos[:, None]
        if case["window"]:
            hidden |= key <= pos[:, None] - case["window"]
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


def _exact_sample(s):
    tokens, probs = [], []
    for i in range(s["case"]["rows"]):
        x = s["logits"][i].double()
        t, k = float(s["temperature"][i]), int(s["top_k"][i])
        if t <= 0:
            tokens.append(int(x.argmax()))
            probs.append(1.0)
            continue
        value, order = torch.sort(x, descending=True, stable=True)
        if 0 < k < x.numel():
            value, order = value[:k], order[:k]
        weight = torch.exp((value - value[0]) / t)
        if float(s["top_p"][i]) < 1:
            total = weight.cumsum(0)
            n = 1 + int((total[:-1] < float(s["top_p"][i]) * total[-1]).sum())
            weight, order = weight[:n], order[:n]
        some = weight >= float(s["min_p"][i])
        weight, order = weight[some], order[some]
        order, by = order.sort()
        weight = weight[by]
        total = weight.cumsum(0)
        at = int((total <= float(s["u"][i]) * total[-1]).sum())
        tokens.append(int(order[at]))
        probs.append(float(weight[at] / total[-1]))
    return {"token": torch.tensor(tokens, dtype=torch.int32), "prob": torch.tensor(probs, dtype=torch.float64)}
