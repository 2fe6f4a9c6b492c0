"""The pages of a cache restated with lists: rows of a table that go on, fork, go
back or end, pages given out, the pool packed."""


def in_pool(i, pages):
    return 0 <= i < pages


def remap(table, refs, slots, source, tokens, page, window=0, sinks=0):
    """(table, refs, slots, copied) after the call."""
    batch, pages = len(table), len(refs)
    wide = len(table[0]) if batch else 0
    source = [s if 0 <= s < batch else -1 for s in (range(batch) if source is None else source)]
    tokens = [min(max(t, 0), wide * page) if s >= 0 else 0 for s, t in zip(source, tokens)]
    refs, new, heirs = list(refs), [], {}
    for row in table:
        for i in row:
            if in_pool(i, pages):
                refs[i] -= 1
    for b, (s, t) in enumerate(zip(source, tokens)):
        row = [-1] * wide
        if s >= 0:
            heirs.setdefault(s, b)
            if s == b:
                heirs[s] = b
            for j in range(-(-t // page) if s == b else t // page):
                # the next row sees tokens from t - window + 1 on, and the sinks
                seen = not window or any(x > t - window or x < sinks for x in (j * page, (j + 1) * page - 1))
                if seen and in_pool(table[s][j], pages):
                    row[j] = table[s][j]
                    refs[row[j]] += 1
        new.append(row)
    ended = [slots[b] for b in range(batch) if b not in heirs]
    taken, copied = [], []
    for b, (s, t) in enumerate(zip(source, tokens)):
        if s >= 0 and heirs[s] == b:
            taken.append(slots[s])
            copied.append(-1)
        else:
            taken.append(ended.pop(0))
            copied.append(slots[s] if s >= 0 and t % page else -1)
    return new, refs, taken, copied


def reserve(table, refs, starts, ends, page):
    """(table, refs, lacking) after the call."""
    pages = len(refs)
    table, refs = [list(r) for r in table], list(refs)
    free = [i for i, r in enumerate(refs) if r <= 0]
    lacking, stuck = [], False
    for row, a, e in zip(table, starts, ends):
        if a < 0 or e < 0 or e > len(row) * page:
            lacking.append(-1)
            continue
        want = [j for j in range(a // page, -(-e // page)) if not in_pool(row[j], pages)]
        stuck |= len(want) > len(free)
        lacking.append(len(want) if stuck else 0)
        if not stuck:
            for j in want:
                row[j] = free.pop(0)
                refs[row[j]] = 1
    return table, refs, lacking


def compact(table, refs):
    """(table, refs, from, to, live) after the call."""
    refs = list(refs)
    live = sum(r > 0 for r in refs)
    frm = [i for i in range(live, len(refs)) if refs[i] > 0]
    to = [i for i in range(live) if refs[i] <= 0]
    name = dict(zip(frm, to))
    table = [[name.get(i, i) for i in row] for row in table]
    for a, b in name.items():
        refs[b], refs[a] = refs[a], 0
    rest = [-1] * (len(refs) // 2 - len(frm))
    return table, refs, frm + rest, to + rest, live
