"""The cache-block pool restated in plain Python over lists (test infrastructure)."""
from __future__ import annotations


def _valid(e, n):
    return 0 <= e < n


def extend(tables, lens, refs, add, bs):
    """-> tables, lens, refs, shortage."""
    width = len(tables[0]) if tables else 0
    need = []
    beyond = 0
    for r, n in enumerate(lens):
        have, want = -(-n // bs), -(-(n + max(add[r], 0)) // bs)
        need += [(r, b) for b in range(have, want)]
        beyond += max(want - width, 0)
    free = [p for p, c in enumerate(refs) if c == 0]
    short = max(len(need) - len(free), 0) + beyond
    if short:
        return tables, lens, refs, short
    tables, refs = [list(t) for t in tables], list(refs)
    for (r, b), p in zip(need, free):
        tables[r][b] = p
        refs[p] = 1
    return tables, [n + max(a, 0) for n, a in zip(lens, add)], refs, 0


def fork(tables, lens, refs, parents, bs):
    """-> tables, lens, refs, shortage, [(from, to)] of the blocks copied."""
    rows, n = len(lens), len(refs)
    width = len(tables[0]) if tables else 0
    parents = [p if 0 <= p < rows else -1 for p in parents]
    new, new_lens, need, seen = [], [], [], set()
    for r, p in enumerate(parents):
        new.append(list(tables[p]) if p >= 0 else [-1] * width)
        new_lens.append(lens[p] if p >= 0 else 0)
        at = new_lens[r] // bs
        if p >= 0 and new_lens[r] % bs and at < width and _valid(new[r][at], n):
            if p in seen or refs[new[r][at]] > 1:
                need.append((r, at))
        seen.add(p)
    free = [q for q, c in enumerate(refs) if c == 0]
    if len(need) > len(free):
        return tables, lens, refs, len(need) - len(free), []
    pairs = []
    for (r, at), q in zip(need, free):
        pairs.append((new[r][at], q))
        new[r][at] = q
    refs = list(refs)
    for t, by in ((tables, -1), (new, 1)):
        for row in t:
            for e in row:
                if _valid(e, n):
                    refs[e] += by
    return new, new_lens, refs, 0, pairs


def free(tables, lens, refs, bs, window, sinks, finished):
    """-> tables, lens, refs."""
    refs, new = list(refs), []
    for r, row in enumerate(tables):
        out = []
        for b, e in enumerate(row):
            drop = finished[r]
            if window and not drop:
                # the tokens of the block that some query at position >= lens[r] sees
                drop = not any(j < sinks or j > lens[r] - window for j in range(b * bs, b * bs + bs))
            if drop and _valid(e, len(refs)):
                refs[e] -= 1
            out.append(-1 if drop else e)
        new.append(out)
    return new, [0 if f else n for n, f in zip(lens, finished)], refs


def compact(tables, refs):
    """-> tables, refs, live, [(from, to)]."""
    live = sum(c > 0 for c in refs)
    holes = [p for p in range(live) if refs[p] <= 0]
    movers = [p for p in range(live, len(refs)) if refs[p] > 0]
    to = dict(zip(movers, holes))
    refs = list(refs)
    for a, b in to.items():
        refs[b], refs[a] = refs[a], 0
    return [[to.get(e, e) for e in row] for row in tables], refs, live, list(to.items())


def slots(tables, lens, refs, new_tokens, tokens, bs):
    """(query starts, positions, slots, rows, excess) of each row's last new_tokens tokens, in
    arrays of `tokens` entries; nothing is mapped where the rows have more."""
    new = [max(min(n, length), 0) for n, length in zip(new_tokens, lens)]
    excess = max(sum(new) - tokens, 0)
    starts, positions, where, rows = [0], [], [], []
    for r, n in enumerate(new):
        for pos in range(lens[r] - n, lens[r]) if not excess else ():
            block = tables[r][pos // bs] if pos // bs < len(tables[r]) else -1
            positions.append(pos)
            where.append(block * bs + pos % bs if 0 <= block < len(refs) else -1)
            rows.append(r)
        starts.append(len(rows))
    pad = tokens - len(rows)
    return starts, positions + [0] * pad, where + [-1] * pad, rows + [-1] * pad, excess
