"""Plain forms of the operators of many requests (include/wgd.h), one request, page and key at a time."""
import numpy as np


def held(length, page):
    return -(-length // page)


def extend(table, lengths, refs, counts, tokens, page):
    """(table, lengths, refs, added, positions, slots) after the call."""
    table, lengths, refs = table.copy(), lengths.copy(), refs.copy()
    R, cap = len(lengths), table.shape[1] * page
    added = np.full(R, -1, np.int32)
    positions, slots = (np.full((R, tokens), -1, np.int32) for _ in range(2))
    for r in range(R):
        n = tokens if counts is None else int(counts[r])
        old = int(lengths[r])
        if not (0 <= n <= tokens and 0 <= old and old + n <= cap):
            continue
        have, need = held(old, page), held(old + n, page) - held(old, page) if n else 0
        free = np.flatnonzero(refs <= 0)
        if need > len(free):
            continue
        table[r, have:have + need] = free[:need]
        refs[free[:need]] = 1
        lengths[r], added[r] = old + n, n
        for t in range(n):
            positions[r, t] = old + t
            p = table[r, (old + t) // page]
            if 0 <= p < len(refs):
                slots[r, t] = p * page + (old + t) % page
    return table, lengths, refs, added, positions, slots


def fork(table, lengths, refs, origin, keep, page):
    """(table, lengths, refs, pairs) after the call, pairs None where the pages do not suffice."""
    R, cap, P = len(lengths), table.shape[1] * page, len(refs)
    new, lens, counts = table.copy(), lengths.copy(), refs.copy()
    true_len = np.clip(lengths, 0, cap)
    ok = lambda p: 0 <= p < P  # noqa: E731
    changed = []
    for r in range(R):
        o = int(origin[r])
        kept = 0
        if 0 <= o < R:
            kept = int(true_len[o]) if keep is None else max(0, min(int(keep[r]), int(true_len[o])))
        if o != r or kept < true_len[r]:
            changed.append((r, o, kept))
    for r, o, kept in changed:
        for p in table[r, :held(int(true_len[r]), page)]:
            if ok(p):
                counts[p] -= 1
        new[r] = -1
        if kept:
            new[r, :held(kept, page)] = table[o, :held(kept, page)]
        for p in new[r, :kept // page]:
            if ok(p):
                counts[p] += 1
        lens[r] = kept
    ends = [(r, kept // page) for r, _, kept in changed if kept % page and ok(new[r, kept // page])]
    alone = {int(new[r, c]) for r, c in ends if counts[new[r, c]] <= 0}
    copied = []
    for r, c in ends:
        p = int(new[r, c])
        if p in alone:
            alone.discard(p)
            counts[p] = 1
        else:
            copied.append((r, c))
    free = np.flatnonzero(counts <= 0)
    if len(copied) > len(free):
        return table, lengths, refs, None
    pairs = []
    for (r, c), to in zip(copied, free):
        pairs.append((int(new[r, c]), int(to)))
        new[r, c], counts[to] = to, 1
    return new, lens, counts, pairs


def compact(table, refs):
    """(table, refs, moved, pairs) after the call."""
    used = np.flatnonzero(refs > 0)
    n = len(used)
    pairs = list(zip(used[used >= n], [p for p in range(n) if refs[p] <= 0]))
    moved = np.full(len(refs), -1, np.int32)
    moved[used] = used
    after = refs.copy()
    for a, b in pairs:
        moved[a] = b
        after[b], after[a] = refs[a], 0
    return np.array([[moved[p] if 0 <= p < len(refs) else p for p in row] for row in table], np.int32), after, moved, pairs


def attention(q, k, v, table, lengths, counts, scale, window):
    """q [requests][tokens][heads][hd]; k, v [pages][page][kvh][hd]; float64, zeros where a row sees nothing."""
    pages, page, kvh, hd = k.shape
    R, T, heads, _ = q.shape
    y = np.zeros(q.shape)
    for r in range(R):
        n = int(np.clip(lengths[r], 0, table.shape[1] * page))
        asked = min(n, T if counts is None else int(np.clip(counts[r], 0, T)))
        for t in range(asked):
            pos = n - asked + t
            keys = [(int(table[r, j // page]), j % page) for j in range(max(0, pos + 1 - window), pos + 1)]
            keys = [(p, o) for p, o in keys if 0 <= p < pages]
            if not keys:
                continue
            at, off = np.array(keys).T
            kk, vv = k[at, off].astype(np.float64), v[at, off].astype(np.float64)
            for h in range(heads):
                g = h // (heads // kvh)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = kk[:, g] @ q[r, t, h].astype(np.float64) * scale
                    p = np.exp(s - s.max())
                    y[r, t, h] = p @ vv[:, g] / p.sum()
    return y


def adapters(y, x, a, b, which, scales):
    """y [batch][rows] after the call, in float64."""
    out = y.astype(np.float64)
    for t, w in enumerate(which):
        if 0 <= w < len(scales):
            out[t] += float(scales[w]) * (b[w].astype(np.float64) @ (a[w].astype(np.float64) @ x[t].astype(np.float64)))
    return out
