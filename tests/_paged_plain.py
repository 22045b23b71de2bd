"""Plain forms of the paged cache's operators: loops over tokens, pages and
rows, float64 for what is computed.  Used by the host and GPU tests."""

from __future__ import annotations

import numpy as np


def attention(q, k_pages, v_pages, table, lengths, scale):
    """(o, bound inputs): float64 o [b, h, dv], and per row and head the
    probabilities, logits' absolute sums and gathered |v|."""
    p, hk, ps, _ = k_pages.shape
    b, h, _ = q.shape
    g = h // hk
    out = np.zeros((b, h, v_pages.shape[3]))
    rows = {}
    for i in range(b):
        n = min(max(int(lengths[i]), 0), table.shape[1] * ps)
        at = [(int(table[i, j // ps]), j % ps) for j in range(n)]
        at = [(e, s) for e, s in at if 0 <= e < p]
        if not at:
            continue
        e, s = np.array(at).T
        for j in range(h):
            k, v = (x[e, j // g, s].astype(np.float64) for x in (k_pages, v_pages))
            x = q[i, j].astype(np.float64)
            logit = scale * k @ x
            w = np.exp(logit - logit.max())
            w /= w.sum()
            out[i, j] = w @ v
            rows[i, j] = (w, logit, abs(scale) * np.abs(k) @ np.abs(x), np.abs(v))
    return out, rows


def write(k_pages, v_pages, k, v, table, starts, offsets):
    p, _, ps, _ = k_pages.shape
    b, m = table.shape
    for s in range(b):
        toks = [s] if offsets is None else range(max(int(offsets[s]), 0),
                                                 min(int(offsets[s + 1]), k.shape[1]))
        for t in toks:
            pos = int(starts[s]) + (0 if offsets is None else t - int(offsets[s]))
            if not 0 <= pos < m * ps:
                continue
            e = int(table[s, pos // ps])
            if 0 <= e < p:
                k_pages[e, :, pos % ps] = k[:, t]
                v_pages[e, :, pos % ps] = v[:, t]


def free(table, lengths, refs, rows):
    table, lengths, refs = table.copy(), lengths.copy(), refs.copy()
    for r in sorted({int(r) for r in rows if 0 <= r < len(table)}):
        for e in table[r]:
            if 0 <= e < len(refs):
                refs[e] -= 1
        table[r] = -1
        lengths[r] = 0
    return table, lengths, refs


def extend(table, lengths, refs, counts, ps):
    b, m = table.shape
    room = m * ps
    out, lens, new = table.copy(), lengths.copy(), refs.copy()
    free_pages = [e for e in range(len(refs)) if refs[e] <= 0]
    for r in range(b):
        n = min(max(int(lengths[r]), 0), room)
        goal = min(n + max(int(counts[r]), 0), room)
        end = goal
        for c in range(-(-n // ps), -(-goal // ps)):
            if 0 <= table[r, c] < len(refs):
                continue
            if free_pages:
                out[r, c] = free_pages.pop(0)
                new[out[r, c]] = 1
            else:
                out[r, c] = -1
                end = min(end, c * ps)
        lens[r] = end
    return out, lens, new


def fork(k_pages, v_pages, table, lengths, refs, src, dst):
    b, m = table.shape
    p, ps = len(refs), k_pages.shape[2]
    out, lens, new = table.copy(), lengths.copy(), refs.copy()
    pairs = [(int(s), int(d)) for s, d in zip(src, dst)]
    good = [0 <= s < b and 0 <= d < b and s != d for s, d in pairs]
    free_pages = [e for e in range(p) if refs[e] <= 0]
    for i, (s, d) in enumerate(pairs):
        if not good[i] or any(good[j] and pairs[j][1] == d for j in range(i + 1, len(pairs))):
            continue
        n = min(max(int(lengths[s]), 0), m * ps)
        full, rest = divmod(n, ps)
        for e in table[d]:
            if 0 <= e < p:
                new[e] -= 1
        row = np.full(m, -1, table.dtype)
        row[:full] = [e if 0 <= e < p else -1 for e in table[s, :full]]
        lens[d] = n
        if rest:
            if free_pages:
                row[full] = free_pages.pop(0)
                e = table[s, full]
                if 0 <= e < p:
                    k_pages[row[full], :, :rest] = k_pages[e, :, :rest]
                    v_pages[row[full], :, :rest] = v_pages[e, :, :rest]
            else:
                lens[d] = full * ps
        for e in row:
            if e >= 0:
                new[e] += 1
        out[d] = row
    return out, lens, new


def compact(k_pages, v_pages, table, refs):
    p = len(refs)
    n = int((refs > 0).sum())
    movers = [e for e in range(n, p) if refs[e] > 0]
    holes = [e for e in range(n) if refs[e] <= 0]
    to = dict(zip(movers, holes))
    new = np.maximum(refs, 0)
    for e, h in to.items():
        k_pages[h], v_pages[h] = k_pages[e], v_pages[e]
        new[h], new[e] = refs[e], 0
    return np.vectorize(lambda e: to.get(int(e), e), otypes=[table.dtype])(table), new


def cache(rng, b, m, p, ps, share=True):
    """A consistent state: (table, lengths, refs) int32, rows of up to m pages
    of a pool with some left free, some rows empty, some sharing whole pages."""
    table = np.full((b, m), -1, np.int32)
    lengths = np.zeros(b, np.int32)
    ids = list(rng.permutation(p))
    for r in range(b):
        if r % 5 == 3 and share and r > 0 and lengths[r - 1] >= ps:
            full = lengths[r - 1] // ps
            table[r, :full] = table[r - 1, :full]
            lengths[r] = full * ps
            continue
        n = int(rng.integers(0, m + 1))
        n = min(n, max(0, len(ids) - p // 4))
        for c in range(n):
            table[r, c] = ids.pop()
        if n:
            lengths[r] = n * ps - rng.integers(0, ps)
    refs = np.zeros(p, np.int32)
    for e in table.reshape(-1):
        if e >= 0:
            refs[e] += 1
    return table, lengths, refs
