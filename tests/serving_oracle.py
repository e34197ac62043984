"""Plain sequential forms of the serving-loop operators, in 64 bits and one stream after the other."""
import math

import numpy as np


def softmax(x, inv_t):
    """Probabilities of a row in 64 bits; None where it is no distribution."""
    x = np.asarray(x, np.float64)
    if np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all():
        return None
    e = np.exp((x - x.max()) * float(np.float32(inv_t)))
    return e / e.sum()


#: How near a number may come to a border: the sums that acceptance goes by are within 2^-18, a draw's are of 64 bits.
ACCEPT, DRAW = 2.0 ** -18, 1e-10


def _number(u):
    return 1.0 if math.isnan(u) else min(max(u, 0.0), 1.0)


def _drawn(w, u):
    """The first index whose cumulative sum passes u of the whole, else the last with any weight; and how near the
    pick was to a border, in units of DRAW of the whole."""
    cdf = np.cumsum(w)
    aim = _number(u) * cdf[-1]
    near = np.min(np.abs(cdf - aim)) / cdf[-1] / DRAW if 0.0 < _number(u) < 1.0 else np.inf
    hit = np.nonzero((cdf > aim) & (w > 0))[0]
    return (int(hit[0]) if len(hit) else int(np.nonzero(w > 0)[0][-1])), near


def _parent(i, mask):
    if mask is None:
        return i - 1 if i else -1
    i = int(i)
    m = int(mask[i]) & ((1 << 64) - 1)
    up = m & ((1 << i) - 1)
    return up.bit_length() - 1 if i and m >> i & 1 and up else -1


def verify_stream(x, tok, u, y=None, mask=None, inv_t=1.0, draft_inv_t=1.0, greedy=False):
    """(path, next token, margin) of one stream's rows.  A margin over 1 is safe."""
    n, vocab = x.shape
    if n == 0:
        return [], -1, np.inf
    parents = [_parent(i, mask) for i in range(n)]
    path, near = [0], np.inf
    while True:
        cur = path[-1]
        row = np.asarray(x[cur], np.float64)
        kids = [i for i in range(cur + 1, n) if parents[i] == cur]
        if greedy:
            top = np.where(np.isnan(row), -np.inf, row)
            best = int(np.argmax(top)) if top.max() > -np.inf else -1
            kids = [i for i in kids if best >= 0 and tok[i] == best]
            if not kids:
                return path, best, near
            path.append(kids[0])
            continue
        p = softmax(row, inv_t)
        q = None if y is None or cur == n - 1 else softmax(y[cur], draft_inv_t)
        if p is None:
            return path, -1, near
        left, gone, taken = 1.0, [], None
        for i in kids:
            t = int(tok[i])
            if not 0 <= t < vocab:
                continue
            if y is not None:
                if q is None:
                    continue
                a, b = _number(u[i]) * q[t], p[t]
            else:
                if t in gone:
                    continue
                a, b = _number(u[i]) * max(left, 0.0), p[t]
            if a != 0.0 and b != 0.0 and a != b:
                near = min(near, abs(a - b) / max(a, b) / ACCEPT)
            if a < b:
                taken = i
                break
            gone.append(t)
            left -= p[t]
        if taken is not None:
            path.append(taken)
            continue
        w = p
        if y is not None:
            if q is not None and cur < n - 1 and np.maximum(p - q, 0).sum() > 0:
                w = np.maximum(p - q, 0)
        else:
            rest = p.copy()
            rest[gone] = 0.0
            w = rest if rest.sum() > 0 else p
        t, d = _drawn(w, u[0])
        return path, t, min(near, d)


def verify(x, tok, start, u, max_rows, y=None, mask=None, inv_t=1.0, draft_inv_t=1.0, greedy=False, path=None):
    """(accepted, path, next tokens, margin); `path` is what it holds before."""
    streams = len(start) - 1
    accepted, nxt, near = np.zeros(streams, np.int32), np.full(streams, -1, np.int32), np.inf
    path = np.array(path, np.int32)
    for s in range(streams):
        a, b = int(start[s]), int(start[s + 1])
        if a < 0 or b < a or b > len(tok):
            continue
        b = min(b, a + max_rows)
        at = slice(a, b)
        got, t, d = verify_stream(x[at], tok[at], None if u is None else u[at], None if y is None else y[at],
                                  None if mask is None else mask[at], inv_t, draft_inv_t, greedy)
        near = min(near, d)
        path[at] = got + [-1] * (b - a - len(got))
        accepted[s], nxt[s] = max(len(got) - 1, 0), t
    return accepted, path, nxt, near


# ---------------------------------------------------------------- pages

def _page(e, n_pages):
    return int(e) if 0 <= e < n_pages else -1


def fork(table, refs, parent, length, page_size):
    """Table and refs afterwards."""
    old, new, refs = table.copy(), np.full_like(table, -1), refs.copy()
    for s in range(len(table)):
        p = parent[s]
        if 0 <= p < len(table):
            n = table.shape[1] if length is None else min(table.shape[1], max(0, -(-int(length[s]) // page_size)))
            for j in range(n):
                new[s, j] = _page(old[p, j], len(refs))
    for t, by in ((old, -1), (new, 1)):
        for e in t.reshape(-1):
            if _page(e, len(refs)) >= 0:
                refs[e] += by
    return new, refs


def reserve(table, refs, start, ctx, max_rows, page_size):
    """(table, refs, ok, copies): copies are (from, to, slots), in the order in which they are made."""
    table, refs, copies = table.copy(), refs.copy(), []
    ok, closed = np.zeros(len(table), np.int32), False
    for s in range(len(table)):
        n, c = int(start[s + 1]) - int(start[s]), int(ctx[s])
        if c < 0 or n < 0 or n > max_rows or c + n > table.shape[1] * page_size:
            continue
        pages = range(c // page_size, (c + n - 1) // page_size + 1) if n else range(0)
        wants = [j for j in pages if _page(table[s, j], len(refs)) < 0 or refs[table[s, j]] > 1]
        free = np.nonzero(refs == 0)[0]
        if not wants:
            ok[s] = 1
            continue
        if closed or len(wants) > len(free):
            closed = True
            continue
        ok[s] = 1
        for j, p in zip(wants, free):
            e = _page(table[s, j], len(refs))
            if e >= 0:
                refs[e] -= 1
                if j == c // page_size and c % page_size:
                    copies.append((e, int(p), c % page_size))
            table[s, j], refs[p] = p, 1
    return table, refs, ok, copies


def compact(pool_places, ctx, start, kept, max_rows):
    """Moves ((page, slot) to (page, slot)) of all streams; pool_places(s, position) is None where there is no place."""
    moves = []
    for s in range(len(start) - 1):
        a, b = int(start[s]), int(start[s + 1])
        if a < 0 or b > len(kept) or ctx[s] < 0:
            continue
        for j in range(min(b - a, max_rows)):
            k = int(kept[a + j])
            if 0 <= k < b - a and k != j:
                src, dst = pool_places(s, int(ctx[s]) + k), pool_places(s, int(ctx[s]) + j)
                if src is not None and dst is not None:
                    moves.append((src, dst))
    return moves
