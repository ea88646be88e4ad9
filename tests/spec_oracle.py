"""The operators of a step with drafted tokens from their definitions, in Python and
float64 NumPy: plain loops over requests, rows and heads."""
import math

import numpy as np


# ------------------------------------------------------------------- pages --
def plan(lens, new, table, held, free, n_free, *, page, n_tokens, n_pages, trim):
    """(table, held, free, n_free, cu, ctx, slots, pos) after a plan."""
    n_seq, entries = table.shape
    table, held, free = table.copy(), held.copy(), free.copy()
    lens, new = [max(int(x), 0) for x in lens], [max(int(x), 0) for x in new]
    total = [min(a + b, entries * page) for a, b in zip(lens, new)]
    need = [-(-t // page) for t in total]
    top = int(n_free[0])
    if trim:
        for b in reversed(range(n_seq)):
            while held[b] > need[b]:
                held[b] -= 1
                if 0 <= table[b, held[b]] < n_pages:
                    free[top] = table[b, held[b]]
                    top += 1
                table[b, held[b]] = -1
    lacking = 0
    for b in range(n_seq):
        at = int(held[b])
        for e in range(at, need[b]):
            if top > 0:
                top -= 1
                table[b, e] = free[top]
                held[b] += 1
            else:
                table[b, e] = -1
                lacking += 1
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    slots, pos = np.full(n_tokens, -1, np.int64), np.full(n_tokens, -1, np.int32)
    for b in range(n_seq):
        for j in range(new[b]):
            r, p = int(cu[b]) + j, lens[b] + j
            pos[r] = p
            if p // page < entries and 0 <= table[b, p // page] < n_pages:
                slots[r] = int(table[b, p // page]) * page + p % page
    return table, held, free, np.array([top, lacking], np.int32), cu, np.array(total, np.int32), slots, pos


# ------------------------------------------------------------------- trees --
def ancestors(parent):
    """Of one request's rows, the rows from each up to its root, itself first."""
    out = []
    for i in range(len(parent)):
        chain, at = [i], i
        while 0 <= parent[at] < at:
            at = int(parent[at])
            chain.append(at)
        out.append(chain)
    return out


def tree(parent, window=0):
    """(depths, sight as a boolean matrix) of one request's rows."""
    chains = ancestors(parent)
    sees = np.zeros((len(parent), len(parent)), bool)
    for i, chain in enumerate(chains):
        sees[i, chain[:window] if window else chain] = True
    return np.array([len(c) - 1 for c in chains], np.int32), sees


def words_of(sees, words):
    """A boolean matrix [rows, at most 64 words] as int64 words, lowest bit first."""
    out = np.zeros((sees.shape[0], words), np.uint64)
    for i, j in zip(*np.nonzero(sees)):
        out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out.view(np.int64)


# --------------------------------------------------------------- attention --
def attend(c, q, sees, *, heads, window=0, pos=None, scale=None):
    """As paged_oracle.attend, for rows that see each other by ``sees`` (a boolean
    matrix a sequence of the PagedCase ``c``)."""
    scale = 1 / math.sqrt(c.hd) if scale is None else scale
    G = heads // c.kv
    out = np.zeros((c.tokens, heads, c.hd))
    mag, prod, vmax = np.zeros_like(out), np.zeros((c.tokens, heads)), np.zeros((c.tokens, heads))
    for b, (n, ctx) in enumerate(zip(c.new, c.ctx)):
        if not n:
            continue
        first = ctx - n
        for h in range(c.kv):
            got = [(p, c.held(b, h, p)) for p in range(ctx)]
            got = [(p, x) for p, x in got if x is not None]
            if not got:
                continue
            P = np.array([p for p, _ in got])
            K, V = np.stack([x[0] for _, x in got]), np.stack([x[1] for _, x in got])
            top = np.abs(V[np.isfinite(V)]).max() if np.isfinite(V).any() else 0.0
            if c.store == "i8":
                scales = np.array([c.v_scale[pg, h, sl] for pg, sl in (c.place(b, p) for p, _ in got)])
                top = max(top, 127 * float(np.max(scales[np.isfinite(scales)])))
            for j in range(n):
                r = int(c.cu[b]) + j
                on = P < first
                if window:
                    on &= P > int(pos[r]) - window
                mine = P >= first
                on[mine] = sees[b][j][P[mine] - first]
                if not on.any():
                    continue
                for g in range(G):
                    x = q[r, h * G + g].astype(np.float64)
                    s = K[on] @ x * scale
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[r, h * G + g] = w @ V[on]
                    mag[r, h * G + g] = w @ np.abs(V[on])
                    prod[r, h * G + g] = (np.abs(K[on]) @ np.abs(x)).max() * abs(scale)
                    vmax[r, h * G + g] = top
    return out, mag, prod, vmax


# -------------------------------------------------------------- prologue --
def turned(x, gain, pos, *, n_rot, eps, base, interleaved, turn_scale, factors=None):
    """One head: RMS norm with gain (None: skipped), n_rot dims turned."""
    x = np.asarray(x, np.float64)
    if gain is not None:
        x = x / math.sqrt(float((x * x).mean()) + eps) * np.asarray(gain, np.float64)
    y = x.copy()
    half = n_rot // 2
    for j in range(half):
        a = pos * float(base) ** (-2.0 * j / n_rot) / (float(factors[j]) if factors is not None else 1.0)
        p, q = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        cos, sin = math.cos(a) * turn_scale, math.sin(a) * turn_scale
        y[p], y[q] = x[p] * cos - x[q] * sin, x[p] * sin + x[q] * cos
    return y


# ------------------------------------------------------------ verification --
def prob(x):
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore"):
        return np.where((x > 0) & np.isfinite(x), x, 0.0)


def pick(w, r):
    """The least t with w[0] + .. + w[t] > r * sum; -1 where w is 0."""
    sums = np.cumsum(w)
    if not sums[-1] > 0:
        return -1
    hit = np.nonzero(sums > max(r, 0.0) * sums[-1])[0]
    return int(hit[0]) if len(hit) else int(np.nonzero(w)[0][-1])


def verify(p, tokens, u, r, parent, q=None, greedy=False):
    """(path, token) of one request: its rows' p [n, vocab], tokens, u, parents."""
    n, vocab = p.shape if len(tokens) else (0, 0)
    if not n:
        return [], -1

    def best(row):
        x = np.asarray(p[row], np.float64)
        return int(np.nanargmax(x)) if not np.isnan(x).all() else -1

    at, path = 0, [0]
    a, W = 0.0, 1.0
    w = None if greedy else prob(p[0])
    for i in range(1, n):
        if parent[i] != at:
            continue
        t = int(tokens[i])
        ok = 0 <= t < vocab
        if greedy:
            passed = ok and t == best(at)
        elif q is not None:
            y = float(prob(q[at][t])) if ok else 0.0
            passed = ok and float(u[i]) * W * y < w[t]
            if ok and not passed:
                a += W
                w = np.maximum(prob(p[at]) - a * prob(q[at]), 0.0)
                W = float(w.sum())
        else:
            passed = ok and float(u[i]) * W < w[t]
            if ok and not passed:
                W -= w[t]
                w = w.copy()
                w[t] = 0.0
        if passed:
            at = i
            path.append(i)
            a, W = 0.0, 1.0
            w = None if greedy else prob(p[i])
    if greedy:
        return path, best(at)
    token = pick(w, float(r))
    return path, token if token >= 0 else pick(prob(p[at]), float(r))


# -------------------------------------------------------------------- keep --
def keep(c, path, accepted, arrays):
    """The pools of a PagedCase ``c`` ([k, v, k_scale, v_scale], None among them) after
    the accepted rows moved (copies)."""
    K, V, KS, VS = (None if x is None else x.copy() for x in arrays)
    for b, (n, ctx) in enumerate(zip(c.new, c.ctx)):
        last = 0
        for j in range(1, min(int(accepted[b]), n)):
            p = int(path[b, j])
            rises, last = p > last, p
            if not (j < p < n and rises):
                continue
            src, dst = c.place(b, ctx - n + p), c.place(b, ctx - n + j)
            if src is None or dst is None:
                continue
            (p0, s0), (p1, s1) = src, dst
            K[p1, :, s1], V[p1, :, :, s1] = K[p0, :, s0], V[p0, :, :, s0]
            if KS is not None:
                KS[p1, :, s1], VS[p1, :, s1] = KS[p0, :, s0], VS[p0, :, s0]
    return K, V, KS, VS
