"""The paged cache's operators from their definitions, in float64 NumPy: slow,
plain loops over sequences, rows and heads."""
import math

import numpy as np


class PagedCase:
    """A ragged batch with its pages in shuffled order.  ``new`` and ``ctx`` are the
    new rows and the lengths; ``spare`` pages and ``pad`` rows belong to nobody."""

    def __init__(self, seed, *, new, ctx, page, kv, hd, store="f16", spare=2, pad=0, extra_entries=1):
        self.rng = np.random.default_rng(seed)
        self.new, self.ctx, self.page, self.kv, self.hd, self.store = list(new), list(ctx), page, kv, hd, store
        per = [-(-c // page) for c in self.ctx]
        self.n_pages = sum(per) + spare
        ids = self.rng.permutation(self.n_pages)
        self.stride = max(1, max(per)) + extra_entries
        self.table = np.full((len(ctx), self.stride), -1, np.int32)
        at = 0
        for b, n in enumerate(per):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.cu = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.rows = int(self.cu[-1])
        self.tokens = self.rows + pad
        shape_k, shape_v = (self.n_pages, kv, page, hd), (self.n_pages, kv, hd, page)
        if store == "f16":
            self.k = self.rng.standard_normal(shape_k).astype(np.float16)
            self.v = self.rng.standard_normal(shape_v).astype(np.float16)
            self.k_scale = self.v_scale = None
        else:
            self.k = self.rng.integers(-127, 128, shape_k).astype(np.int8)
            self.v = self.rng.integers(-127, 128, shape_v).astype(np.int8)
            s = (self.n_pages, kv, page)
            self.k_scale = (0.014 * np.exp(0.3 * self.rng.standard_normal(s))).astype(np.float32)
            self.v_scale = (0.014 * np.exp(0.5 * self.rng.standard_normal(s))).astype(np.float32)

    def place(self, b, pos):
        """(page, slot) of a position, or None."""
        e = pos // self.page
        if pos < 0 or e >= self.stride:
            return None
        p = int(self.table[b, e])
        return (p, pos % self.page) if 0 <= p < self.n_pages else None

    def row_places(self):
        """(row, sequence, position, place) of every row of the batch."""
        for b, (n, c) in enumerate(zip(self.new, self.ctx)):
            for j in range(n):
                pos = c - n + j
                yield int(self.cu[b]) + j, b, pos, self.place(b, pos)

    def held(self, b, h, pos):
        """K and V of one position in float64; None where it is in no page."""
        at = self.place(b, pos)
        if at is None:
            return None
        p, s = at
        k, v = self.k[p, h, s].astype(np.float64), self.v[p, h, :, s].astype(np.float64)
        if self.store == "i8":
            with np.errstate(invalid="ignore"):
                k, v = k * float(self.k_scale[p, h, s]), v * float(self.v_scale[p, h, s])
        return k, v


def quantise(x):
    """(ints, scale) of one row head in f32: the exact quotient, ties to even."""
    x = np.asarray(x, np.float32)
    if not np.all(np.isfinite(x)):
        return np.zeros(x.shape, np.int8), np.float32(np.nan)
    amax = np.abs(x).max()
    if amax < 2.0 ** -100:
        return np.zeros(x.shape, np.int8), np.float32(0)
    s = np.float32(np.float64(amax) / 127.0)
    # |x| <= 127 s (1 + 2^-23): 24-bit numbers' quotient in 53 bits keeps its side of every half
    return np.clip(np.rint(x.astype(np.float64) / np.float64(s)), -127, 127).astype(np.int8), s


def append(c, k, v):
    """The pools after rows k, v [tokens, kv, hd] are stored (copies)."""
    K, V = c.k.copy(), c.v.copy()
    KS, VS = (None, None) if c.store == "f16" else (c.k_scale.copy(), c.v_scale.copy())
    for row, _, _, at in c.row_places():
        if at is None:
            continue
        p, s = at
        for h in range(c.kv):
            if c.store == "f16":
                with np.errstate(over="ignore"):
                    K[p, h, s], V[p, h, :, s] = k[row, h].astype(np.float16), v[row, h].astype(np.float16)
            else:
                K[p, h, s], KS[p, h, s] = quantise(k[row, h])
                V[p, h, :, s], VS[p, h, s] = quantise(v[row, h])
    return K, V, KS, VS


def rope_norm(x, gain, pos, *, n_rot, eps, base, factors=None):
    """One head: RMS norm with gain (None: skipped), NeoX rotation of n_rot dims."""
    x = np.asarray(x, np.float64)
    if gain is not None:
        x = x / math.sqrt(float((x * x).mean()) + eps) * np.asarray(gain, np.float64)
    y = x.copy()
    half = n_rot // 2
    for j in range(half):
        a = pos * float(base) ** (-2.0 * j / n_rot) / (float(factors[j]) if factors is not None else 1.0)
        y[j] = x[j] * math.cos(a) - x[j + half] * math.sin(a)
        y[j + half] = x[j] * math.sin(a) + x[j + half] * math.cos(a)
    return y


def attend(c, q, *, heads, window=0, scale=None):
    """(out, weighted |v|, most of sum |q k|, largest |v|) per row and head of q
    [tokens, heads, hd]; rows that see nothing are 0.  The last three are what
    bounds of rounding are made of; the largest |v| is that of the sequence's keys
    (127 scales in 8 bits), as other rows beside a row may see more of them."""
    scale = 1 / math.sqrt(c.hd) if scale is None else scale
    G = heads // c.kv
    out = np.zeros((c.tokens, heads, c.hd))
    mag, prod, vmax = np.zeros_like(out), np.zeros((c.tokens, heads)), np.zeros((c.tokens, heads))
    for b, (n, ctx) in enumerate(zip(c.new, c.ctx)):
        if not n:
            continue
        first = ctx - n
        lo = max(0, first - window + 1) if window else 0
        for h in range(c.kv):
            got = [(p, c.held(b, h, p)) for p in range(lo, ctx)]
            got = [(p, x) for p, x in got if x is not None]
            if not got:
                continue
            P = np.array([p for p, _ in got])
            K, V = np.stack([x[0] for _, x in got]), np.stack([x[1] for _, x in got])
            top = np.abs(V).max()
            if c.store == "i8":
                scales = [c.v_scale[pg, h, sl] for pg, sl in (c.place(b, p) for p, _ in got)]
                top = max(top, 127 * float(np.max(scales)))
            for j in range(n):
                pos = first + j
                on = (P <= pos) & ((P > pos - window) if window else True)
                if not on.any():
                    continue
                r = int(c.cu[b]) + j
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


def attend_bound(c, mag, prod, vmax, keys, *, f32):
    """How far a result may be from the exact one, element by element.

    A score is a sum of head_dim products in fp32, q in 22 bits (f32) or as it
    is: off by at most (hd 2^-24 + 2^-22) prod, twice that between two keys; the
    exponent's own roundings (scale, subtraction, exp2) are below 8 half steps of
    a number below prod + 8.  A weight is so off by the sum of these, relatively;
    f16 rows round weights to 11 bits where chunks are long (2^-11), fp32 sums over
    `keys` keys add keys 2^-24, and a f16 result is rounded by 2^-11 of itself.

    A weight's last f16 part ends at 2^-24: it is off by 2^-25 at most, where the
    row's largest weight is held as 2^10 or more (2^6 where f16 rows round weights
    to one part), so `keys` weights move a result by keys 2^-35 (2^-31) of the
    largest |v|; an 8-bit weight also carries its scale over one that is at most 4
    times the largest, four times that."""
    rel = 2 * (c.hd * 2.0 ** -24 + 2.0 ** -22) * prod + 8 * 2.0 ** -24 * (prod + 8) + (keys + 16) * 2.0 ** -24
    if not f32:
        rel = rel + 2.0 ** -11 + 2.0 ** -11
    floor = keys * (2.0 ** -35 if f32 else 2.0 ** -31) * (4 if c.store == "i8" else 1) * vmax
    # the weights and their sum are both off: twice
    return 2 * rel[..., None] * mag + floor[..., None] + 2.0 ** -24 * (0 if f32 else 1) + 1e-30
