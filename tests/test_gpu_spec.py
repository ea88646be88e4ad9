"""Steps with drafted tokens on the GPU against their definitions (spec_oracle):
pages and row maps, trees, the prologue at positions, attention by masks, the
verification, the keeping, and all of them as one loop."""
import ctypes

import numpy as np
import pytest

from tests import paged_oracle as po
from tests import spec_oracle as so

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import llmoxide_amd as lmx  # noqa: E402
from llmoxide_amd import spec  # noqa: E402
from tests.test_gpu_paged import gpu, on_gpu, rows, say  # noqa: E402


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def trees_of(c, seed, kind="tree"):
    """A tree for each sequence of a PagedCase."""
    rng = np.random.default_rng(seed)
    out = []
    for n in c.new:
        if kind == "chain":
            out.append(np.arange(-1, n - 1))
        else:  # some rows are roots of their own, some parents are no earlier rows
            p = np.array([rng.integers(0, i) if i else -1 for i in range(n)], int)
            if kind == "forest":
                p[rng.random(n) < 0.2] = -1
                bad = rng.random(n) < 0.1
                p[bad] = np.where(rng.random(bad.sum()) < 0.5, n + 3, -9)
                p[1:2] = 1
            out.append(p)
    return out


# ------------------------------------------------------------------- pages --
def plan_case(seed, n_seq, page, most, *, short=False, holes=False):
    """Tables with requests that stay, grow and leave; entries behind `held` hold anything."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, most, n_seq)
    held = -(-lens // page) + rng.integers(0, 3, n_seq)  # some have pages to spare
    entries = int(-(-2 * most // page) + 4)
    new = np.where(rng.random(n_seq) < 0.3, 0, rng.integers(0, most, n_seq))
    left = rng.random(n_seq) < 0.2
    lens, new = np.where(left, 0, lens), np.where(left, 0, new)
    n_pages = int(held.sum() + (3 if short else -(-(lens + new) // page).sum()) + 5)
    ids = rng.permutation(n_pages).astype(np.int32)
    table = rng.integers(-5, 1 << 30, (n_seq, entries)).astype(np.int32)
    at = 0
    for b in range(n_seq):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
        if holes and held[b] > 1:
            table[b, rng.integers(0, held[b])] = rng.choice([-1, -100, n_pages, 1 << 30])
    free = rng.integers(-5, 1 << 30, n_pages).astype(np.int32)
    free[:n_pages - at] = ids[at:]
    return dict(lens=lens, new=new, table=table, held=held.astype(np.int32), free=free,
                n_free=np.array([n_pages - at, 7], np.int32), n_pages=n_pages)


@pytest.mark.parametrize("n_seq,page,most", [(1, 16, 1), (1, 16, 300), (3, 32, 40), (64, 16, 200), (65, 64, 90),
                                             (1024, 16, 20), (2500, 128, 40), (7, 256, 3000)])
@pytest.mark.parametrize("trim", [False, True])
@pytest.mark.parametrize("how", ["", "short", "holes"])
def test_plan(n_seq, page, most, trim, how):
    say("plan", n_seq, page, most, trim, how)
    c = plan_case(n_seq + most, n_seq, page, most, short=how == "short", holes=how == "holes")
    for extra in (0, 3, 5000):  # rows mapped by either kernel, some of nobody
        n = int(c["new"].sum()) + extra
        if n == 0:
            continue
        t = lmx.PageTables(ints(c["table"]), ints(c["held"]), ints(c["free"]), ints(c["n_free"]), page_size=page)
        got = lmx.spec_plan(t, ints(c["lens"]), ints(c["new"]), n_tokens=n, trim=trim)
        want = so.plan(c["lens"], c["new"], c["table"], c["held"], c["free"], c["n_free"], page=page, n_tokens=n,
                       n_pages=c["n_pages"], trim=trim)
        names = "table held free n_free cu ctx slots pos".split()
        for name, g, w in zip(names, (t.page_table, t.held, t.free_pages, t.n_free, *got), want):
            assert np.array_equal(g.cpu().numpy(), w), name


def test_a_plan_that_is_withdrawn_leaves_everything_as_it_was():
    c = plan_case(5, 40, 16, 300)
    keep = -(-c["lens"] // 16)
    for b in range(40):  # requests hold what their lengths need
        c["table"][b, keep[b]:] = -1
    c["held"] = keep.astype(np.int32)
    n = int(c["new"].sum())
    t = lmx.PageTables(ints(c["table"]), ints(c["held"]), ints(c["free"]), ints(c["n_free"]), page_size=16)
    free = int(c["n_free"][0])
    for _ in range(3):
        lmx.spec_plan(t, ints(c["lens"]), ints(c["new"]), n_tokens=n, trim=True)
        lmx.spec_plan(t, ints(c["lens"]), ints(np.zeros(40)), n_tokens=n, trim=True)
        assert np.array_equal(t.page_table.cpu().numpy(), c["table"]) and np.array_equal(t.held.cpu().numpy(), c["held"])
        assert t.n_free.tolist() == [free, 0]
        assert np.array_equal(t.free_pages.cpu().numpy()[:free], c["free"][:free])


def test_a_plan_without_maps_and_lengths_out_of_range():
    t = lmx.PageTables.empty(6, page_size=16, n_seq=4, entries=3)
    out = lmx.StepPlan.empty(t, n_tokens=1, rows=False)
    # negative lengths are 0, one beyond the table ends there
    got = lmx.spec_plan(t, ints([-5, 40, 0, 0]), ints([3, 100, -2, 0]), n_tokens=200, out=out)
    assert got.cu.tolist() == [0, 3, 103, 103, 103] and got.ctx_lens.tolist() == [3, 48, 0, 0]
    assert t.held.tolist() == [1, 3, 0, 0] and t.n_free.tolist() == [2, 0]
    got = lmx.spec_plan(t, ints([-5, 40, 0, 0]), ints([3, 100, -2, 0]), n_tokens=200)
    slots = got.slots.cpu().numpy()
    assert np.all(slots[3:11] >= 0) and np.all(slots[11:] == -1) and np.all(slots[:3] >= 0)
    # counts that no list has: forced into range
    t.held.fill_(1 << 30)
    t.n_free.copy_(ints([1 << 30, 0]))
    lmx.spec_plan(t, ints([2147483647] * 4), ints([2147483647] * 4), n_tokens=64, trim=True)
    t.held.fill_(-(1 << 30))
    t.n_free.copy_(ints([-3, 0]))
    lmx.spec_plan(t, ints([2147483647] * 4), ints([2147483647] * 4), n_tokens=64)
    assert t.n_free.tolist() == [0, 12]


# ------------------------------------------------------------------- trees --
@pytest.mark.parametrize("new", [[1], [64, 0, 65, 3], [17, 128, 2], [1024], [300, 1, 700]])
@pytest.mark.parametrize("kind", ["tree", "chain", "forest"])
@pytest.mark.parametrize("window", [0, 1, 5])
def test_tree(new, kind, window):
    say("tree", new, kind, window)
    c = po.PagedCase(1, new=new, ctx=[n + 9 * b for b, n in enumerate(new)], page=16, kv=1, hd=64, pad=3)
    _, batch = on_gpu(c)
    trees = trees_of(c, 2, kind)
    parent = ints(np.concatenate(trees + [np.full(3, 5)]))
    words = -(-max(new) // 64)
    for w in {words, 16}:
        out = spec.SpecTree(ints(np.full(c.tokens, 77)), torch.full((c.tokens, w), 77, dtype=torch.int64, device="cuda"))
        lmx.spec_tree(parent, batch, window=window, out=out)
        pos, seen = np.full(c.tokens, 77), np.full((c.tokens, w), 77)
        for b, t in enumerate(trees):
            depth, sees = so.tree(t, window)
            at = slice(int(c.cu[b]), int(c.cu[b + 1]))
            pos[at], seen[at] = c.ctx[b] - c.new[b] + depth, so.words_of(sees, w)
        assert np.array_equal(out.pos.cpu().numpy(), pos) and np.array_equal(out.seen.cpu().numpy(), seen)
    got = lmx.spec_tree(parent, batch, window=window)
    assert got.seen.shape == (c.tokens, words) and torch.equal(got.pos[:c.rows], out.pos[:c.rows])


# ----------------------------------------------------------------- prologue --
PROLOGUES = [
    (64, 64, 16, 2, 6, "f16"), (128, 128, 32, 2, 8, "f16"), (128, 128, 16, 1, 5, "i8"), (128, 48, 64, 2, 2, "f16"),
    (256, 64, 16, 1, 2, "i8"), (256, 256, 32, 2, 4, "f16"), (512, 510, 16, 1, 2, "f16"), (64, 0, 16, 1, 1, "f16"),
    (128, 6, 16, 1, 2, "f16"), (64, 2, 16, 1, 1, "i8"),
]


@pytest.mark.parametrize("hd,n_rot,page,kv,heads,store", PROLOGUES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("new", [[3, 0, 1], [3, 0, 37, 1]])  # a row in a few lanes, blocks of rows
@pytest.mark.parametrize("q16", [False, True])
def test_prologue(hd, n_rot, page, kv, heads, store, interleaved, new, q16):
    say("prologue", hd, n_rot, page, kv, heads, store, interleaved, new, q16)
    c = po.PagedCase(11, new=new, ctx=[3, 9, 500, 1200][:len(new)], page=page, kv=kv, hd=hd, store=store, pad=2)
    q, k, v = rows(c, 12, heads, 2.0), rows(c, 13, kv, 0.3), rows(c, 14, kv)
    rng = np.random.default_rng(15)
    qg, kg = (1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32)
    factors = (1 + rng.random(max(1, n_rot // 2))).astype(np.float32) if n_rot in (48, 128) else None
    gains, turn_scale = hd != 64, 1.0 if n_rot == 64 else 1.25
    pos = rng.integers(0, 1 << 20, c.tokens).astype(np.int32)
    pos[:2] = 0, (1 << 31) - 1
    cache, batch = on_gpu(c)
    fused = torch.cat([gpu(x.reshape(c.tokens, -1)) for x in (q, k, v)], 1)
    nq, nk = heads * hd, kv * hd
    out = torch.full((c.tokens, nq), 9.0, dtype=torch.float16 if q16 else torch.float32, device="cuda")
    eps, base = 1e-6, 5e5
    lmx.spec_prologue(fused[:, :nq], fused[:, nq:nq + nk], fused[:, nq + nk:], cache, batch, pos=gpu(pos),
                      n_heads=heads, n_rot=n_rot, interleaved=interleaved, turn_scale=turn_scale, v_norm=hd == 256,
                      rms_eps=eps, rope_base=base, q_gain=gpu(qg) if gains else None, k_gain=gpu(kg) if gains else None,
                      rope_factors=None if factors is None else gpu(factors), q_out=out)
    kw = dict(eps=eps, base=base, factors=factors, interleaved=interleaved, turn_scale=turn_scale)
    one = np.ones(hd) if hd == 256 else None
    want_q, want = np.full((c.tokens, heads, hd), 9.0), {}
    for row, b, _, at in c.row_places():
        for h in range(heads):
            want_q[row, h] = so.turned(q[row, h], qg if gains else None, int(pos[row]), n_rot=n_rot, **kw)
        for h in range(kv):
            want[at, h] = (so.turned(k[row, h], kg if gains else None, int(pos[row]), n_rot=n_rot, **kw),
                           so.turned(v[row, h], one, 0, n_rot=0, **kw))
    # f32 steps as in the prologue at slots, one more for turn_scale; the angle of position 2^31 is off by
    # 2^31 2^-50 in its double steps (the power of the base, its product, the factor)
    far = 2.0 ** -17 * (pos > 1 << 30)[:, None, None]
    rel = (hd + 34) * 2.0 ** -24 + far
    big = np.abs(want_q).max(-1, keepdims=True)
    got = out.float().cpu().numpy().reshape(c.tokens, heads, hd)
    own = np.zeros(c.tokens, bool)
    own[[r for r, *_ in c.row_places()]] = True
    assert np.all(got[~own] == 9)
    assert np.all(np.abs(got - want_q) <= 2 * rel * big * max(1, turn_scale) + (2.0 ** -11 * np.abs(want_q) + 2.0 ** -24 if q16 else 0))
    K, V = cache.k.float().cpu().numpy(), cache.v.float().cpu().numpy()
    touched = np.zeros((c.n_pages, c.page), bool)
    for row, _, _, (p, s) in c.row_places():
        touched[p, s] = True
        r = float(np.broadcast_to(rel, (c.tokens, 1, 1))[row, 0, 0]) * max(1, turn_scale)
        for h in range(kv):
            for got1, w, scale in zip((K[p, h, s], V[p, h, :, s]), want[(p, s), h], (cache.k_scale, cache.v_scale)):
                m = np.abs(w).max()
                if store == "f16":
                    assert np.all(np.abs(got1 - w) <= 2 * r * m + 2.0 ** -11 * np.abs(w) + 2.0 ** -24)
                else:  # half a step of the scale, and the f32 steps before it
                    sc = float(scale[p, h, s])
                    assert abs(sc - m / 127) <= 4 * r * m / 127
                    assert np.all(np.abs(got1 * sc - w) <= (0.5 + 1e-3) * sc + 4 * r * m)
    assert np.array_equal(cache.k.cpu().numpy()[~touched.any(1)], c.k[~touched.any(1)])
    assert np.array_equal(cache.v.cpu().numpy()[~touched.any(1)], c.v[~touched.any(1)])


@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("new", [[3, 1], [33, 1]])
def test_prologue_at_the_slots_positions_is_the_paged_one(store, new):
    c = po.PagedCase(16, new=new, ctx=[200, 300], page=16, kv=2, hd=128, store=store)
    q, k, v = (gpu(rows(c, s, h).reshape(c.tokens, -1)) for s, h in ((17, 4), (18, 2), (19, 2)))
    gain = gpu((1 + 0.1 * np.random.default_rng(1).standard_normal(128)).astype(np.float32))
    slots = ints([p for _, _, p, _ in c.row_places()])
    results = []
    for call, kw in ((lmx.paged_prologue, {}), (lmx.spec_prologue, {}), (lmx.spec_prologue, dict(pos=slots))):
        cache, batch = on_gpu(c)
        out = call(q, k, v, cache, batch, n_heads=4, q_gain=gain, k_gain=gain, **kw)
        results.append([out, cache.k, cache.v] + ([cache.k_scale, cache.v_scale] if store == "i8" else []))
    for other in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(results[0], other))


# ---------------------------------------------------------------- attention --
def check(c, heads, sees, *, q16, window=0, pos=None, seed=21, q_scale=1.0, extra_words=0, ws=None, scale=None):
    """spec_attention of case ``c`` under boolean matrices ``sees``, against the oracle."""
    cache, batch = on_gpu(c)
    q = rows(c, seed, heads, q_scale)
    if q16:
        q = q.astype(np.float16).astype(np.float32)
    dt = torch.float16 if q16 else torch.float32
    words = -(-max(c.new) // 64) + extra_words
    seen = np.full((c.tokens, words), -1, np.int64)
    for b, m in enumerate(sees):
        if c.new[b]:
            seen[int(c.cu[b]):int(c.cu[b + 1])] = so.words_of(m, words)
    out = torch.full((c.tokens, heads * c.hd), 5.0, dtype=dt, device="cuda")
    lmx.spec_attention(gpu(q.reshape(c.tokens, -1)).to(dt), cache, batch, gpu(seen), n_heads=heads, window=window,
                       pos=None if pos is None else ints(pos), out=out, workspace=ws, scale=scale)
    got = out.float().cpu().numpy().reshape(c.tokens, heads, c.hd).astype(np.float64)
    want, mag, prod, top = so.attend(c, q, sees, heads=heads, window=window, pos=pos, scale=scale)
    own = np.zeros(c.tokens, bool)
    own[[r for r, *_ in c.row_places()]] = True
    assert np.all(got[~own] == 5), "rows of no sequence were written"
    bound = po.attend_bound(c, mag, prod, top, max(c.ctx), f32=not q16)
    assert np.all(np.isfinite(got[own])), "non-finite"
    off = np.abs(got - want) - bound
    assert off[own].max() <= 0, f"{off[own].max():.3g} over the bound {bound[own].max():.3g}"
    return got


def masks(c, seed, kind):
    """Sight of each sequence's rows; "any": bits at random, some rows none at all."""
    if kind != "any":
        return [so.tree(t)[1] for t in trees_of(c, seed, kind)]
    rng = np.random.default_rng(seed)
    out = []
    for n in c.new:
        m = rng.random((n, n)) < rng.choice([0.05, 0.5, 0.95], (n, 1))
        m[rng.random(n) < 0.2] = False
        out.append(m)
    return out


LENS = [
    dict(new=[1], ctx=[1]), dict(new=[6], ctx=[518]), dict(new=[5, 0, 33, 1], ctx=[5, 20, 70, 64], pad=3),
    dict(new=[64, 7], ctx=[131, 7], pad=1), dict(new=[130, 2], ctx=[300, 40]), dict(new=[33, 16], ctx=[2000, 900]),
]


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("hd,page,kv,heads", [(64, 16, 2, 6), (128, 16, 2, 8), (128, 64, 1, 1), (256, 32, 1, 4),
                                              (512, 16, 1, 3), (128, 256, 2, 10)])
@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("q16", [False, True])
def test_attention(lens, hd, page, kv, heads, store, q16):
    say("tree attention", lens, hd, page, kv, heads, store, q16)
    c = po.PagedCase(20, page=page, kv=kv, hd=hd, store=store, **lens)
    kind = {64: "tree", 128: "any", 256: "forest", 512: "any"}[hd]
    check(c, heads, masks(c, 3, kind), q16=q16, extra_words=hd == 256)


@pytest.mark.parametrize("window", [1, 7, 64, 150])
@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("hd,q16", [(128, True), (128, False), (256, True), (512, False)])
def test_attention_windows(window, store, hd, q16):
    """Prefixes cut by position, rows by what their masks leave of the ancestors."""
    say("tree window", window, store, hd, q16)
    c = po.PagedCase(22, new=[1, 100, 40, 3], ctx=[400, 100, 333, 3], page=32, kv=2, hd=hd, store=store, pad=2)
    trees = trees_of(c, 4)
    depth = np.concatenate([so.tree(t)[0] for t in trees] + [np.full(2, -99)])
    first = np.concatenate([np.full(n, k - n) for n, k in zip(c.new, c.ctx)] + [np.zeros(2, int)])
    check(c, 4, [so.tree(t, window)[1] for t in trees], q16=q16, window=window, pos=first + depth)


@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("q16", [False, True])
def test_attention_of_many_rows(store, hd, q16):
    """Masks of several words: rows see each other across tiles and words."""
    say("tree many rows", store, hd, q16)
    c = po.PagedCase(23, new=[200, 3, 129], ctx=[1300, 700, 129], page=32, kv=1, hd=hd, store=store, pad=2)
    check(c, 3, masks(c, 5, "any"), q16=q16, extra_words=2)


@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("q16", [False, True])
@pytest.mark.parametrize("new", [[3, 1, 2], [60, 130, 4]])
def test_attention_without_some_pages(store, q16, new):
    c = po.PagedCase(25, new=new, ctx=[200, 260, 4], page=16, kv=2, hd=128, store=store)
    c.table[0, 2] = -1
    c.table[0, 5] = c.n_pages
    c.table[0, 11] = -1  # some of the rows' own
    c.table[1, :9] = -7
    c.table[2, 0] = 1 << 30
    got = check(c, 4, masks(c, 6, "any"), q16=q16)
    assert np.all(got[int(c.cu[2]):int(c.cu[3])] == 0)


def test_attention_of_rows_that_see_nothing():
    """No prefix and no bits: zeros, whatever the pages hold."""
    for n in (2, 100):
        c = po.PagedCase(26, new=[n], ctx=[n], page=16, kv=1, hd=64)
        c.v[:] = np.inf
        c.k[:] = np.nan
        got = check(c, 2, [np.zeros((n, n), bool)], q16=True)
        assert np.all(got == 0)


@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("hd,new", [(128, [5, 9]), (64, [90, 40]), (256, [60, 1]), (512, [40, 20])])
@pytest.mark.parametrize("q16", [False, True])
def test_what_a_row_does_not_see_has_no_part_in_it(store, hd, new, q16):
    """Infinities and NaN in rows that some see and some do not: the others keep
    their results, bit for bit, and who sees one has what the formula gives."""
    say("tree unseen", store, hd, new, q16)
    c = po.PagedCase(27, new=new, ctx=[300, 170], page=16, kv=1, hd=hd, store=store, spare=3)
    sees = masks(c, 7, "tree")
    heads = 2
    clean = check(c, heads, sees, q16=q16)
    bad = [min(4, n - 1) for n in new]  # this row of each request
    for b, j in enumerate(bad):
        p, s = c.place(b, c.ctx[b] - new[b] + j)
        if store == "f16":
            c.k[p, 0, s, 3], c.v[p, 0, 5, s] = np.nan, np.inf
        else:
            c.k_scale[p, 0, s] = np.nan
    # pages of nobody and slots behind the lengths
    used = {c.place(b, p) for b in range(2) for p in range(c.ctx[b])}
    for p in range(c.n_pages):
        for s in range(c.page):
            if (p, s) not in used:
                if store == "f16":
                    c.k[p, :, s], c.v[p, :, :, s] = np.nan, np.inf
                else:
                    c.k_scale[p, :, s] = c.v_scale[p, :, s] = np.nan
    cache, batch = on_gpu(c)
    q = rows(c, 21, heads)
    dt = torch.float16 if q16 else torch.float32
    seen = np.concatenate([so.words_of(m, -(-max(new) // 64)) for m in sees])
    got = lmx.spec_attention(gpu(q.reshape(c.tokens, -1)).to(dt), cache, batch, gpu(seen), n_heads=heads)
    got = got.float().cpu().numpy().reshape(clean.shape)
    for b, j in enumerate(bad):
        for i in range(new[b]):
            r = int(c.cu[b]) + i
            if sees[b][i, j]:
                assert np.isnan(got[r]).all()  # a NaN score
            else:
                assert np.array_equal(got[r], clean[r])


@pytest.mark.parametrize("new", [[7, 3], [80, 50]])
def test_infinite_values_reach_the_rows_that_see_them(new):
    c = po.PagedCase(28, new=new, ctx=[200, 90], page=16, kv=1, hd=128)
    sees = masks(c, 8, "tree")
    for b in range(2):
        p, s = c.place(b, c.ctx[b] - new[b] + 1)
        c.v[p, 0, 7, s] = -np.inf
    cache, batch = on_gpu(c)
    for dt in (torch.float16, torch.float32):
        q = gpu(rows(c, 21, 2).reshape(c.tokens, -1)).to(dt)
        seen = np.concatenate([so.words_of(m, -(-max(new) // 64)) for m in sees])
        got = lmx.spec_attention(q, cache, batch, gpu(seen), n_heads=2).float().cpu().numpy().reshape(c.tokens, 2, 128)
        for b in range(2):
            for i in range(new[b]):
                r = int(c.cu[b]) + i
                rest = np.delete(got[r], 7, 1)
                assert np.isfinite(rest).all()
                assert (got[r][:, 7] == -np.inf).all() if sees[b][i, 1] else np.isfinite(got[r][:, 7]).all()


@pytest.mark.parametrize("new", [[1, 1, 1], [4, 30, 1], [150, 3, 20]])
@pytest.mark.parametrize("store", ["f16", "i8"])
def test_a_chain_is_causal_attention(new, store):
    """Against lmxp_attn on the same inputs: the same formula, off by both bounds at most."""
    c = po.PagedCase(29, new=new, ctx=[300, 70, 900], page=32, kv=2, hd=128, store=store)
    sees = masks(c, 1, "chain")
    got = check(c, 8, sees, q16=False, seed=30)
    cache, batch = on_gpu(c)
    q = rows(c, 30, 8)
    want = lmx.paged_attention(gpu(q.reshape(c.tokens, -1)), cache, batch, n_heads=8).cpu().numpy().reshape(got.shape)
    _, mag, prod, top = so.attend(c, q, sees, heads=8)
    assert np.all(np.abs(got - want) <= 2 * po.attend_bound(c, mag, prod, top, 900, f32=True))


def test_attention_strides_streams_and_workspace():
    c = po.PagedCase(31, new=[9, 1], ctx=[900, 70], page=16, kv=2, hd=128)
    sees = masks(c, 9, "tree")
    cache, batch = on_gpu(c)
    seen = gpu(np.concatenate([so.words_of(m, 1) for m in sees]))
    q = gpu(rows(c, 32, 4)).half()
    want = lmx.spec_attention(q.view(c.tokens, -1), cache, batch, seen, n_heads=4)
    wide = torch.full((c.tokens, 4 * 256 + 8), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, :1024].view(c.tokens, 4, 256)[:, :, :128] = q
    side, ws = torch.cuda.Stream(), lmx.Workspace()
    side.wait_stream(torch.cuda.current_stream())
    got = lmx.spec_attention(wide[:, :1024], cache, batch, seen, n_heads=4, q_head_stride=256, workspace=ws, stream=side)
    side.synchronize()
    assert torch.equal(got, want)


# ------------------------------------------------------------ verification --
def verify_case(seed, new, vocab, kind, drafts, dt=np.float32, pad=0):
    rng = np.random.default_rng(seed)
    trees = []
    for n in new:
        trees.append(np.arange(-1, n - 1) if kind == "chain" else
                     np.array([-1] + [int(rng.integers(max(0, i - 4), i)) for i in range(1, n)][:max(0, n - 1)])[:n])
    tokens = sum(new) + pad
    x = rng.standard_normal((tokens, vocab)) * 2
    e = np.exp(x - x.max(1, keepdims=True))
    p = (e / e.sum(1, keepdims=True)).astype(dt)
    p[rng.random(p.shape) < 0.1] = 0
    y = np.exp(x * 0.7 + rng.standard_normal(x.shape) * 0.5)
    q = (y / y.sum(1, keepdims=True)).astype(dt) if drafts == "sampled" else None
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    tok = rng.integers(0, vocab, tokens).astype(np.int32)
    for b, t in enumerate(trees):
        for i in range(1, len(t)):
            if t[i] < 0:
                continue
            row = int(cu[b]) + int(t[i])
            # likely tokens, sometimes a sibling's once more
            tok[cu[b] + i] = rng.choice(np.argsort(-p[row].astype(np.float32))[:min(vocab, 3)])
    u, r = rng.random(tokens).astype(np.float32), rng.random(len(new)).astype(np.float32)
    return dict(new=new, trees=trees, p=p, q=q, cu=cu, tok=tok, u=u, r=r, kind=kind)


def check_verify(c, *, greedy=False, views=False, ws=None):
    n_seq, most = len(c["new"]), max(max(c["new"]), 1)
    tokens, vocab = c["p"].shape
    parent = np.concatenate([*c["trees"], np.zeros(tokens - sum(c["new"]))])
    p, q = gpu(c["p"]), None if c["q"] is None else gpu(c["q"])
    if views:  # columns of wider rows
        def wide(x, by):
            y = torch.full((tokens, vocab + by), float("nan"), dtype=x.dtype, device="cuda")
            y[:, by - 1:by - 1 + vocab] = x
            return y[:, by - 1:by - 1 + vocab]
        p, q = wide(p, 3), None if q is None else wide(q, 6)
    lens = ints(np.arange(n_seq) * 10)
    out = spec.Verified(ints(np.full((n_seq, most), 55)), ints(np.full(n_seq, 55)), ints(np.full(n_seq, 55)))
    lmx.spec_verify(p, gpu(c["tok"]), None if greedy else gpu(c["u"]), None if greedy else gpu(c["r"]), gpu(c["cu"]),
                    max_new=most, parent=None if c["kind"] == "chain" else ints(parent), q=q, lens=lens, greedy=greedy,
                    out=out, workspace=ws)
    path, accepted, token = (x.cpu().numpy() for x in out)
    for b, n in enumerate(c["new"]):
        at = slice(int(c["cu"][b]), int(c["cu"][b + 1]))
        want, t = so.verify(c["p"][at], c["tok"][at], c["u"][at], c["r"][b], c["trees"][b],
                            None if c["q"] is None else c["q"][at], greedy)
        assert accepted[b] == len(want) and path[b].tolist() == want + [-1] * (most - len(want)), (b, path[b], want)
        assert token[b] == t, (b, token[b], t)
        assert lens[b] == 10 * b + len(want)
    return path, accepted, token


@pytest.mark.parametrize("new,vocab", [([1], 1), ([5], 7), ([4, 0, 9, 1], 31), ([33, 64, 2], 4096), ([70, 3], 4097),
                                       ([6] * 40, 100), ([8, 5], 20011), ([12], 131072),
                                       ([3, 0, 9], 32768), ([33, 1, 20], 32769), ([4] * 20, 40000)])
@pytest.mark.parametrize("kind", ["chain", "tree"])
@pytest.mark.parametrize("drafts", ["best", "sampled"])
@pytest.mark.parametrize("dt", [np.float32, np.float16])
def test_verify(new, vocab, kind, drafts, dt):
    say("verify", new, vocab, kind, drafts, dt.__name__)
    for seed in range(3):
        c = verify_case(100 * seed + vocab, new, vocab, kind, drafts, dt, pad=2)
        check_verify(c, views=seed == 1)
        if drafts == "best":
            check_verify(c, greedy=True, views=seed == 1)


@pytest.mark.parametrize("drafts", ["best", "sampled"])
@pytest.mark.parametrize("vocab", [50, 33000])  # one workgroup a request, and many
def test_verify_siblings(drafts, vocab):
    """All rows are children of the root: refusals one after another, tokens that come
    twice, tokens that are none, draws of 0 and just below 1."""
    for seed in range(6):
        c = verify_case(seed, [40, 1000 if vocab == 50 else 70, 3], vocab, "tree", drafts)
        c["trees"] = [np.array([-1] + [0] * (n - 1)) for n in c["new"]]
        c["u"][:] = np.where(np.random.default_rng(seed).random(c["u"].shape) < 0.9, np.float32(1 - 2 ** -24), 0.3)
        c["tok"][::7] = -1
        c["tok"][3::11] = vocab
        c["tok"][5::13] = 1 << 30
        c["r"][:] = [0, 1 - 2 ** -24, 0.5]
        check_verify(c)


@pytest.mark.parametrize("vocab", [9000, 40000])
def test_verify_of_rows_with_nothing_left(vocab):
    """Refused drafts that had all of p, rows of zeros, negative, infinite and NaN entries."""
    c = verify_case(3, [4, 3, 2, 2, 3], vocab, "tree", "best")
    c["trees"] = [np.array([-1] + [0] * (n - 1)) for n in c["new"]]
    p = c["p"]
    p[:] = 0
    p[0, 4000], p[0, 8000] = 0.25, 0.75        # both drafted and refused: the token is p's own
    c["tok"][1:4] = 4000, 8000, 4000
    p[4, 17], p[4, 8999] = np.nan, 1.0         # entries that are no probability count as 0
    p[4, 18], p[4, 19] = -3.0, np.inf
    c["tok"][5:7] = 17, 19
    p[7] = 0                                    # nothing at all: no token
    p[9, 5] = 1e-38                             # tiny ones are something
    p[11, 3] = p[11, 4] = 0.5
    c["tok"][12:14] = 3, 3
    c["u"][:] = 1 - 2 ** -24
    c["u"][1:4] = 1 - 2 ** -24
    _, accepted, token = check_verify(c)
    assert token[1] == 8999 and token[2] == -1
    for r in (0.0, 0.2, 0.3, 0.999):
        c["r"][:] = r
        check_verify(c)


def test_verify_greedy_of_logits():
    """Largest scores: ties, infinities, rows of NaN."""
    c = verify_case(4, [3, 3, 3, 3], 5000, "chain", "best")
    p = c["p"]
    p[:] = np.random.default_rng(1).standard_normal(p.shape)
    p[0, [4999, 31, 4097]] = 9      # the lowest of equals
    p[3] = np.nan
    p[6] = -np.inf
    p[9, 77], p[9, 78] = np.nan, np.inf
    c["tok"][[1, 4, 7, 10]] = 31, 0, 0, 78
    path, accepted, token = check_verify(c, greedy=True)
    assert accepted.tolist()[0] >= 2 and token[1] == -1 and accepted[1] == 1 and accepted[2] >= 2


@pytest.mark.parametrize("vocab", [100, 40000])
def test_verify_of_rows_out_of_range(vocab):
    """Offsets that name rows beyond the batch, and more rows than max_new: in bounds."""
    c = verify_case(5, [4, 4], vocab, "chain", "best")
    out = lmx.spec_verify(gpu(c["p"]), gpu(c["tok"]), gpu(c["u"]), gpu(c["r"]), ints([-3, 1 << 30, 2]), max_new=2)
    assert out.path.shape == (2, 2) and out.accepted.tolist()[1] == 0


# -------------------------------------------------------------------- keep --
@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("hd,page,kv", [(64, 16, 3), (128, 32, 2), (256, 64, 1), (512, 16, 2), (128, 256, 8)])
@pytest.mark.parametrize("layers", [1, 3, 70])
def test_keep(store, hd, page, kv, layers):
    say("keep", store, hd, page, kv, layers)
    new = [1, 5, 0, 40, 200, 64]
    c = po.PagedCase(40, new=new, ctx=[9, 5, 0, 100, 300, 77], page=page, kv=kv, hd=hd, store=store, pad=1)
    c.table[5, 77 // page] = -1 if page < 64 else c.table[5, 77 // page]  # some rows in no page
    rng = np.random.default_rng(41)
    path = np.full((6, 210), -1, np.int32)
    accepted = np.zeros(6, np.int32)
    for b, n in enumerate(new):
        if n:
            accepted[b] = n if b == 3 else rng.integers(1, n + 1)
            path[b, 0] = 0
            path[b, 1:accepted[b]] = 1 + np.sort(rng.permutation(n - 1)[:accepted[b] - 1])
    cache, batch = on_gpu(c)
    # the layers are the case's pools, turned by a page each
    parts = [None if x is None else [np.roll(x, i, 0) for i in range(layers)] for x in (c.k, c.v, c.k_scale, c.v_scale)]
    caches = [lmx.PagedCache(*(None if x is None else gpu(x[i]) for x in parts)) for i in range(layers)]
    lmx.spec_keep(caches, batch, gpu(path), gpu(accepted))
    for i, cache in enumerate(caches):
        if layers > 3 and i not in (0, 1, 63, 64, 69):
            continue
        want = so.keep(c, path, accepted, [None if x is None else x[i] for x in parts])
        for got, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):
            if w is not None:
                assert np.array_equal(got.cpu().numpy(), w)


def test_keep_of_paths_that_break_the_rules():
    """Entries that fall, repeat, lie before their place or name no row: not moved."""
    c = po.PagedCase(42, new=[8, 8], ctx=[20, 8], page=16, kv=1, hd=64)
    path = np.array([[0, 3, 3, 2, 6, 99, -1, 7], [0, -4, 1, 8, 1 << 30, 7, 6, 5]], np.int32)
    accepted = np.array([8, 1 << 30], np.int32)
    cache, batch = on_gpu(c)
    lmx.spec_keep([cache], batch, gpu(path), gpu(accepted))
    k, v = cache.k.cpu().numpy(), cache.v.cpu().numpy()
    own = {c.place(b, p) for b in range(2) for p in range(c.ctx[b] - 8, c.ctx[b])}
    for p in range(c.n_pages):
        for s in range(c.page):
            if (p, s) not in own:
                assert np.array_equal(k[p, :, s], c.k[p, :, s]) and np.array_equal(v[p, :, :, s], c.v[p, :, :, s])


# ------------------------------------------------------------ all together --
class Loop:
    """A small model's steps: two layers, rows whose q, k and v follow from the token
    and the position alone (so that a cache is what its tokens say)."""
    heads, kv, hd, page, vocab, n_seq, entries = 4, 2, 64, 16, 97, 3, 16

    def __init__(self, store):
        torch.manual_seed(3)
        dt = torch.float16 if store == "f16" else torch.int8
        n_pages = 40
        self.caches = [lmx.PagedCache.empty(n_pages, page_size=self.page, n_kv_heads=self.kv, head_dim=self.hd, dtype=dt)
                       for _ in range(2)]
        for c in self.caches:  # pages need no clearing
            for x in (c.k, c.v, c.k_scale, c.v_scale):
                if x is not None:
                    x.fill_(float("nan") if x.is_floating_point() else 100)
        self.tables = lmx.PageTables.empty(n_pages, page_size=self.page, n_seq=self.n_seq, entries=self.entries)
        width = (self.heads + 2 * self.kv) * self.hd
        self.rows = [torch.randn(self.vocab, width, device="cuda") for _ in range(2)]
        self.head = torch.randn(2 * self.heads * self.hd, self.vocab, device="cuda") * 0.6
        self.T, self.most = 40, 14
        self.step = lmx.StepPlan.empty(self.tables, n_tokens=self.T)
        self.batch = lmx.PagedBatch(self.step.cu, self.step.ctx_lens, self.tables.page_table, n_tokens=self.T,
                                    max_new=self.most, max_ctx=self.entries * self.page)
        self.lens, self.new = ints([0] * 3), ints([0] * 3)
        self.tokens, self.parent = ints([0] * self.T), ints([-1] * self.T)
        self.u, self.r = torch.zeros(self.T, device="cuda"), torch.zeros(3, device="cuda")
        self.tree = spec.SpecTree(ints([0] * self.T), torch.zeros(self.T, 1, dtype=torch.int64, device="cuda"))
        self.ws, self.ws2 = lmx.Workspace(1 << 22), lmx.Workspace(1 << 16)
        self.p = torch.zeros(self.T, self.vocab, device="cuda")
        self.attn = [torch.zeros(self.T, self.heads * self.hd, device="cuda") for _ in range(2)]
        self.q = torch.zeros(self.T, self.heads * self.hd, device="cuda")
        self.got = spec.Verified(ints(np.zeros((3, self.most))), ints([0] * 3), ints([0] * 3))

    def prefill(self, texts):
        """All but the last token of each text into the cache, ten at a time."""
        done = [0] * 3
        while any(d < len(t) - 1 for d, t in zip(done, texts)):
            parts = [t[d:len(t) - 1][:10] for d, t in zip(done, texts)]
            self.load([(p, np.arange(-1, len(p) - 1)) for p in parts], np.random.default_rng(0))
            lmx.spec_plan(self.tables, self.lens, self.new, out=self.step)
            self.layers()
            self.lens.add_(self.new)
            done = [d + len(p) for d, p in zip(done, parts)]

    def layers(self):
        nq, nk = self.heads * self.hd, self.kv * self.hd
        lmx.spec_tree(self.parent, self.batch, out=self.tree)
        for cache, rows_, attn in zip(self.caches, self.rows, self.attn):
            x = rows_[self.tokens.long()]
            lmx.spec_prologue(x[:, :nq], x[:, nq:nq + nk], x[:, nq + nk:], cache, self.batch, n_heads=self.heads,
                              pos=self.tree.pos, q_out=self.q)
            lmx.spec_attention(self.q, cache, self.batch, self.tree.seen, n_heads=self.heads, out=attn, workspace=self.ws)

    def run(self):
        """One step over what lens, new, tokens and parent hold."""
        lmx.spec_plan(self.tables, self.lens, self.new, out=self.step, trim=True)
        self.layers()
        torch.softmax(torch.cat(self.attn, 1) @ self.head, 1, out=self.p)
        lmx.spec_verify(self.p, self.tokens, self.u, self.r, self.step.cu, max_new=self.most, parent=self.parent,
                        lens=self.lens, greedy=True, out=self.got, workspace=self.ws2)
        lmx.spec_keep(self.caches, self.batch, self.got.path, self.got.accepted)

    def load(self, trees, rng):
        """Rows of a step: per request (tokens, parents)."""
        tok, par = np.zeros(self.T, np.int32), np.full(self.T, -1, np.int32)
        at = 0
        for t, p in trees:
            tok[at:at + len(t)], par[at:at + len(t)] = t, p
            at += len(t)
        self.new.copy_(ints([len(t) for t, _ in trees]))
        self.tokens.copy_(gpu(tok))
        self.parent.copy_(gpu(par))
        self.u.copy_(gpu(rng.random(self.T).astype(np.float32)))
        self.r.copy_(gpu(rng.random(3).astype(np.float32)))


def next_distributions(loop, text):
    """The model's distribution behind each token of a text, from a cache of its own."""
    n = len(text)
    tables = torch.arange(loop.entries, dtype=torch.int32, device="cuda")[None]
    batch = lmx.PagedBatch(ints([0, n]), ints([n]), tables, n_tokens=n, max_new=n, max_ctx=n)
    nq, nk = loop.heads * loop.hd, loop.kv * loop.hd
    outs = []
    for cache, rows_ in zip(loop.caches, loop.rows):
        c = lmx.PagedCache.empty(loop.entries, page_size=loop.page, n_kv_heads=loop.kv, head_dim=loop.hd, dtype=cache.dtype)
        x = rows_[torch.tensor(text, device="cuda")]
        q = lmx.paged_prologue(x[:, :nq], x[:, nq:nq + nk], x[:, nq + nk:], c, batch, n_heads=loop.heads)
        outs.append(lmx.paged_attention(q, c, batch, n_heads=loop.heads))
    return torch.softmax(torch.cat(outs, 1) @ loop.head, 1)


@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("captured", [False, True])
def test_a_loop_of_steps_writes_what_the_model_says(store, captured):
    """Greedy steps with trees of drafts, some of them right: the texts are those that
    one token at a time gives (checked where the model's choice is clear), the cache
    holds each text's rows, and the distributions of every step's rows are those of
    their own texts."""
    say("loop", store, captured)
    loop, rng = Loop(store), np.random.default_rng(4)
    texts = [[5], [17, 3, 40, 41, 42, 8, 9], [2] * 30]
    loop.prefill(texts)
    state = [loop.lens, loop.tables.page_table, loop.tables.held, loop.tables.free_pages, loop.tables.n_free]
    state += [x for c in loop.caches for x in (c.k, c.v, c.k_scale, c.v_scale) if x is not None]

    def step(trees):
        loop.load(trees, rng)
        if not captured:
            loop.run()
        elif not hasattr(loop, "graph"):  # once eagerly, taken back, captured, replayed
            before = [x.clone() for x in state]
            loop.run()
            torch.cuda.synchronize()
            loop.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(loop.graph):
                loop.run()
            for x, y in zip(state, before):
                x.copy_(y)
            loop.graph.replay()
        else:
            loop.graph.replay()
        torch.cuda.synchronize()

    for _ in range(9):
        trees = []
        for b in range(3):
            p = next_distributions(loop, texts[b])
            best = int(p[-1].argmax())
            n = int(rng.integers(1, loop.most)) if b else 12
            tok, par = [texts[b][-1]], [-1]
            for i in range(1, n):
                par.append(int(rng.integers(max(0, i - 3), i)))
                tok.append(int(rng.integers(0, loop.vocab)))
            if n > 3:  # the right continuation among them, two tokens deep, behind wrong ones
                tok[2], par[2] = best, 0
                tok[3], par[3] = int(next_distributions(loop, texts[b] + [best])[-1].argmax()), 2
            trees.append((tok, par))
        step(trees)
        cu = loop.step.cu.tolist()
        path, accepted, token = loop.got.path.tolist(), loop.got.accepted.tolist(), loop.got.token.tolist()
        for b, (tok, par) in enumerate(trees):
            # every row's distribution is that of its own text
            for i, chain in enumerate(so.ancestors(par)):
                text = texts[b] + [tok[j] for j in reversed(chain[:-1])]
                want = next_distributions(loop, text)[-1]
                # scores and values in 22 bits, sums over some 50 keys, a product over 512 terms: far below
                assert (loop.p[cu[b] + i] - want).abs().max() < 2e-3
            # the walk over these rows; the right continuation is found in row 2, or before it
            want, t = so.verify(loop.p[cu[b]:cu[b] + len(tok)].cpu().numpy(), tok, None, None, par, greedy=True)
            assert path[b][:accepted[b]] == want and token[b] == t
            if len(tok) > 3:
                assert accepted[b] >= 2 and (want[1] == 1 or want[1:3] == [2, 3])
            texts[b] = texts[b] + [tok[j] for j in path[b][1:accepted[b]]] + [token[b]]
            assert int(next_distributions(loop, texts[b][:-1])[-1].argmax()) == token[b]
        assert loop.lens.tolist() == [len(t) - 1 for t in texts]
        # nobody's pages are lost
        held = sum(loop.tables.held.tolist())
        assert held + int(loop.tables.n_free[0]) == 40
    # the caches hold the texts' rows
    for b in range(3):
        n = len(texts[b]) - 1
        batch = lmx.PagedBatch(ints([0, n]), ints([n]), loop.tables.page_table[b:b + 1].contiguous(), n_tokens=n, max_new=n,
                               max_ctx=n)
        nq, nk = loop.heads * loop.hd, loop.kv * loop.hd
        for cache, rows_ in zip(loop.caches, loop.rows):
            k, v = lmx.paged_read(cache, batch)
            c = lmx.PagedCache.empty(loop.entries, page_size=loop.page, n_kv_heads=loop.kv, head_dim=loop.hd, dtype=cache.dtype)
            table = torch.arange(loop.entries, dtype=torch.int32, device="cuda")[None]
            own = lmx.PagedBatch(ints([0, n]), ints([n]), table, n_tokens=n, max_new=n, max_ctx=n)
            x = rows_[torch.tensor(texts[b][:n], device="cuda")]
            lmx.paged_prologue(x[:, :nq], x[:, nq:nq + nk], x[:, nq + nk:], c, own, n_heads=loop.heads)
            k2, v2 = lmx.paged_read(c, own)
            assert torch.equal(v, v2)
            assert (k - k2).abs().max() <= 2.0 ** -6 * k2.abs().max()  # one step of 8 bits, or of f16


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,n_rot,store", [(128, 128, "f16"), (128, 40, "i8"), (256, 256, "i8"), (512, 512, "f16")])
def test_prologue_in_blocks_of_rows_is_that_of_single_rows(hd, n_rot, store, interleaved):
    """A batch of many rows and the same rows in small batches.  The arithmetic is the
    same but for where a product is fused into the sum behind it, so that each is
    within test_prologue's bound of the exact result, and the two within twice that."""
    say("prologue blocks", hd, n_rot, store, interleaved)
    c = po.PagedCase(50, new=[700, 1, 400], ctx=[900, 30, 400], page=32, kv=2, hd=hd, store=store, pad=3)
    heads = 3
    q, k, v = (gpu(rows(c, 51 + i, h).reshape(c.tokens, -1)) for i, h in enumerate((heads, 2, 2)))
    gain = gpu((1 + 0.1 * np.random.default_rng(1).standard_normal(hd)).astype(np.float32))
    pos = ints(np.random.default_rng(2).integers(0, 1 << 20, c.tokens))
    kw = dict(n_heads=heads, n_rot=n_rot, interleaved=interleaved, turn_scale=1.1, q_gain=gain, k_gain=gain)
    cache, batch = on_gpu(c)
    want = torch.zeros(c.tokens, heads * hd, device="cuda")
    lmx.spec_prologue(q, k, v, cache, batch, pos=pos, q_out=want, **kw)
    small, _ = on_gpu(c)
    got = torch.zeros_like(want)
    for b, n in enumerate(c.new):
        for j in range(0, n, 100):
            m = min(100, n - j)
            at = slice(int(c.cu[b]) + j, int(c.cu[b]) + j + m)
            part = lmx.PagedBatch(ints([0, m]), ints([c.ctx[b] - n + j + m]), ints(c.table[b:b + 1]), n_tokens=m, max_new=m,
                                  max_ctx=max(c.ctx))
            lmx.spec_prologue(q[at], k[at], v[at], small, part, pos=pos[at], q_out=got[at], **kw)
    rel = 2 * (hd + 34) * 2.0 ** -24 * 1.1  # test_prologue's, of a row head's largest element
    big = want.view(c.tokens, heads, hd).abs().amax(-1, keepdim=True)
    assert ((got - want).view(c.tokens, heads, hd).abs() <= 2 * rel * big).all()
    for name in ("k", "v"):
        x, y = (getattr(p, name).float() for p in (cache, small))
        if store == "i8":  # the scales by the same bound; an int where the quotient lies beside a half
            sx, sy = (getattr(p, name + "_scale") for p in (cache, small))
            assert ((sx - sy).abs() <= 4 * rel * sx).all() and (x - y).abs().max() <= 1
        else:  # a place of f16 where the value lies beside a half
            top = x.abs().amax(-1 if name == "k" else -2, keepdim=True)
            assert ((x - y).abs() <= 2 * rel * top + 2.0 ** -10 * x.abs() + 2.0 ** -24).all()


# --------------------------------------------- calls that tests above do not make --
@pytest.mark.parametrize("kind", ["tree", "chain", "forest"])
@pytest.mark.parametrize("window", [63, 64, 65, 130, 1000, 1 << 29])
def test_windows_of_trees_that_end_in_earlier_words(kind, window):
    say("tree window", kind, window)
    c = po.PagedCase(2, new=[1024, 200, 64], ctx=[1030, 200, 99], page=16, kv=1, hd=64)
    _, batch = on_gpu(c)
    trees = [np.array([-1] + [max(i - (1 + i % 3), 0) for i in range(1, n)]) for n in c.new] if kind == "tree" else \
        trees_of(c, 3, kind)
    got = lmx.spec_tree(ints(np.concatenate(trees)), batch, window=window)
    for b, t in enumerate(trees):
        depth, sees = so.tree(t, window)
        at = slice(int(c.cu[b]), int(c.cu[b + 1]))
        assert np.array_equal(got.pos[at].cpu().numpy(), c.ctx[b] - c.new[b] + depth)
        assert np.array_equal(got.seen[at].cpu().numpy(), so.words_of(sees, 16))


def far_pages(store, hd):
    """A pool whose K and V pass 2^31 elements and 2^32 bytes each, its pages' number, and
    two tables of two requests: the first pages and the last ones."""
    dt = torch.float16 if store == "f16" else torch.int8
    page, kv = 256, 8
    per = page * kv * hd
    n_pages = ((1 << 32) + (1 << 28)) // (per * (2 if store == "f16" else 1)) + 12
    cache = lmx.PagedCache.empty(n_pages, page_size=page, n_kv_heads=kv, head_dim=hd, dtype=dt)
    for x in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        if x is not None:
            x.zero_()
    ids = np.arange(12).reshape(2, 6)
    return cache, n_pages, ints(ids), ints(n_pages - 1 - ids)


@pytest.mark.parametrize("store,hd,new", [("f16", 128, 7), ("f16", 128, 60), ("i8", 64, 7), ("i8", 64, 100), ("f16", 512, 3)])
def test_pages_beyond_32_bits_of_offset(store, hd, new):
    """The same requests in the first pages of a pool and in the last: the same bits
    come out of every call, and land where they belong."""
    say("far pages", store, hd, new)
    torch.manual_seed(5)
    cache, n_pages, near, far = far_pages(store, hd)
    kv, heads, first, n_seq = 8, 16, [1300, 255], 2
    results = []
    for table in (near, far):
        for n, at in ((np.array(first), 0), (np.array([new, new]), 1)):
            torch.manual_seed(6 + at)
            T = int(n.sum())
            ctx = n if at == 0 else n + first
            batch = lmx.PagedBatch(ints(np.concatenate([[0], np.cumsum(n)])), ints(ctx), table, n_tokens=T,
                                   max_new=int(n.max()), max_ctx=int(ctx.max()))
            q, k, v = (torch.randn(T, h * hd, device="cuda") for h in (heads, kv, kv))
            if at == 0:
                lmx.paged_append(k, v, cache, batch)
        parent = ints(np.concatenate([[-1] + [max(i - 2, 0) for i in range(1, new)]] * n_seq))
        tree = lmx.spec_tree(parent, batch)
        q = lmx.spec_prologue(q, k, v, cache, batch, n_heads=heads, pos=tree.pos, q_dtype=torch.float16)
        out = lmx.spec_attention(q, cache, batch, tree.seen, n_heads=heads)
        path = np.full((n_seq, new), -1)
        path[:, :(new + 1) // 2] = np.arange(0, new, 2)
        lmx.spec_keep([cache], batch, ints(path), ints([min((new + 1) // 2, 4)] * n_seq))
        k2, v2 = lmx.paged_read(cache, lmx.PagedBatch(ints([0, *np.cumsum(ctx)]), ints(ctx), table, n_tokens=int(ctx.sum()),
                                                      max_new=int(ctx.max()), max_ctx=int(ctx.max())))
        results.append((q, out, k2, v2))
    assert results[0][1].abs().max() > 0
    for x, y in zip(*results):
        assert torch.equal(x, y)
    assert not cache.k[20:n_pages - 20].any() and not cache.v[20:n_pages - 20].any()


def test_distributions_beyond_32_bits_of_offset():
    """The last of 1100 rows of 2^21 entries: their own words, not those that 32 bits reach."""
    say("far rows")
    vocab, T = 1 << 21, 1100
    p = torch.zeros(T, vocab, dtype=torch.float16, device="cuda")
    tokens = np.zeros(T, np.int32)
    rng = np.random.default_rng(8)
    best = rng.integers(0, vocab, T)
    p[torch.arange(T, device="cuda"), gpu(best)] = 1
    new = [1000, 100]
    cu = ints([0, 1000, 1100])
    for b, at in ((0, 0), (1, 1000)):  # chains that are right up to a wrong token
        n = new[b]
        tokens[at + 1:at + n] = best[at:at + n - 1]
        tokens[at + n - 2] += 1 if tokens[at + n - 2] == 0 else -1
    u, r = torch.full((T,), 0.5, device="cuda"), torch.tensor([0.25, 0.75], device="cuda")
    for kw in (dict(), dict(greedy=True), dict(q=p)):
        got = lmx.spec_verify(p, ints(tokens), u, r, cu, max_new=1000, **kw)
        assert got.accepted.tolist() == [998, 98]
        if "q" not in kw:
            assert got.token.tolist() == [int(best[997]), int(best[1097])]
        else:  # the draft was p itself and is refused for a token it never gives: nothing left, p's own
            assert got.token.tolist() == [int(best[997]), int(best[1097])]


class Captured:
    """Every call of a step, with inputs that `fill` changes and outputs of its own."""

    def __init__(self, drafts, ws, vocab=5000):
        self.c = po.PagedCase(60, new=[20, 3, 9], ctx=[900, 70, 9], page=16, kv=2, hd=128, store="i8", pad=4, spare=60)
        c = self.c
        self.cache, _ = on_gpu(c)
        self.kept = [x.clone() for x in (self.cache.k, self.cache.v, self.cache.k_scale, self.cache.v_scale)]
        table = np.full((3, 80), -1)
        for b, row in enumerate(c.table):
            table[b, :-(-c.ctx[b] // 16)] = row[:-(-c.ctx[b] // 16)]
        held = [-(-x // 16) for x in c.ctx]
        used = {int(x) for b in range(3) for x in table[b, :held[b]]}
        free = [x for x in range(c.n_pages) if x not in used]
        self.start = [ints(table), ints(held), ints(free + [0] * (c.n_pages - len(free))), ints([len(free), 0])]
        self.tables = lmx.PageTables(*[x.clone() for x in self.start], page_size=16)
        self.T, self.most = 48, 16
        self.step = lmx.StepPlan.empty(self.tables, n_tokens=self.T)
        self.batch = lmx.PagedBatch(self.step.cu, self.step.ctx_lens, self.tables.page_table, n_tokens=self.T,
                                    max_new=self.most, max_ctx=80 * 16)
        self.lens, self.new = ints([0] * 3), ints([0] * 3)
        self.parent, self.tokens = ints([-1] * self.T), ints([0] * self.T)
        self.q, self.k, self.v = (torch.zeros(self.T, h * 128, device="cuda") for h in (8, 2, 2))
        self.p, self.draft = (torch.zeros(self.T, vocab, device="cuda") for _ in range(2))
        self.u, self.r = torch.zeros(self.T, device="cuda"), torch.zeros(3, device="cuda")
        self.tree = spec.SpecTree(ints([0] * self.T), torch.zeros(self.T, 1, dtype=torch.int64, device="cuda"))
        self.turned, self.out = (torch.zeros(self.T, 8 * 128, device="cuda") for _ in range(2))
        self.got = spec.Verified(ints(np.zeros((3, self.most))), ints([0] * 3), ints([0] * 3))
        self.drafts, self.ws = drafts, ws

    def fill(self, seed):
        g, rng = torch.Generator("cuda").manual_seed(seed), np.random.default_rng(seed)
        for x, y in zip((self.tables.page_table, self.tables.held, self.tables.free_pages, self.tables.n_free), self.start):
            x.copy_(y)
        for x, y in zip((self.cache.k, self.cache.v, self.cache.k_scale, self.cache.v_scale), self.kept):
            x.copy_(y)
        new = rng.integers(0, 17, 3)
        self.lens.copy_(ints([int(rng.integers(0, x + 1)) for x in self.c.ctx]))
        self.new.copy_(ints(new))
        self.parent.copy_(ints([int(rng.integers(-1, 4)) for _ in range(self.T)]))
        self.tokens.copy_(ints(rng.integers(0, 4, self.T)))  # the likely ones, and one that is not
        for x in (self.q, self.k, self.v):
            x.normal_(generator=g)
        for x in (self.u, self.r):
            x.uniform_(generator=g)
        for x in (self.p, self.draft):
            x.uniform_(generator=g)
            x[:, :3] *= 5000
            x.div_(x.sum(1, keepdim=True))
        self.step.slots.fill_(9)
        for x in (self.out, self.turned):
            x.fill_(3)

    def run(self):
        lmx.spec_plan(self.tables, self.lens, self.new, out=self.step, trim=True)
        lmx.spec_tree(self.parent, self.batch, out=self.tree)
        lmx.spec_prologue(self.q, self.k, self.v, self.cache, self.batch, n_heads=8, pos=self.tree.pos, q_out=self.turned)
        lmx.spec_attention(self.turned, self.cache, self.batch, self.tree.seen, n_heads=8, out=self.out, workspace=self.ws)
        kw = dict(q=self.draft) if self.drafts == "sampled" else dict(greedy=True) if self.drafts == "greedy" else {}
        lmx.spec_verify(self.p, self.tokens, self.u, self.r, self.step.cu, max_new=self.most, parent=self.parent,
                        lens=self.lens, out=self.got, workspace=self.ws, **kw)
        lmx.spec_keep([self.cache], self.batch, self.got.path, self.got.accepted)

    def results(self):
        rows_ = int(self.step.cu[-1])
        return [x.clone() for x in (*self.step, self.lens, self.tables.page_table, self.tables.held, self.tables.n_free,
                                    self.tree.pos[:rows_], self.tree.seen[:rows_], self.turned, self.out, *self.got,
                                    self.cache.k, self.cache.v, self.cache.k_scale, self.cache.v_scale)]

    def capture(self):
        self.fill(99)
        self.run()
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.run()

    def same(self, want):
        return all(torch.equal(x, y) for x, y in zip(self.results(), want))


@pytest.mark.parametrize("vocab", [5000, 40000])
def test_graphs_that_share_a_workspace_replay_as_eager_steps(vocab):
    """Three graphs, of drafts of each kind, over one workspace; eager steps of another
    program in between."""
    ws = lmx.Workspace(1 << 24)
    steps = {d: Captured(d, ws, vocab) for d in ("sampled", "best", "greedy")}
    other = Captured("sampled", None, vocab)
    for s in steps.values():
        s.capture()
    for seed in range(6):
        for d, s in steps.items():
            say("graph", d, seed)
            s.fill(seed)
            s.run()
            torch.cuda.synchronize()
            want = s.results()
            other.fill(seed + 50)
            s.fill(seed)
            s.graph.replay()
            other.run()  # eager work behind the replay
            assert s.same(want)
            torch.cuda.synchronize()
            s.fill(seed)
            s.graph.replay()
            assert s.same(want)


def test_steps_on_two_streams_at_once():
    """Each with its own tables, cache and workspace."""
    steps = [Captured("sampled", lmx.Workspace(1 << 24), 40000), Captured("best", None)]
    wants = []
    for i, s in enumerate(steps):
        s.fill(i)
        s.run()
        torch.cuda.synchronize()
        wants.append(s.results())
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(5):
        for i, s in enumerate(steps):
            s.fill(i)
        torch.cuda.synchronize()
        for s, st in zip(steps, streams):
            with torch.cuda.stream(st):
                s.run()
        torch.cuda.synchronize()
        for s, want in zip(steps, wants):
            assert s.same(want)


def test_verification_on_a_stream_without_a_workspace():
    """What the call allocates belongs to the stream that uses it."""
    c = verify_case(70, [9, 30], 50000, "tree", "sampled")
    args = (gpu(c["p"]), gpu(c["tok"]), gpu(c["u"]), gpu(c["r"]), gpu(c["cu"]))
    kw = dict(max_new=30, parent=ints(np.concatenate(c["trees"])), q=gpu(c["q"]))
    want = lmx.spec_verify(*args, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        got = lmx.spec_verify(*args, stream=side, **kw)
        torch.empty(1 << 20, dtype=torch.uint8, device="cuda").fill_(255)  # of the other stream
        side.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_what_python_refuses():
    c = po.PagedCase(71, new=[4, 2], ctx=[40, 9], page=16, kv=1, hd=64)
    cache, batch = on_gpu(c)
    parent, seen = ints([-1, 0, 1, 1, -1, 0]), torch.full((6, 1), -1, dtype=torch.int64, device="cuda")
    q, kv = torch.randn(6, 128, device="cuda"), torch.randn(6, 64, device="cuda")
    p, tok, u, r, cu = torch.rand(6, 30, device="cuda"), ints([0] * 6), torch.rand(6, device="cuda"), torch.rand(2, device="cuda"), batch.cu
    path, accepted = ints([[0, -1, -1, -1]] * 2), ints([1, 1])
    good = dict(n_heads=2)
    bad = [
        lambda: lmx.spec_tree(parent.cpu(), batch), lambda: lmx.spec_tree(parent.long(), batch),
        lambda: lmx.spec_tree(parent[:5], batch), lambda: lmx.spec_tree(ints([0] * 12)[::2], batch),
        lambda: lmx.spec_tree(parent, batch, out=spec.SpecTree(ints([0] * 7), torch.zeros(7, 1, dtype=torch.int64, device="cuda"))),
        lambda: spec.SpecTree(ints([0] * 6), seen.int()), lambda: spec.SpecTree(ints([0] * 6), seen.view(-1)),
        lambda: lmx.spec_prologue(q, kv, kv, cache, batch, pos=parent.float(), **good),
        lambda: lmx.spec_prologue(q, kv, kv, cache, batch, pos=parent.cpu(), **good),
        lambda: lmx.spec_prologue(q.half(), kv, kv, cache, batch, **good),
        lambda: lmx.spec_prologue(q, kv, None, cache, batch, **good),
        lambda: lmx.spec_prologue(q, kv, kv, cache, batch, n_heads=3),
        lambda: lmx.spec_attention(q, cache, batch, seen[:5], **good), lambda: lmx.spec_attention(q, cache, batch, seen.cpu(), **good),
        lambda: lmx.spec_attention(q, cache, batch, seen.int(), **good), lambda: lmx.spec_attention(q.double(), cache, batch, seen, **good),
        lambda: lmx.spec_attention(q, cache, batch, seen, window=5, **good),  # a window asks for positions
        lambda: lmx.spec_attention(q, cache, batch, seen, out=q.half(), **good),
        lambda: lmx.spec_verify(p.double(), tok, u, r, cu, max_new=4), lambda: lmx.spec_verify(p, tok, u, None, cu, max_new=4),
        lambda: lmx.spec_verify(p, tok, u[:5], r, cu, max_new=4), lambda: lmx.spec_verify(p, tok, u, r.half(), cu, max_new=4),
        lambda: lmx.spec_verify(p, tok.cpu(), u, r, cu, max_new=4), lambda: lmx.spec_verify(p, tok, u, r, cu, max_new=7),
        lambda: lmx.spec_verify(p, tok, u, r, cu, max_new=0), lambda: lmx.spec_verify(p[0], tok, u, r, cu, max_new=4),
        lambda: lmx.spec_verify(p, tok, u, r, cu, max_new=4, q=p.half()), lambda: lmx.spec_verify(p, tok, u, r, cu, max_new=4, lens=ints([0])),
        lambda: lmx.spec_verify(p, tok, u, r, cu, max_new=4, out=lmx.Verified.empty(2, 3, p.device)),
        lambda: lmx.spec_keep([cache], batch, path.long(), accepted), lambda: lmx.spec_keep([cache], batch, path[:1], accepted),
        lambda: lmx.spec_keep([cache], batch, path[:, :2].contiguous(), accepted), lambda: lmx.spec_keep([cache], batch, path, accepted[:1]),
        lambda: lmx.spec_keep([cache, cache], batch, path, accepted),  # one pool twice
    ]
    before = [cache.k.clone(), cache.v.clone()]
    for i, call in enumerate(bad):
        say("refused", i)
        with pytest.raises((TypeError, ValueError, RuntimeError, lmx.LmxError)):
            call()
    assert torch.equal(cache.k, before[0]) and torch.equal(cache.v, before[1])


@pytest.mark.parametrize("store,most", [("f16", 700), ("i8", 700), ("f16", 1024), ("f16", 1025), ("i8", 2048), ("i8", 2049)])
def test_attention_of_sequences_that_fill_the_cus(store, most):
    """Enough of them that the shorter are not split, and the first length at which they are."""
    say("many sequences", store, most)
    rng = np.random.default_rng(most)
    ctx = [most] + [int(x) for x in rng.integers(3, most // 8, 63)]
    c = po.PagedCase(80, new=[1 + i % 3 for i in range(64)], ctx=ctx, page=16, kv=4, hd=64, store=store)
    check(c, 4, masks(c, 81, "tree"), q16=store == "f16")
