"""Steps with drafted tokens on the GPU at their limits: what a result's own rounding
leaves, full tables, many requests, and streams beside the current one."""
from types import SimpleNamespace

import numpy as np
import pytest

from tests import paged_oracle as po
from tests import spec_oracle as so

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import llmoxide_amd as lmx  # noqa: E402
from tests.test_gpu_paged import gpu, on_gpu, rows, say  # noqa: E402
from tests.test_gpu_spec import ints, masks, trees_of  # noqa: E402
from tests.test_spec_plan import requests  # noqa: E402


# ------------------------------------------------------------------ precision --
@pytest.mark.parametrize("new,ctx", [([1], [40]), ([4, 1, 3], [70, 5, 33]), ([20, 7], [60, 90]), ([70], [100])])
@pytest.mark.parametrize("hd,kv,heads,store", [(64, 2, 8, "f16"), (64, 2, 8, "i8"), (128, 2, 8, "f16"), (128, 2, 8, "i8"),
                                               (256, 1, 4, "i8"), (256, 1, 4, "f16"), (512, 1, 2, "f16"), (512, 1, 2, "i8")])
def test_f16_results_by_masks_are_off_by_their_own_rounding(new, ctx, hd, kv, heads, store):
    """With f16 q the weights have 22 bits, as with f32.  q has one element that is not 0
    in each row head, so that a score is one product (exact: 22 bits) and attend_bound's
    term of head_dim products is that of one.  What it then gives for f32 results, b, is
    some 1e-5 of the result; f16(y) is off from y by 2^-11 |y|, or 2^-25 where f16's
    steps are 2^-24: together (1 + 2^-11) b + 2^-11 |want| + 2^-25.  Weights of 11 bits
    would add 2^-12 of each weighted value or so, half of the last place."""
    say("f16 rounding", new, hd, store)
    c = po.PagedCase(101, new=new, ctx=ctx, page=16, kv=kv, hd=hd, store=store)
    cache, batch = on_gpu(c)
    rng = np.random.default_rng(102)
    q = np.zeros((c.tokens, heads, hd), np.float32)
    at = rng.integers(0, hd, (c.tokens, heads, 1))
    np.put_along_axis(q, at, (rng.standard_normal(at.shape) * 8).astype(np.float16).astype(np.float32), 2)
    sees = masks(c, 103, "tree")
    seen = gpu(np.concatenate([so.words_of(m, -(-max(new) // 64)) for m in sees]))
    got = lmx.spec_attention(gpu(q.reshape(c.tokens, -1)).half(), cache, batch, seen, n_heads=heads)
    want, mag, prod, top = so.attend(c, q, sees, heads=heads)
    b = po.attend_bound(SimpleNamespace(hd=1, store=store), mag, prod, top, max(ctx), f32=True)
    off = np.abs(got.double().cpu().numpy().reshape(want.shape) - want)
    most = (1 + 2.0 ** -11) * b + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    assert np.all(off <= most), f"{(off > most).sum()} of {off.size} are off by up to {(off / most).max():.2f} times the bound"


# --------------------------------------------------------------- verification --
@pytest.mark.parametrize("vocab", [3, 700, 32768, 40000])
def test_a_test_beside_its_border_is_decided_in_64_bits(vocab):
    """The root's second child: a is 1, W = (3/8 - 2^-27) + (5/8 - 1/2) = 1/2 - 2^-27, and
    u W q = 1/2 W 1/2 = 1/8 - 2^-29 lies below w = 1/8.  With 3/8 - 2^-27 rounded to 24
    bits W is 1/2, and the child, for which 1/8 < 1/8 fails, is refused."""
    p, q = np.zeros((3, vocab), np.float32), np.zeros((3, vocab), np.float32)
    p[0, :3], q[0, :3] = (0, 3 / 8, 5 / 8), (0.5, 2.0 ** -27, 0.5)
    p[1:, 1] = q[1:, 1] = 1
    tokens, u, r, parent = [0, 0, 2], [0, 0.5, 0.5], [0.5], [-1, 0, 0]
    path, token = so.verify(p, tokens, u, r[0], parent, q)
    assert path == [0, 2] and token == 1  # child 1, of p 0, is refused and makes a 1
    got = lmx.spec_verify(gpu(p), ints(tokens), gpu(np.float32(u)), gpu(np.float32(r)), ints([0, 3]), max_new=3,
                          parent=ints(parent), q=gpu(q))
    assert got.path.tolist() == [[0, 2, -1]] and got.accepted.tolist() == [2] and got.token.tolist() == [1]


# ----------------------------------------------------------------------- plans --
@pytest.mark.parametrize("n_seq", [129, 160, 192, 257, 300, 448, 513, 700, 832, 960, 1024 + 160])
@pytest.mark.parametrize("trim", [False, True])
@pytest.mark.parametrize("extra", [1, 9000])
def test_plans_of_any_number_of_requests(n_seq, trim, extra):
    """Numbers of requests between a power of two and the next, rows mapped by either
    kernel; the tables lie among rows that have to stay as they are."""
    say("plan", n_seq, trim, extra)
    lens, new, table, held, free, n_free = requests(n_seq, n_seq, 16, 40)
    n = int(new.sum()) + extra
    wide = torch.full((3 * n_seq, table.shape[1]), 77, dtype=torch.int32, device="cuda")
    wide[n_seq:2 * n_seq] = ints(table)
    t = lmx.PageTables(wide[n_seq:2 * n_seq], ints(held), ints(free), ints(n_free), page_size=16)
    got = lmx.spec_plan(t, ints(lens), ints(new), n_tokens=n, trim=trim)
    want = so.plan(lens, new, table.astype(np.int32), held.astype(np.int32), free.astype(np.int32), n_free, page=16, n_tokens=n,
                   n_pages=len(free), trim=trim)
    for name, g, w in zip("table held free n_free cu ctx slots pos".split(), (t.page_table, t.held, t.free_pages, t.n_free, *got), want):
        assert np.array_equal(g.cpu().numpy(), w), name
    assert (wide[:n_seq] == 77).all() and (wide[2 * n_seq:] == 77).all()


def beyond(c, entries):
    """The cache of a PagedCase, and its batch with tables that end after ``entries``."""
    c.table, c.stride = np.ascontiguousarray(c.table[:, :entries]), entries
    cache, _ = on_gpu(c)
    return cache, lmx.PagedBatch(gpu(c.cu), ints(c.ctx), gpu(c.table), n_tokens=c.tokens, max_new=max(c.new), max_ctx=entries * c.page)


@pytest.mark.parametrize("new,ctx", [([1, 3, 2], [65, 66, 9]), ([4, 4, 4], [63, 70, 99]), ([40, 9, 3], [70, 80, 400]),
                                     ([64, 7, 33], [127, 64, 65]), ([70, 2, 65], [64, 60, 80])])
@pytest.mark.parametrize("store,hd", [("f16", 128), ("i8", 64), ("f16", 256)])
def test_rows_behind_the_end_of_a_table(new, ctx, store, hd):
    """Sequences that are longer than the 64 positions of their table: rows within it are
    stored and attend as they should, the others are stored nowhere and see what is there;
    what was cached keeps every bit.  Those with a length below their rows are in no page."""
    say("table's end", new, ctx, store, hd)
    heads, kv = 4, 2
    c = po.PagedCase(110, new=new, ctx=ctx, page=16, kv=kv, hd=hd, store=store)
    cache, batch = beyond(c, 4)
    none = [b for b in range(3) if new[b] > ctx[b]]  # of these no row has a position
    x = [rows(c, 111 + i, h) for i, h in enumerate((heads, kv, kv))]
    q, k, v = (gpu(y.reshape(c.tokens, -1)) for y in x)
    for b in none:
        c.table[b] = -1  # the oracle's, whose rows would have positions below 0 and above
    want = po.append(c, x[1], x[2])
    lmx.paged_append(k, v, cache, batch)
    for got, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):
        if w is not None:
            assert np.array_equal(got.cpu().numpy(), w)
    k2, v2 = lmx.paged_read(cache, batch)
    for row, _, _, at in c.row_places():
        assert (k2[row].any() and v2[row].any()) == (at is not None)
    # prologues: the same places
    stored = np.zeros((c.n_pages, 16), bool)
    for _, _, _, at in c.row_places():
        if at is not None:
            stored[at] = True
    for call in (lmx.paged_prologue, lmx.spec_prologue):
        twin, _ = on_gpu(c)
        call(q, k, v, twin, batch, n_heads=heads)
        assert np.array_equal((twin.k.cpu().numpy() != c.k).any((1, 3)), stored)
        assert np.array_equal((twin.v.cpu().numpy() != c.v).any((1, 2)), stored)
    c.k, c.v, c.k_scale, c.v_scale = want
    # attention, causal and by masks
    for window in (0, 20):
        ref, mag, prod, top = po.attend(c, x[0], heads=heads, window=window)
        got = lmx.paged_attention(q, cache, batch, n_heads=heads, window=window).cpu().numpy().reshape(ref.shape)
        assert np.all(np.abs(got - ref) <= po.attend_bound(c, mag, prod, top, 64, f32=True))
        trees = trees_of(c, 112)
        sees = [so.tree(t, window)[1] for t in trees]
        pos = np.concatenate([ctx[b] - new[b] + so.tree(t)[0] for b, t in enumerate(trees)])
        seen = gpu(np.concatenate([so.words_of(m, 2) for m in sees]))
        ref, mag, prod, top = so.attend(c, x[0], sees, heads=heads, window=window, pos=pos)
        got = lmx.spec_attention(q, cache, batch, seen, n_heads=heads, window=window, pos=ints(pos)).cpu().numpy().reshape(ref.shape)
        assert np.all(np.abs(got - ref) <= po.attend_bound(c, mag, prod, top, 64, f32=True))
    # keeping: from places and to places that there are
    path = np.full((3, max(new)), -1)
    for b, n in enumerate(new):
        path[b, :(n + 1) // 2] = np.arange(0, n, 2)
    accepted = [(n + 1) // 2 for n in new]
    want = so.keep(c, path, accepted, want)
    lmx.spec_keep([cache], batch, ints(path), ints(accepted))
    for got, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):
        if w is not None:
            assert np.array_equal(got.cpu().numpy(), w)


class Cut(po.PagedCase):
    """What queries see of a case whose batch has ``max_ctx``."""
    limit = 1 << 30

    def place(self, b, pos):
        return super().place(b, pos) if pos < self.limit else None


@pytest.mark.parametrize("limit", [40, 48, 63])
@pytest.mark.parametrize("new", [[3, 9, 1], [30, 5, 20], [60, 47, 64]])
@pytest.mark.parametrize("store,hd,q16", [("f16", 128, False), ("f16", 64, True), ("i8", 128, True), ("i8", 256, False)])
def test_rows_behind_a_batchs_longest_length(limit, new, store, hd, q16):
    """Lengths that pass max_ctx, within the table: all rows are stored where they belong,
    and none sees a position from max_ctx on."""
    say("beyond max_ctx", limit, new, store, hd, q16)
    heads, kv = 4, 2
    c = Cut(115, new=new, ctx=[61, 64, 64], page=16, kv=kv, hd=hd, store=store)
    cache, _ = on_gpu(c)
    batch = lmx.PagedBatch(gpu(c.cu), ints(c.ctx), gpu(c.table), n_tokens=c.tokens, max_new=max(new), max_ctx=limit)
    x = [rows(c, 116 + i, h) for i, h in enumerate((heads, kv, kv))]
    q, k, v = (gpu(y.reshape(c.tokens, -1)) for y in x)
    want = po.append(c, x[1], x[2])
    lmx.paged_append(k, v, cache, batch)
    for got, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):
        if w is not None:
            assert np.array_equal(got.cpu().numpy(), w)
    c.k, c.v, c.k_scale, c.v_scale = want
    c.limit = limit
    if q16:
        x[0] = x[0].astype(np.float16).astype(np.float32)
        q = q.half()
    for window in (0, 13):
        trees = trees_of(c, 117)
        sees = [so.tree(t, window)[1] for t in trees]
        pos = np.concatenate([c.ctx[b] - new[b] + so.tree(t)[0] for b, t in enumerate(trees)])
        seen = gpu(np.concatenate([so.words_of(m, 1) for m in sees]))
        for ref, got in ((po.attend(c, x[0], heads=heads, window=window),
                          lmx.paged_attention(q, cache, batch, n_heads=heads, window=window)),
                         (so.attend(c, x[0], sees, heads=heads, window=window, pos=pos),
                          lmx.spec_attention(q, cache, batch, seen, n_heads=heads, window=window, pos=ints(pos)))):
            ref, mag, prod, top = ref
            got = got.double().cpu().numpy().reshape(ref.shape)
            assert np.all(np.abs(got - ref) <= po.attend_bound(c, mag, prod, top, 64, f32=not q16))


def test_a_full_request_leaves_its_prefix_and_its_neighbours():
    """Two requests share their first pages; one reaches the end of its row of the table in
    this step, the other goes on.  The plan's lengths lead the prologue to the map's slots."""
    page, kv, hd, heads, entries = 16, 1, 64, 2, 3
    free = np.zeros(12, np.int32)
    free[:6] = np.arange(6, 12)
    t = lmx.PageTables(ints([[0, 1, -1], [0, 2, -1]]), ints([2, 2]), ints(free), ints([6, 0]), page_size=page)
    cache = lmx.PagedCache.empty(12, page_size=page, n_kv_heads=kv, head_dim=hd)
    cache.k.fill_(7), cache.v.fill_(9)
    for new in ([18, 4], [40, 4], [5, 4]):
        n, lens = sum(new), [32, 30]
        step = lmx.spec_plan(t, ints(lens), ints(new), n_tokens=n, trim=True)
        batch = lmx.PagedBatch(step.cu, step.ctx_lens, t.page_table, n_tokens=n, max_new=max(new), max_ctx=entries * page)
        q, k, v = (torch.randn(n, h * hd, device="cuda") for h in (heads, kv, kv))
        tree = lmx.spec_tree(ints(np.concatenate([np.arange(-1, m - 1) for m in new])), batch)
        assert tree.pos.tolist() == step.pos.tolist() == [a + j for a, m in zip(lens, new) for j in range(m)]
        cache.k.fill_(7), cache.v.fill_(9)
        lmx.spec_prologue(q, k, v, cache, batch, n_heads=heads, n_rot=0, pos=tree.pos)
        want_k, want_v = torch.full_like(cache.k, 7), torch.full_like(cache.v, 9)
        for row, at in enumerate(step.slots.tolist()):
            if at >= 0:
                want_k[at // page, 0, at % page], want_v[at // page, 0, :, at % page] = k[row].half(), v[row].half()
        assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v), new
