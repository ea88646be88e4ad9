"""The paged cache on the GPU against its float64 definitions (paged_oracle):
write, read-back, prologue and attention, over types, head sizes, pages, ragged
lengths, missing pages, non-finite values in places no row sees, strides, streams
and captured graphs."""
import numpy as np
import pytest

from tests import paged_oracle as po

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import llmoxide_amd as lmx  # noqa: E402


def gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def on_gpu(c):
    """(cache, batch) of a PagedCase."""
    scales = [None if s is None else gpu(s) for s in (c.k_scale, c.v_scale)]
    cache = lmx.PagedCache(gpu(c.k), gpu(c.v), *scales)
    batch = lmx.PagedBatch(gpu(c.cu), gpu(np.array(c.ctx, np.int32)), gpu(c.table), n_tokens=c.tokens,
                           max_new=max(c.new), max_ctx=max(c.ctx))
    return cache, batch


def say(*a):
    print(*a, flush=True)


def rows(c, seed, heads, scale=1.0):
    return (np.random.default_rng(seed).standard_normal((c.tokens, heads, c.hd)) * scale).astype(np.float32)


RAGGED = [
    dict(new=[1], ctx=[1]),
    dict(new=[1, 1, 1], ctx=[1, 17, 40]),
    dict(new=[5, 0, 33, 1], ctx=[5, 20, 70, 64], pad=3),
    dict(new=[70, 2], ctx=[131, 16], pad=1),
]


# ------------------------------------------------------------- append, read --
@pytest.mark.parametrize("lens", RAGGED)
@pytest.mark.parametrize("hd,page,kv", [(64, 16, 3), (128, 32, 2), (256, 64, 1), (512, 16, 2), (128, 256, 1)])
@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("src", ["f32", "f16"])
def test_append_writes_exactly_its_rows(lens, hd, page, kv, store, src):
    say("append", lens, hd, page, kv, store, src)
    c = po.PagedCase(1, page=page, kv=kv, hd=hd, store=store, **lens)
    k, v = rows(c, 2, kv), rows(c, 3, kv, 3.0)
    if src == "f16":
        k, v = k.astype(np.float16).astype(np.float32), v.astype(np.float16).astype(np.float32)
    cache, batch = on_gpu(c)
    dt = torch.float32 if src == "f32" else torch.float16
    # columns of a fused row, other columns around them
    fused = torch.full((c.tokens, 8 + 2 * kv * hd), float("nan"), dtype=dt, device="cuda")
    fused[:, 4:4 + kv * hd], fused[:, 8 + kv * hd:] = gpu(k.reshape(c.tokens, -1)), gpu(v.reshape(c.tokens, -1))
    lmx.paged_append(fused[:, 4:4 + kv * hd], fused[:, 8 + kv * hd:], cache, batch)
    torch.cuda.synchronize()
    want = po.append(c, k, v)
    for got, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):
        if w is not None:
            assert np.array_equal(got.cpu().numpy(), w)


@pytest.mark.parametrize("lens", RAGGED)
@pytest.mark.parametrize("hd,page,kv", [(64, 16, 3), (128, 32, 2), (256, 64, 1), (512, 16, 2), (128, 128, 2)])
@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("out", ["f32", "f16"])
def test_read_gives_the_pages_values(lens, hd, page, kv, store, out):
    say("read", lens, hd, page, kv, store, out)
    c = po.PagedCase(4, page=page, kv=kv, hd=hd, store=store, **lens)
    if max(c.ctx) > 2 * page:
        c.table[int(np.argmax(c.ctx)), 0] = -1  # let go
        c.table[int(np.argmax(c.ctx)), 1] = c.n_pages  # no page either
    cache, batch = on_gpu(c)
    dt = torch.float32 if out == "f32" else torch.float16
    wide = torch.full((c.tokens, 2 * kv * hd + 4), 7.0, dtype=dt, device="cuda")
    k, v = wide[:, :kv * hd], wide[:, kv * hd + 4:]
    lmx.paged_read(cache, batch, k_out=k, v_out=v)
    torch.cuda.synchronize()
    want = np.full((2, c.tokens, kv, hd), 7.0, np.float32)
    for row, b, pos, at in c.row_places():
        for h in range(kv):
            if at is None:
                want[:, row, h] = 0
            else:
                want[:, row, h] = c.held(b, h, pos)  # int * f32: one rounding
    np_dt = np.float32 if out == "f32" else np.float16
    for got, w in zip((k, v), want):
        got = got.cpu().numpy().reshape(c.tokens, kv, hd)
        # the value is rounded once to f32, and for f16 once more
        assert np.array_equal(got, w.astype(np_dt))
    assert torch.all(wide[:, kv * hd:kv * hd + 4] == 7)


def test_append_one_side_and_missing_pages():
    c = po.PagedCase(5, new=[40, 3], ctx=[80, 3], page=16, kv=2, hd=128, store="i8")
    c.table[0, 3] = -1
    c.table[0, 4] = 1 << 30
    k, v = rows(c, 6, 2), rows(c, 7, 2)
    want = po.append(c, k, v)
    cache, batch = on_gpu(c)
    lmx.paged_append(gpu(k.reshape(c.tokens, -1)), None, cache, batch)
    assert np.array_equal(cache.v.cpu().numpy(), c.v)
    lmx.paged_append(None, gpu(v.reshape(c.tokens, -1)), cache, batch)
    for got, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):
        assert np.array_equal(got.cpu().numpy(), w)


def test_eight_bit_rounding_at_its_borders():
    """Ties, values one place beside them, tiny and huge heads, infinities and NaN."""
    kv, hd = 2, 128
    c = po.PagedCase(8, new=[24], ctx=[24], page=16, kv=kv, hd=hd, store="i8")
    rng = np.random.default_rng(9)
    x = np.zeros((24, kv, hd), np.float32)
    for r in range(24):
        for h in range(kv):
            s = np.float32(rng.uniform(0.5, 2) * 2.0 ** rng.integers(-80, 80))
            amax = np.float32(s * 127)
            s = np.float32(np.float64(amax) / 127)
            half = ((np.arange(hd - 1) - 63 + 0.5) * np.float64(s)).astype(np.float32)  # near k + 1/2
            y = np.where(rng.random(hd - 1) < 0.5, half, np.nextafter(half, np.float32(np.inf)))
            x[r, h, 1:], x[r, h, 0] = y, amax
    x[3, 0] = 0
    x[4, 1, 5] = np.inf
    x[5, 0, 9] = np.nan
    x[6, 1] *= 0
    x[6, 1, 3] = 1e-40
    x[7, 0] = np.float32(3e38)
    x[8, 0] = 0
    x[8, 0, 7] = np.float32(2.0 ** -100)
    k, v = x, x[::-1].copy()
    cache, batch = on_gpu(c)
    lmx.paged_append(gpu(k.reshape(24, -1)), gpu(v.reshape(24, -1)), cache, batch)
    for got, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), po.append(c, k, v)):
        assert np.array_equal(got.cpu().numpy(), w, equal_nan=got.dtype == torch.float32)


# ----------------------------------------------------------------- prologue --
@pytest.mark.parametrize("hd,n_rot,page,kv,heads,store", [
    (64, 64, 16, 2, 6, "f16"), (128, 128, 32, 2, 8, "f16"), (128, 128, 16, 1, 5, "i8"), (128, 48, 64, 2, 2, "f16"),
    (256, 64, 16, 1, 2, "i8"), (256, 256, 32, 2, 4, "f16"), (512, 510, 16, 1, 2, "f16"), (64, 0, 16, 1, 1, "f16"),
    (128, 6, 16, 1, 2, "f16"),
])
@pytest.mark.parametrize("q16", [False, True])
def test_prologue(hd, n_rot, page, kv, heads, store, q16):
    say("prologue", hd, n_rot, page, kv, heads, store, q16)
    c = po.PagedCase(11, new=[3, 0, 37, 1], ctx=[3, 9, 500, 1200], page=page, kv=kv, hd=hd, store=store, pad=2)
    q, k, v = rows(c, 12, heads, 2.0), rows(c, 13, kv, 0.3), rows(c, 14, kv)
    rng = np.random.default_rng(15)
    qg, kg = (1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32)
    factors = (1 + rng.random(max(1, n_rot // 2))).astype(np.float32) if n_rot == 48 else None
    v_norm, gains = hd == 256, hd != 64
    eps, base = 1e-6, 5e5
    cache, batch = on_gpu(c)
    fused = torch.cat([gpu(x.reshape(c.tokens, -1)) for x in (q, k, v)], 1)
    nq, nk = heads * hd, kv * hd
    out = torch.full((c.tokens, nq), 9.0, dtype=torch.float16 if q16 else torch.float32, device="cuda")
    lmx.paged_prologue(fused[:, :nq], fused[:, nq:nq + nk], fused[:, nq + nk:], cache, batch, n_heads=heads,
                       n_rot=n_rot, v_norm=v_norm, rms_eps=eps, rope_base=base, q_gain=gpu(qg) if gains else None,
                       k_gain=gpu(kg) if gains else None, rope_factors=None if factors is None else gpu(factors),
                       q_out=out)
    want_q = np.full((c.tokens, heads, hd), 9.0)
    want_k, want_v = np.zeros((c.tokens, kv, hd)), np.zeros((c.tokens, kv, hd))
    kw = dict(eps=eps, base=base, factors=factors)
    one = np.ones(hd) if v_norm else None
    for row, b, pos, at in c.row_places():
        for h in range(heads):
            want_q[row, h] = po.rope_norm(q[row, h], qg if gains else None, pos, n_rot=n_rot, **kw)
        for h in range(kv):
            want_k[row, h] = po.rope_norm(k[row, h], kg if gains else None, pos, n_rot=n_rot, **kw)
            want_v[row, h] = po.rope_norm(v[row, h], one, pos, n_rot=0, **kw)
    # f32 steps: the row's sum (hd 2^-24 at worst), its root, two products, sin and cos to 2^-22, the turn's
    # two products and sum; a result is a combination of two elements, bounded by the row's largest
    rel = (hd + 32) * 2.0 ** -24
    got = out.float().cpu().numpy().reshape(c.tokens, heads, hd)
    own = np.zeros(c.tokens, bool)
    own[[r for r, *_ in c.row_places()]] = True
    assert np.all(got[~own] == 9)
    tol = 2 * rel * np.abs(want_q).max(-1, keepdims=True) + (2.0 ** -11 * np.abs(want_q) + 2.0 ** -24 if q16 else 0)
    assert np.all(np.abs(got - want_q) <= tol)
    K, V = cache.k.float().cpu().numpy(), cache.v.float().cpu().numpy()
    touched = np.zeros((c.n_pages, c.page), bool)
    for row, b, pos, (p, s) in c.row_places():
        touched[p, s] = True
        for h in range(kv):
            for got1, w, scale in ((K[p, h, s], want_k[row, h], cache.k_scale), (V[p, h, :, s], want_v[row, h], cache.v_scale)):
                big = np.abs(w).max()
                if store == "f16":
                    assert np.all(np.abs(got1 - w) <= 2 * rel * big + 2.0 ** -11 * np.abs(w) + 2.0 ** -24)
                else:  # half a step of the scale, and the f32 steps before it
                    sc = float(scale[p, h, s])
                    assert abs(sc - big / 127) <= 4 * rel * big / 127
                    assert np.all(np.abs(got1 * sc - w) <= (0.5 + 1e-3) * sc + 4 * rel * big)
    assert np.array_equal(cache.k.cpu().numpy()[~touched.any(1)], c.k[~touched.any(1)])
    assert np.array_equal(cache.v.cpu().numpy()[~touched.any(1)], c.v[~touched.any(1)])


def test_prologue_in_place_and_strided_heads():
    """q_out may be q; [query | gate] heads are read at their stride; both as by default."""
    c = po.PagedCase(16, new=[20, 1], ctx=[20, 300], page=16, kv=2, hd=128)
    q, k, v = gpu(rows(c, 17, 4).reshape(c.tokens, -1)), gpu(rows(c, 18, 2).reshape(c.tokens, -1)), gpu(rows(c, 19, 2).reshape(c.tokens, -1))
    cache, batch = on_gpu(c)
    want = lmx.paged_prologue(q, k, v, cache, batch, n_heads=4)
    pair = torch.full((c.tokens, 4, 256), float("nan"), device="cuda")
    pair[:, :, :128] = q.view(c.tokens, 4, 128)
    assert torch.equal(lmx.paged_prologue(pair.view(c.tokens, -1), k, v, cache, batch, n_heads=4, q_head_stride=256), want)
    lmx.paged_prologue(q, k, v, cache, batch, n_heads=4, q_out=q)
    assert torch.equal(q, want)


def test_prologue_at_far_positions():
    """Position 2^24 and beyond: the angle keeps its bits."""
    hd, page = 64, 256
    ctx = (1 << 24) + 5
    entries = -(-ctx // page)
    table = torch.full((1, entries), -1, dtype=torch.int32, device="cuda")
    table[0, -1] = 0
    cache = lmx.PagedCache.empty(1, page_size=page, n_kv_heads=1, head_dim=hd)
    batch = lmx.PagedBatch(torch.tensor([0, 5], dtype=torch.int32, device="cuda"),
                           torch.tensor([ctx], dtype=torch.int32, device="cuda"), table, n_tokens=5, max_new=5, max_ctx=ctx)
    x = np.random.default_rng(1).standard_normal((5, hd)).astype(np.float32)
    got = lmx.paged_prologue(gpu(x), gpu(x), gpu(x), cache, batch, n_heads=1, rope_base=1e4).cpu().numpy()
    for i in range(5):
        want = po.rope_norm(x[i], None, ctx - 5 + i, n_rot=hd, eps=0, base=1e4)
        # doubles: the angle is off by 2^24 * 2^-50, far below the f32 steps
        assert np.abs(got[i] - want).max() <= 16 * 2.0 ** -24 * np.abs(x[i]).max() * 2


# ---------------------------------------------------------------- attention --
def check_attention(c, heads, *, q16, window=0, scale=None, seed=21, q_scale=1.0, ws=None):
    cache, batch = on_gpu(c)
    q = rows(c, seed, heads, q_scale)
    if q16:
        q = q.astype(np.float16).astype(np.float32)
    dt = torch.float16 if q16 else torch.float32
    out = torch.full((c.tokens, heads * c.hd), 5.0, dtype=dt, device="cuda")
    lmx.paged_attention(gpu(q.reshape(c.tokens, -1)).to(dt), cache, batch, n_heads=heads, window=window, scale=scale,
                        out=out, workspace=ws)
    got = out.float().cpu().numpy().reshape(c.tokens, heads, c.hd).astype(np.float64)
    want, mag, prod, top = po.attend(c, q, heads=heads, window=window, scale=scale)
    own = np.zeros(c.tokens, bool)
    own[[r for r, *_ in c.row_places()]] = True
    assert np.all(got[~own] == 5), "rows of no sequence were written"
    bound = po.attend_bound(c, mag, prod, top, max(c.ctx), f32=not q16)
    off = np.abs(got - want) - bound
    assert np.all(np.isfinite(got[own])), "non-finite"
    assert off[own].max() <= 0, f"{off[own].max():.3g} over the bound {bound[own].max():.3g}"
    return got


@pytest.mark.parametrize("lens", RAGGED + [dict(new=[1, 1], ctx=[600, 1]), dict(new=[130], ctx=[300])])
@pytest.mark.parametrize("hd,page,kv,heads", [(64, 16, 2, 6), (128, 16, 2, 8), (128, 64, 1, 1), (256, 32, 1, 4),
                                              (512, 16, 1, 3), (128, 256, 2, 10)])
@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("q16", [False, True])
def test_attention(lens, hd, page, kv, heads, store, q16):
    say("attention", lens, hd, page, kv, heads, store, q16)
    check_attention(po.PagedCase(20, page=page, kv=kv, hd=hd, store=store, **lens), heads, q16=q16)


@pytest.mark.parametrize("window", [1, 7, 64, 100])
@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("hd,q16", [(128, True), (128, False), (256, True)])
def test_attention_windows(window, store, hd, q16):
    say("window", window, store, hd, q16)
    c = po.PagedCase(22, new=[1, 150, 40, 1], ctx=[400, 150, 333, 3], page=32, kv=2, hd=hd, store=store)
    check_attention(c, 4, q16=q16, window=window)


@pytest.mark.parametrize("window", [0, 200])
@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("hd,q16", [(64, True), (128, True), (128, False), (256, True), (256, False), (512, True),
                                    (512, False)])
def test_attention_chunks_cut_along_their_keys(window, store, hd, q16):
    """Chunks behind prefixes that several workgroups share, heads that several waves share."""
    say("cut chunks", window, store, hd, q16)
    c = po.PagedCase(23, new=[70, 3, 70], ctx=[1500, 700, 70], page=32, kv=1, hd=hd, store=store, pad=2)
    check_attention(c, 3, q16=q16, window=window)


@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("new", [[1, 1], [90, 140]])
def test_attention_scores_that_climb(store, new):
    """Scores that keep passing the running reference, and a scale of 0 and below."""
    c = po.PagedCase(23, new=new, ctx=[700, 300], page=16, kv=1, hd=64, store=store)
    for p in range(700):  # keys grow along the sequence
        pg, s = c.place(0, p)
        if store == "f16":
            c.k[pg, 0, s] *= np.float16(0.02 * p)
        else:
            c.k_scale[pg, 0, s] *= np.float32(0.02 * p)
    for scale in (None, 0.0, -0.3):
        check_attention(c, 2, q16=False, scale=scale)
        check_attention(c, 2, q16=True, scale=scale)


@pytest.mark.parametrize("q16", [False, True])
def test_attention_value_scales_far_apart(q16):
    """8-bit rows whose scales span 2^-60 .. 2^40, growing and falling along the keys."""
    c = po.PagedCase(24, new=[1, 30], ctx=[500, 200], page=16, kv=1, hd=64, store="i8")
    e = np.linspace(-60, 40, 500)
    for p in range(500):
        pg, s = c.place(0, p)
        c.v_scale[pg, 0, s] = np.float32(2.0 ** (e[p] if p % 2 else -20)) if not q16 else np.float32(2.0 ** (e[p] / 8))
    check_attention(c, 3, q16=q16)


@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("q16", [False, True])
@pytest.mark.parametrize("new", [[1, 1, 1], [60, 130, 4]])
def test_attention_without_some_pages(store, q16, new):
    """Missing pages anywhere hide their keys; a row that sees none is zero."""
    c = po.PagedCase(25, new=new, ctx=[200, 260, 4], page=16, kv=2, hd=128, store=store)
    c.table[0, 2] = -1
    c.table[0, 5] = c.n_pages
    c.table[1, :9] = -7  # the first 144 positions: rows there see nothing
    c.table[2, 0] = 1 << 30
    got = check_attention(c, 4, q16=q16)
    assert np.all(got[int(c.cu[2]):int(c.cu[3])] == 0)


@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("hd,new,window", [(128, [1, 1], 0), (128, [50, 140], 0), (64, [50, 140], 33), (256, [50, 1], 0),
                                           (512, [3, 20], 9)])
@pytest.mark.parametrize("q16", [False, True])
def test_attention_takes_nothing_from_what_it_does_not_see(store, hd, new, window, q16):
    """Infinities and NaN behind the sequence's end, in later rows of the batch, before
    the window and in pages of nobody leave every other row's result as it is."""
    c = po.PagedCase(26, new=new, ctx=[150, 260], page=16, kv=1, hd=hd, store=store)
    clean_k, clean_v = c.k.copy(), c.v.copy()
    q = rows(c, 27, 2).reshape(c.tokens, -1)
    dt = torch.float16 if q16 else torch.float32

    def run():
        cache, batch = on_gpu(c)
        return lmx.paged_attention(gpu(q).to(dt), cache, batch, n_heads=2, window=window).float().cpu().numpy()

    base = run()
    own = {c.place(b, p) for b in range(2) for p in range(c.ctx[b])}
    bad = [np.inf, -np.inf, np.nan]
    last = {c.place(b, c.ctx[b] - 1): int(c.cu[b + 1]) - 1 for b in range(2)}
    for page in range(c.n_pages):
        for s in range(16):
            if (page, s) in own and (page, s) not in last:
                continue
            x = bad[(page + s) % 3]
            if store == "f16":
                c.k[page, 0, s, s % hd] = x
                c.v[page, 0, (3 * s) % hd, s] = x
            else:
                c.k_scale[page, 0, s] = c.v_scale[page, 0, s] = x
    if window:  # a key that has left every row's window
        pg, s = c.place(1, 260 - new[1] - window - 2)
        if store == "f16":
            c.v[pg, 0, :, s] = np.nan
        else:
            c.v_scale[pg, 0, s] = np.nan
    got = run()
    keep = np.ones(c.tokens, bool)
    keep[list(last.values())] = False  # the rows that do see a bad key
    assert np.array_equal(got[keep], base[keep])
    assert not np.all(np.isfinite(got[~keep]), axis=1).any()
    c.k, c.v = clean_k, clean_v


def test_attention_gives_infinities_to_the_rows_that_see_them():
    c = po.PagedCase(28, new=[40], ctx=[40], page=16, kv=1, hd=64)
    pg, s = c.place(0, 17)
    c.v[pg, 0, 5, s], c.v[pg, 0, 9, s] = np.inf, -np.inf
    cache, batch = on_gpu(c)
    for dt in (torch.float32, torch.float16):
        q = gpu(rows(c, 29, 1).reshape(40, -1)).to(dt)
        got = lmx.paged_attention(q, cache, batch, n_heads=1).cpu().numpy()
        assert np.all(np.isfinite(got[:17])) and np.all(got[17:, 5] == np.inf) and np.all(got[17:, 9] == -np.inf)
        assert np.all(np.isfinite(np.delete(got, [5, 9], 1)))


@pytest.mark.parametrize("hd", [128, 256, 512])
def test_attention_gives_infinities_to_their_dims(hd):
    """Each part of a head that a wave has, in chunks and in single tokens."""
    dims = [3, hd // 4 + 40, hd // 2 + 7, hd - 1]
    for new in ([60], [2]):
        c = po.PagedCase(28, new=new, ctx=[60], page=16, kv=1, hd=hd)
        n = new[0]
        pg, s = c.place(0, 59)
        c.v[pg, 0, dims, s] = [np.inf, -np.inf, np.nan, np.inf]
        cache, batch = on_gpu(c)
        for dt in (torch.float32, torch.float16):
            q = gpu(rows(c, 29, 1).reshape(n, -1)).to(dt)
            got = lmx.paged_attention(q, cache, batch, n_heads=1).cpu().numpy()
            assert np.all(np.isfinite(got[:-1])) and np.all(np.isfinite(np.delete(got, dims, 1)))
            assert np.array_equal(got[-1, dims], [np.inf, -np.inf, np.nan, np.inf], equal_nan=True)


@pytest.mark.parametrize("q16", [False, True])
def test_attention_strided_queries(q16):
    """Queries as columns of a fused row, and heads at a stride, give what dense ones give."""
    c = po.PagedCase(30, new=[9, 200], ctx=[50, 230], page=32, kv=2, hd=128)
    cache, batch = on_gpu(c)
    dt = torch.float16 if q16 else torch.float32
    q = gpu(rows(c, 31, 4).reshape(c.tokens, -1)).to(dt)
    want = lmx.paged_attention(q, cache, batch, n_heads=4)
    fused = torch.full((c.tokens, 2048 + 64), float("nan"), dtype=dt, device="cuda")
    fused[:, 64:64 + 512] = q
    assert torch.equal(lmx.paged_attention(fused[:, 64:64 + 512], cache, batch, n_heads=4), want)
    pair = torch.full((c.tokens, 4, 256), float("nan"), dtype=dt, device="cuda")
    pair[:, :, :128] = q.view(c.tokens, 4, 128)
    assert torch.equal(lmx.paged_attention(pair.view(c.tokens, -1), cache, batch, n_heads=4, q_head_stride=256), want)


def test_attention_large_and_tiny_queries():
    """f32 rows near the ends of f32's range keep 22 bits of every element that counts."""
    c = po.PagedCase(32, new=[6], ctx=[90], page=16, kv=1, hd=64)
    cache, batch = on_gpu(c)
    q = rows(c, 33, 1)
    base, mag, prod, top = po.attend(c, q, heads=1, scale=0.1)
    bound = po.attend_bound(c, mag, prod, top, 90, f32=True)
    for e in (-90, -20, 30, 90):
        got = lmx.paged_attention(gpu((q * 2.0 ** e).astype(np.float32).reshape(6, -1)), cache, batch, n_heads=1,
                                  scale=0.1 * 2.0 ** -e).cpu().numpy().reshape(base.shape)
        assert np.all(np.abs(got - base) <= bound), e


@pytest.mark.parametrize("n_seq", [65, 200])
@pytest.mark.parametrize("store", ["f16", "i8"])
def test_many_sequences(n_seq, store):
    """More sequences than a wave has lanes: write, read back and attend."""
    rng = np.random.default_rng(34)
    new = [int(x) for x in rng.choice([0, 1, 1, 1, 2, 20], n_seq)]
    new[3] = 37
    ctx = [max(n, int(x)) for n, x in zip(new, rng.integers(1, 90, n_seq))]
    ctx[5] = 700
    c = po.PagedCase(35, new=new, ctx=ctx, page=16, kv=1, hd=64, store=store, pad=5)
    k, v = rows(c, 36, 1), rows(c, 37, 1)
    c.k, c.v, c.k_scale, c.v_scale = po.append(c, k, v)
    cache, batch = on_gpu(c)
    lmx.paged_append(gpu(k.reshape(c.tokens, -1)), gpu(v.reshape(c.tokens, -1)), cache, batch)
    assert np.array_equal(cache.k.cpu().numpy(), c.k) and np.array_equal(cache.v.cpu().numpy(), c.v)
    back, _ = lmx.paged_read(cache, batch)
    for row, b, pos, at in c.row_places():
        assert np.array_equal(back[row].cpu().numpy(), c.held(b, 0, pos)[0].astype(np.float32))
    check_attention(c, 3, q16=False)
    check_attention(c, 3, q16=True)


def test_shared_prefix_pages():
    """Two sequences over the same pages of a prefix give what two copies give."""
    c = po.PagedCase(38, new=[1, 1], ctx=[100, 100], page=16, kv=1, hd=128)
    for e in range(6):
        a, b = c.table[0, e], c.table[1, e]
        c.k[b], c.v[b] = c.k[a], c.v[a]
    q = gpu(rows(c, 39, 2).reshape(2, -1))
    want = lmx.paged_attention(q, *on_gpu(c), n_heads=2)
    c.table[1, :6] = c.table[0, :6]
    assert torch.equal(lmx.paged_attention(q, *on_gpu(c), n_heads=2), want)


def test_offsets_past_32_bits():
    """Pages behind 2^31 elements of the pool are written, read and attended at their places."""
    kv, hd, page = 8, 256, 256
    n_pages = (1 << 31) // (kv * hd * page) + 3
    k = torch.empty((n_pages, kv, page, hd), dtype=torch.float16, device="cuda")
    v = torch.empty((n_pages, kv, hd, page), dtype=torch.float16, device="cuda")
    c = po.PagedCase(40, new=[40], ctx=[40], page=page, kv=kv, hd=hd, spare=0)
    c.table[0, 0] = n_pages - 1
    x, y = rows(c, 41, kv), rows(c, 42, kv)
    batch = lmx.PagedBatch(gpu(c.cu), gpu(np.array(c.ctx, np.int32)), gpu(c.table), n_tokens=40, max_new=40, max_ctx=40)
    big = lmx.PagedCache(k, v)
    lmx.paged_append(gpu(x.reshape(40, -1)), gpu(y.reshape(40, -1)), big, batch)
    assert np.array_equal(k[-1, :, :40].cpu().numpy(), x.transpose(1, 0, 2).astype(np.float16))
    assert np.array_equal(v[-1, :, :, :40].cpu().numpy(), y.transpose(1, 2, 0).astype(np.float16))
    kb, vb = lmx.paged_read(big, batch, dtype=torch.float16)
    assert np.array_equal(kb.cpu().numpy(), x.reshape(40, -1).astype(np.float16))
    assert np.array_equal(vb.cpu().numpy(), y.reshape(40, -1).astype(np.float16))
    q = gpu(rows(c, 43, kv).reshape(40, -1))
    got = lmx.paged_attention(q, big, batch, n_heads=kv)
    small = lmx.PagedCache(k[-1:].contiguous(), v[-1:].contiguous())
    batch.page_table.zero_()
    assert torch.equal(lmx.paged_attention(q, small, batch, n_heads=kv), got)


# -------------------------------------------------------- streams and graphs --
def test_the_path_replays_from_a_graph_with_new_lengths():
    """prologue and attention captured once, replayed while the sequences grow, with
    eager work between: every replay against the eager calls."""
    page, kv, hd, heads = 16, 2, 128, 8
    c = po.PagedCase(44, new=[1, 1, 1], ctx=[60, 100, 9], page=page, kv=kv, hd=hd, store="i8", extra_entries=40, spare=130)
    free = [p for p in range(c.n_pages) if p not in set(c.table.ravel().tolist())]
    for b in range(3):
        for e in range(c.stride):
            if c.table[b, e] < 0:
                c.table[b, e] = free.pop()
    cache, _ = on_gpu(c)
    twin, _ = on_gpu(c)
    cu, table = gpu(c.cu), gpu(c.table)
    ctx = gpu(np.array(c.ctx, np.int32))
    batch = lmx.PagedBatch(cu, ctx, table, n_tokens=3, max_new=1, max_ctx=640)
    fused = torch.zeros(3, (heads + 2 * kv) * hd, device="cuda")
    nq, nk = heads * hd, kv * hd
    ws, ws2 = lmx.Workspace(), lmx.Workspace()

    def path(cache, ws):
        q = lmx.paged_prologue(fused[:, :nq], fused[:, nq:nq + nk], fused[:, nq + nk:], cache, batch, n_heads=heads)
        return lmx.paged_attention(q, cache, batch, n_heads=heads, workspace=ws)

    path(twin, ws2)  # sizes the workspaces; both caches have the same past
    path(cache, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = path(cache, ws)
    for step in range(5):
        fused.copy_(torch.randn(fused.shape, generator=torch.Generator().manual_seed(step)))
        ctx += torch.tensor([1, 100 if step == 2 else 1, 1], dtype=torch.int32, device="cuda")
        graph.replay()
        got = out.clone()
        want = path(twin, ws2)
        torch.cuda.synchronize()
        assert torch.equal(got, want), step
        assert torch.equal(cache.k, twin.k) and torch.equal(cache.v, twin.v)


def test_calls_on_another_stream():
    c = po.PagedCase(45, new=[1, 30], ctx=[900, 200], page=32, kv=2, hd=128)
    cache, batch = on_gpu(c)
    q = gpu(rows(c, 46, 4).reshape(c.tokens, -1))
    want = lmx.paged_attention(q, cache, batch, n_heads=4)
    wk, wv = lmx.paged_read(cache, batch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = lmx.paged_attention(q, cache, batch, n_heads=4, stream=side)
    gk, gv = lmx.paged_read(cache, batch, stream=side)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(gk, wk) and torch.equal(gv, wv)


def test_two_streams_at_once():
    """Calls that overlap in time, a workspace each, on pages that both read."""
    c = po.PagedCase(47, new=[200, 1, 1], ctx=[3000, 2500, 700], page=16, kv=2, hd=128, store="i8")
    cache, batch = on_gpu(c)
    qs = [gpu(rows(c, s, 4).reshape(c.tokens, -1)) for s in (48, 49)]
    want = [lmx.paged_attention(q, cache, batch, n_heads=4) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    spaces = [lmx.Workspace() for _ in qs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        got = [lmx.paged_attention(q, cache, batch, n_heads=4, workspace=ws, stream=s)
               for q, ws, s in zip(qs, spaces, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_a_workspace_serves_calls_of_other_shapes():
    """Partials that one call leaves do not reach the next."""
    ws = lmx.Workspace()
    for new, ctx in (([1, 1], [900, 300]), ([20], [400]), ([1], [130]), ([1, 1, 1], [70, 1000, 2])):
        check_attention(po.PagedCase(47, new=new, ctx=ctx, page=16, kv=2, hd=128), 4, q16=False, ws=ws)


def test_the_same_call_gives_the_same_bits():
    c = po.PagedCase(48, new=[1, 70, 1], ctx=[1500, 90, 800], page=16, kv=2, hd=128, store="i8")
    cache, batch = on_gpu(c)
    q = gpu(rows(c, 49, 8).reshape(c.tokens, -1))
    first = lmx.paged_attention(q, cache, batch, n_heads=8)
    for _ in range(3):
        assert torch.equal(lmx.paged_attention(q, cache, batch, n_heads=8), first)


# ------------------------------------------------------------------ together --
@pytest.mark.parametrize("store", ["f16", "i8"])
def test_a_prompt_then_tokens_match_one_long_prompt(store):
    """Prologue and attention of a prompt in chunks, then token by token, and the output
    projection, give what the whole prompt at once gives: the same pages, and rows within
    the bounds of their roundings."""
    page, kv, hd, heads, T = 32, 2, 128, 8, 90
    rng = np.random.default_rng(50)
    x = torch.from_numpy(rng.standard_normal((T, (heads + 2 * kv) * hd)).astype(np.float32)).cuda()
    w = torch.from_numpy(rng.standard_normal((256, heads * hd)).astype(np.float32) * 0.03).cuda()
    nq, nk = heads * hd, kv * hd
    dt = torch.int8 if store == "i8" else torch.float16

    def run(cuts):
        cache = lmx.PagedCache.empty(3, page_size=page, n_kv_heads=kv, head_dim=hd, dtype=dt)
        table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
        outs, at = [], 0
        for n in cuts:
            y = x[at:at + n]
            at += n
            batch = lmx.PagedBatch(torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                                   torch.tensor([at], dtype=torch.int32, device="cuda"), table, n_tokens=n, max_new=n,
                                   max_ctx=at)
            q = lmx.paged_prologue(y[:, :nq], y[:, nq:nq + nk], y[:, nq + nk:], cache, batch, n_heads=heads)
            o = lmx.paged_attention(q, cache, batch, n_heads=heads)
            outs.append((q, o, lmx.matvec(w.view(torch.uint8), o, qtype="f32", rows=256, in_dim=nq)))
        k, v = lmx.paged_read(cache, lmx.PagedBatch(torch.tensor([0, T], dtype=torch.int32, device="cuda"),
                                                    torch.tensor([T], dtype=torch.int32, device="cuda"), table,
                                                    n_tokens=T, max_new=T, max_ctx=T))
        return [torch.cat(t) for t in zip(*outs)] + [k, v]

    whole, parts = run([T]), run([40, 33] + [1] * 17)
    for i in (0, 3, 4):  # q and the pages: the same arithmetic whatever the batch
        assert torch.equal(whole[i], parts[i])
    c = po.PagedCase(51, new=[T], ctx=[T], page=page, kv=kv, hd=hd, spare=0)
    pos = np.arange(T)
    for name, src in (("k", whole[3]), ("v", whole[4])):  # the pages' values, in f64 through held()
        setattr(c, "_" + name, src.cpu().numpy().reshape(T, kv, hd).astype(np.float64))
    c.held = lambda b, h, p: (c._k[p, h], c._v[p, h])
    c.store = store
    c.v_scale = np.full((c.n_pages, kv, page), np.abs(c._v).max() / 127)
    want, mag, prod, top = po.attend(c, whole[0].cpu().numpy().reshape(T, heads, hd), heads=heads)
    bound = po.attend_bound(c, mag, prod, top, T, f32=True)
    for r in (whole, parts):
        o = r[1].cpu().numpy().reshape(T, heads, hd)
        assert np.all(np.abs(o - want) <= bound)
        y = want.reshape(T, -1) @ w.double().cpu().numpy().T
        lim = (bound.reshape(T, -1) + nq * 2.0 ** -24 * np.abs(want.reshape(T, -1))) @ np.abs(w.double().cpu().numpy().T)
        assert np.all(np.abs(r[2].cpu().numpy() - y) <= lim)
    assert pos[-1] == T - 1


def test_python_refusals():
    c = po.PagedCase(52, new=[2], ctx=[20], page=16, kv=1, hd=64)
    cache, batch = on_gpu(c)
    good = torch.zeros(2, 64, device="cuda")
    with pytest.raises(TypeError):
        lmx.paged_append(good.double(), good.double(), cache, batch)
    with pytest.raises(ValueError):
        lmx.paged_append(good, good.half(), cache, batch)
    with pytest.raises(ValueError):
        lmx.paged_append(good[:1], good[:1], cache, batch)
    with pytest.raises(ValueError):
        lmx.paged_append(None, None, cache, batch)
    with pytest.raises(ValueError):
        lmx.paged_append(good.cpu(), good.cpu(), cache, batch)
    with pytest.raises(ValueError):
        lmx.paged_attention(torch.zeros(2, 100, device="cuda"), cache, batch, n_heads=2)
    with pytest.raises(ValueError):
        lmx.paged_attention(good, cache, batch, n_heads=1, out=torch.zeros(2, 64, device="cuda").half())
    with pytest.raises(lmx.LmxError):
        lmx.paged_attention(good, cache, batch, n_heads=1, out=good)
    with pytest.raises(TypeError):
        lmx.PagedCache(cache.k.float(), cache.v.float())
    with pytest.raises(ValueError):
        lmx.PagedCache(cache.k, cache.k)
    with pytest.raises(ValueError):
        lmx.PagedCache(cache.k.to(torch.int8), cache.v.to(torch.int8))
    with pytest.raises(TypeError):
        lmx.PagedBatch(batch.cu.long(), batch.ctx_lens, batch.page_table, n_tokens=2, max_new=2, max_ctx=20)
    with pytest.raises(lmx.LmxError):  # max_ctx beyond the table
        big = lmx.PagedBatch(batch.cu, batch.ctx_lens, batch.page_table, n_tokens=2, max_new=2, max_ctx=1000)
        lmx.paged_append(good, good, cache, big)
