"""The paged cache on batches and contexts long enough for every loop of its kernels:
several heads a workgroup in write, read-back and prologue, walks past one window of 64
pages, and joins of more splits than one pass takes.  Against the float64 definitions,
attention at sampled rows."""
import numpy as np
import pytest

from tests import paged_oracle as po

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import llmoxide_amd as lmx  # noqa: E402
from tests.test_gpu_paged import gpu, on_gpu, rows, say  # noqa: E402


# ------------------------------------------------- write, read-back, prologue --
LENS = dict(new=[700, 1, 0, 461], ctx=[731, 5, 9, 461], pad=3)  # 1165 rows


def places(c):
    """(rows, positions, pages, slots) of the batch's rows."""
    got = [(r, pos, *at) for r, _, pos, at in c.row_places()]
    return [np.array(x) for x in zip(*got)]


def stored(c, k, v):
    """The pools after float rows are stored: as po.append, all rows at once."""
    r, _, pg, sl = places(c)
    out = []
    for pool, scale, x, last in ((c.k, c.k_scale, k, False), (c.v, c.v_scale, v, True)):
        pool = pool.copy()
        x = x[r]  # [rows, kv, hd]
        if c.store == "i8":
            s = (np.abs(x).max(-1).astype(np.float64) / 127).astype(np.float32)
            scale = scale.copy()
            scale[pg, :, sl] = s
            x = np.rint(x.astype(np.float64) / s.astype(np.float64)[..., None])
        for i in range(len(r)):
            if last:
                pool[pg[i], :, :, sl[i]] = x[i].astype(pool.dtype)
            else:
                pool[pg[i], :, sl[i]] = x[i].astype(pool.dtype)
        out += [pool, scale]
    return out[0], out[2], out[1], out[3]


@pytest.mark.parametrize("hd,page,kv", [(64, 16, 3), (128, 64, 5), (256, 32, 3), (512, 16, 3)])
@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("src", [torch.float32, torch.float16])
def test_long_batches_are_written_and_read_back(hd, page, kv, store, src):
    say("long append", hd, page, kv, store, src)
    c = po.PagedCase(70, page=page, kv=kv, hd=hd, store=store, **LENS)
    k, v = (gpu(rows(c, s, kv)).to(src).float().cpu().numpy() for s in (71, 72))
    cache, batch = on_gpu(c)
    lmx.paged_append(gpu(k.reshape(c.tokens, -1)).to(src), gpu(v.reshape(c.tokens, -1)).to(src), cache, batch)
    want = stored(c, k, v)
    for got, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):
        assert w is None or np.array_equal(got.cpu().numpy(), w)
    r, _, pg, sl = places(c)
    for out in (torch.float32, torch.float16):
        back = [torch.full((c.tokens, kv * hd), 7.0, dtype=out, device="cuda") for _ in range(2)]
        lmx.paged_read(cache, batch, k_out=back[0], v_out=back[1])
        for got, pool, scale, last in ((back[0], want[0], want[2], False), (back[1], want[1], want[3], True)):
            x = pool[pg, :, :, sl] if last else pool[pg, :, sl]
            x = x.astype(np.float32) * (scale[pg, :, sl][..., None] if store == "i8" else np.float32(1))
            w = np.full((c.tokens, kv, hd), 7.0, np.float32)
            w[r] = x  # int * scale is rounded to f32, and for f16 once more
            np_out = np.float16 if out == torch.float16 else np.float32
            assert np.array_equal(got.cpu().numpy().reshape(w.shape), w.astype(np_out))


def turned(x, gain, pos, n_rot, base):
    """po.rope_norm of heads x [rows, heads, hd] at once."""
    x = x.astype(np.float64)
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * gain.astype(np.float64)
    half = n_rot // 2
    a = pos[:, None, None] * float(base) ** (-2.0 * np.arange(half) / n_rot)
    y = x.copy()
    y[..., :half] = x[..., :half] * np.cos(a) - x[..., half:n_rot] * np.sin(a)
    y[..., half:n_rot] = x[..., :half] * np.sin(a) + x[..., half:n_rot] * np.cos(a)
    return y


@pytest.mark.parametrize("hd,n_rot,page,kv,heads", [(64, 64, 16, 3, 9), (128, 128, 32, 2, 10), (128, 48, 16, 3, 9),
                                                    (256, 256, 16, 1, 7), (512, 512, 64, 3, 6)])
@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("q16", [False, True])
def test_long_batches_through_the_prologue(hd, n_rot, page, kv, heads, store, q16):
    """Four heads a workgroup and a last group of fewer, the angles kept from head to head."""
    say("long prologue", hd, n_rot, page, kv, heads, store, q16)
    c = po.PagedCase(73, page=page, kv=kv, hd=hd, store=store, **LENS)
    q, k, v = rows(c, 74, heads, 2.0), rows(c, 75, kv, 0.5), rows(c, 76, kv)
    qg, kg = (1 + 0.2 * np.random.default_rng(77).standard_normal((2, hd))).astype(np.float32)
    cache, batch = on_gpu(c)
    fused = torch.cat([gpu(x.reshape(c.tokens, -1)) for x in (q, k, v)], 1)
    nq, nk = heads * hd, kv * hd
    out = torch.full((c.tokens, nq), 9.0, dtype=torch.float16 if q16 else torch.float32, device="cuda")
    lmx.paged_prologue(fused[:, :nq], fused[:, nq:nq + nk], fused[:, nq + nk:], cache, batch, n_heads=heads, n_rot=n_rot,
                       rope_base=5e5, q_gain=gpu(qg), k_gain=gpu(kg), q_out=out, v_norm=hd == 256)
    r, pos, pg, sl = places(c)
    rel = (hd + 32) * 2.0 ** -24  # as for short batches: the row's sum, its root, the turn
    got = out.float().cpu().numpy().reshape(c.tokens, heads, hd)
    want = turned(q[r], qg, pos, n_rot, 5e5)
    tol = 2 * rel * np.abs(want).max(-1, keepdims=True) + (2.0 ** -11 * np.abs(want) + 2.0 ** -24 if q16 else 0)
    assert np.all(np.abs(got[r] - want) <= tol)
    others = np.setdiff1d(np.arange(c.tokens), r)
    assert len(others) == 3 and np.all(got[others] == 9)
    one = np.ones(hd, np.float32) if hd == 256 else None
    K, V = cache.k.float().cpu().numpy(), cache.v.float().cpu().numpy()
    for x, scale, w in ((K[pg, :, sl], cache.k_scale, turned(k[r], kg, pos, n_rot, 5e5)),
                        (V[pg, :, :, sl], cache.v_scale, turned(v[r], one, pos, 0, 5e5))):
        big = np.abs(w).max(-1, keepdims=True)
        if store == "f16":
            assert np.all(np.abs(x - w) <= 2 * rel * big + 2.0 ** -11 * np.abs(w) + 2.0 ** -24)
        else:  # half a step of the scale, and the f32 steps before it
            s = scale.cpu().numpy()[pg, :, sl][..., None].astype(np.float64)
            assert np.all(np.abs(s - big / 127) <= 4 * rel * big / 127)
            assert np.all(np.abs(x * s - w) <= (0.5 + 1e-3) * s + 4 * rel * big)


# ----------------------------------------------------------------- attention --
def one_long(seed, *, ctx, new, **kw):
    return po.PagedCase(seed, new=[new], ctx=[ctx], **kw)


def shared(c, ctx):
    """As many sequences of one new token over c's pages as ``ctx`` has lengths."""
    n = len(ctx)
    c.table = np.repeat(c.table[:1], n, 0)
    c.new, c.ctx, c.rows, c.tokens = [1] * n, list(ctx), n, n
    c.cu = np.arange(n + 1, dtype=np.int32)
    return c


def check_rows(c, heads, picks, *, q16, window=0, seed=80, at_v=None):
    """paged_attention against the definition at rows ``picks`` ((sequence, row of it));
    at_v: (position, dim) where V is +inf in every head."""
    if at_v:
        pg, s = c.place(0, at_v[0])
        c.v[pg, :, at_v[1], s] = np.inf
    cache, batch = on_gpu(c)
    q = rows(c, seed, heads)
    dt = torch.float16 if q16 else torch.float32
    if q16:
        q = q.astype(np.float16).astype(np.float32)
    got = lmx.paged_attention(gpu(q.reshape(c.tokens, -1)).to(dt), cache, batch, n_heads=heads, window=window)
    got = got.float().cpu().numpy().reshape(c.tokens, heads, c.hd).astype(np.float64)
    G = heads // c.kv
    assert np.all(np.isfinite(np.delete(got, at_v[1] if at_v else [], 2)))
    for b, j in picks:
        r = int(c.cu[b]) + j
        pos = c.ctx[b] - c.new[b] + j
        p = np.arange(max(0, pos - window + 1) if window else 0, pos + 1)
        pg, sl = c.table[b, p // c.page], p % c.page
        out, mag = np.zeros((heads, c.hd)), np.zeros((heads, c.hd))
        prod, top = np.zeros(heads), np.zeros(heads)
        for h in range(c.kv):
            K, V = c.k[pg, h, sl].astype(np.float64), c.v[pg, h, :, sl].astype(np.float64)
            if c.store == "i8":
                K, V = K * c.k_scale[pg, h, sl][:, None], V * c.v_scale[pg, h, sl][:, None]
            V = np.where(np.isfinite(V), V, 0)
            for g in range(G):
                x = q[r, h * G + g].astype(np.float64)
                s = K @ x / np.sqrt(c.hd)
                w = np.exp(s - s.max())
                w /= w.sum()
                i = h * G + g
                out[i], mag[i], prod[i] = w @ V, w @ np.abs(V), (np.abs(K) @ np.abs(x)).max() / np.sqrt(c.hd)
                # in 8 bits the largest scale's, seen by this row or by one beside it
                top[i] = 127 * float(c.v_scale.max()) if c.store == "i8" else np.abs(V).max()
        bound = po.attend_bound(c, mag, prod, top, len(p), f32=not q16)
        off = np.abs(got[r] - out) - bound
        if at_v:
            sees = p[0] <= at_v[0] <= pos
            assert np.all(got[r][:, at_v[1]] == np.inf) == sees, (b, j)
            off = np.delete(off, at_v[1], 1) if sees else off
        assert off.max() <= 0, (b, j, off.max())


@pytest.mark.parametrize("hd,kv,heads,new", [(64, 8, 32, 1100), (128, 8, 32, 1100), (256, 8, 32, 1100), (512, 4, 8, 1100)])
@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("q16", [False, True])
def test_a_chunk_that_walks_past_a_window_of_pages(hd, kv, heads, new, store, q16):
    """More tiles than are split (512 workgroups start at once at most, half as many at 512 dims;
    two splits a tile would not), on 16-slot pages: a walk of 2700 keys takes three windows of
    64 pages."""
    assert 2 * kv * -(-new * (heads // kv) // (64 if hd == 512 else 128)) > (256 if hd == 512 else 512)
    say("long walk", hd, kv, heads, new, store, q16)
    c = one_long(81, ctx=2700, new=new, page=16, kv=kv, hd=hd, store=store)
    check_rows(c, heads, [(0, j) for j in (0, 1, 31, 447, 448, 640, new - 1)], q16=q16)


@pytest.mark.parametrize("q16", [False, True])
@pytest.mark.parametrize("window", [0, 1500])
def test_an_infinity_behind_the_first_window_of_pages(q16, window):
    c = one_long(82, ctx=2700, new=1100, page=16, kv=8, hd=64)
    check_rows(c, 32, [(0, j) for j in (0, 398, 399, 400, 1099)], q16=q16, window=window, at_v=(1999, 17))


@pytest.mark.parametrize("hd,kv,n_seq", [(64, 8, 64), (128, 8, 64), (256, 4, 64), (512, 4, 32)])
@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("q16", [False, True])
def test_steps_whose_splits_pass_a_window_of_pages(hd, kv, n_seq, store, q16):
    """So many sequences (over the same pages) that a split is longer than 64 pages of 16."""
    say("long splits", hd, kv, n_seq, store, q16)
    c = one_long(83, ctx=3000, new=1, page=16, kv=kv, hd=hd, store=store)
    units = sum(-(-(3000 - 7 * b) // 64) for b in range(n_seq)) * kv
    assert units / (1024 if hd <= 128 else 512 if hd == 256 else 256) > 17  # units of 64 keys a split
    c = shared(c, [3000 - 7 * b for b in range(n_seq)])
    check_rows(c, 2 * kv, [(b, 0) for b in (0, 1, 15, n_seq - 1)], q16=q16)


@pytest.mark.parametrize("q16", [False, True])
def test_an_infinity_behind_the_first_window_of_a_split(q16):
    c = shared(one_long(84, ctx=3000, new=1, page=16, kv=8, hd=64), [3000 - 7 * b for b in range(64)])
    check_rows(c, 8, [(b, 0) for b in (0, 20, 63)], q16=q16, at_v=(1300, 50))


@pytest.mark.parametrize("hd,ctx", [(64, 68000), (128, 36000), (256, 19000), (512, 9000)])
@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("q16", [False, True])
def test_a_token_whose_splits_take_the_merge_two_passes(hd, ctx, store, q16):
    """One kv head: 8 units (512 dims: 4) a split, more splits than a pass of the merge has."""
    say("many splits", hd, ctx, store, q16)
    splits = -(-(-(-ctx // 64)) // (4 if hd == 512 else 8))
    assert splits > 8 * (1024 // hd)
    check_rows(one_long(85, ctx=ctx, new=1, page=256, kv=1, hd=hd, store=store), 3, [(0, 0)], q16=q16)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("q16", [False, True])
def test_a_chunk_whose_splits_take_the_merge_several_passes(hd, store, q16):
    say("many splits of a chunk", hd, store, q16)
    c = one_long(86, ctx=6000, new=140, page=32, kv=1, hd=hd, store=store)
    check_rows(c, 2, [(0, 0), (0, 63), (0, 64), (0, 139)], q16=q16)
