"""The paged cache's attention where its numbers, lengths and grids reach their
limits, against the float64 definitions (paged_oracle)."""
import numpy as np
import pytest

from tests import paged_oracle as po

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import llmoxide_amd as lmx  # noqa: E402
from tests.test_gpu_paged import check_attention, gpu, on_gpu, rows, say  # noqa: E402


# ------------------------------------------------------------ 8-bit V scales --
def quiet_and_loud(c, b, quiet, loud):
    """Sequence b's V rows: zeros where ``quiet``, a scale of 2^loud elsewhere."""
    for p in range(c.ctx[b]):
        pg, s = c.place(b, p)
        c.v_scale[pg, 0, s] = 0 if quiet(p) else np.float32(2.0 ** loud)
        if quiet(p):
            c.v[pg, 0, :, s] = 0


@pytest.mark.parametrize("loud", [20, 47, 100])
@pytest.mark.parametrize("quiet", ["first half", "every second", "all but one", "last half"])
@pytest.mark.parametrize("new", [[1, 3], [60, 130]])
@pytest.mark.parametrize("hd", [64, 512])
def test_zero_values_keep_their_share_beside_loud_ones(hd, new, quiet, loud):
    """Rows of zeros (scale 0) beside values up to 2^107: each key has its share of the
    softmax's sum, whichever comes first, in one walk and where several join."""
    say("zero values", hd, new, quiet, loud)
    c = po.PagedCase(60, new=new, ctx=[900, 140], page=16, kv=1, hd=hd, store="i8")
    for b in range(2):
        n = c.ctx[b]
        at = {"first half": lambda p: p < n // 2, "every second": lambda p: p % 2 == 0,
              "all but one": lambda p: p != 5, "last half": lambda p: p >= n // 2}[quiet]
        quiet_and_loud(c, b, at, loud)
    check_attention(c, 2, q16=False)
    check_attention(c, 2, q16=False, scale=0.0)  # a plain mean


def test_zero_values_of_half_precision_rows():
    for new in ([1, 3], [60, 130]):
        c = po.PagedCase(61, new=new, ctx=[900, 140], page=16, kv=1, hd=128, store="i8")
        for b in range(2):
            quiet_and_loud(c, b, lambda p: p % 3 != 0, 8)
        check_attention(c, 2, q16=True)


@pytest.mark.parametrize("new", [[2], [150]])
def test_small_values_beside_loud_ones(new):
    """Scales from 2^-80 to 2^100 along the keys, the loud ones at scores far below the
    others': a weight follows score and scale, the sum the score alone."""
    c = po.PagedCase(62, new=new, ctx=[700], page=16, kv=1, hd=64, store="i8")
    for p in range(700):
        pg, s = c.place(0, p)
        c.v_scale[pg, 0, s] = np.float32(2.0 ** (100 if p % 7 == 3 else -80 + p // 8))
        c.k_scale[pg, 0, s] *= np.float32(12 if p % 7 == 3 else 0.5)
    check_attention(c, 2, q16=False)


# ------------------------------------------------------- infinities that are seen --
def attend(c, q, dt, heads, **kw):
    cache, batch = on_gpu(c)
    return lmx.paged_attention(gpu(q.reshape(c.tokens, -1)).to(dt), cache, batch, n_heads=heads, **kw).float().cpu().numpy()


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("new", [[2], [150]])
def test_a_key_whose_score_is_minus_infinity_has_no_weight(new, hd, dt):
    """Infinite elements of f16 keys against queries of both parts' signs: as a key of a
    score so low that its weight is 0; nothing but such keys leaves zeros."""
    say("minus infinity", new, hd, dt)
    c = po.PagedCase(63, new=new, ctx=[600], page=16, kv=1, hd=hd)
    q = rows(c, 64, 2)
    q[..., 7] = np.abs(q[..., 7]) + 0.5
    q[..., 9] = -np.abs(q[..., 9]) - 0.5
    places = [c.place(0, p) for p in (0, 3, 17, 300, 430, 449)]
    for x in (60000, np.inf):  # a score of -60000 / 2 / sqrt(512) and below: exp is 0
        for i, (pg, s) in enumerate(places):
            c.k[pg, 0, s] = 0
            c.k[pg, 0, s, 7 if i % 2 else 9] = -x if i % 2 else x
            if i > 3:
                c.k[pg, 0, s, 9 if i % 2 else 7] = x if i % 2 else -x
        got = attend(c, q, dt, 2)
        if np.isfinite(x):
            want = got
    assert np.all(np.isfinite(want)) and np.array_equal(got, want)
    c.k[:, 0, :, 7] = -np.inf
    assert np.all(attend(c, q, dt, 2) == 0)


@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("new", [[2], [150]])
def test_infinite_queries(store, new):
    """A row that is infinite where every key is positive: every score is -inf, the row zero;
    +inf: not a number.  The other heads and rows are as they are without it."""
    c = po.PagedCase(65, new=new, ctx=[200], page=16, kv=1, hd=64, store=store)
    c.k[:, 0, :, 5] = np.maximum(np.abs(c.k[:, 0, :, 5]), 1)
    q = rows(c, 66, 3, 3e3)
    base = attend(c, q, torch.float32, 3).reshape(c.tokens, 3, 64)
    q[1, 0, 5], q[1, 2, 5] = -np.inf, np.inf
    q[1, 0, 6] = 1e9
    got = attend(c, q, torch.float32, 3).reshape(c.tokens, 3, 64)
    assert np.all(got[1, 0] == 0) and np.all(np.isnan(got[1, 2]))
    assert np.array_equal(got[:, 1], base[:, 1])
    keep = np.arange(c.tokens) != 1
    assert np.array_equal(got[keep], base[keep])


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("new", [[2], [150]])
def test_infinite_values_of_small_weight_survive_a_join(new, dt):
    """V's infinities at keys whose scores lie hundreds below the rest of the row's: those
    of one wave's share, and of one split's."""
    say("joined infinities", new, dt)
    c = po.PagedCase(67, new=new, ctx=[64] if new == [2] else [1500], page=16, kv=1, hd=64)
    low, at = (range(32, 64), 40) if new == [2] else (range(0, 1300), 700)
    q = rows(c, 68, 2)
    q[..., 3] = np.abs(q[..., 3]) + 1
    for p in low:  # 4800 / 8 below in natural units
        pg, s = c.place(0, p)
        c.k[pg, 0, s, 3] = -4800
    base = attend(c, q, dt, 2).reshape(c.tokens, 2, 64)
    pg, s = c.place(0, at)
    c.v[pg, 0, 11, s], c.v[pg, 0, 60, s] = np.inf, -np.inf
    got = attend(c, q, dt, 2).reshape(c.tokens, 2, 64)
    assert np.all(got[..., 11] == np.inf) and np.all(got[..., 60] == -np.inf)
    assert np.array_equal(np.delete(got, [11, 60], 2), np.delete(base, [11, 60], 2))


# ---------------------------------------------------------------- the workspace --
def test_a_workspace_sized_by_a_long_prompt_stays_where_it_is():
    """A prompt that is not split, then a chunk and a token that are."""
    kv, hd, ctx, page = 8, 64, 4200, 64
    entries = -(-ctx // page)
    cache = lmx.PagedCache(torch.randn(entries, kv, page, hd, device="cuda").half(),
                           torch.randn(entries, kv, hd, page, device="cuda").half())
    table = torch.arange(entries, dtype=torch.int32, device="cuda")[None]
    ws, where, q = lmx.Workspace(), None, torch.randn(ctx, kv * hd, device="cuda").half()
    for n in (ctx, 300, 1):
        batch = lmx.PagedBatch(torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                               torch.tensor([ctx], dtype=torch.int32, device="cuda"), table, n_tokens=n, max_new=n, max_ctx=ctx)
        out = lmx.paged_attention(q[-n:], cache, batch, n_heads=kv, workspace=ws)
        where = where or ws.base
        assert ws.base == where
        if n == ctx:
            whole = out
    # the same rows: each within 2^-11 of weights and of the result, values below 6
    assert (out[-1].float() - whole[-1].float()).abs().max() <= 6 * 3 * 2.0 ** -11


# ------------------------------------------------------ garbage that nobody sees --
@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("name,new,ctx,window", [
    ("a step", [1] * 8, [8190 - 7 * i for i in range(8)], 0), ("a chunk", [700], [8190], 0),
    ("a chunk in a window", [700], [8190], 1000), ("a step in a window", [1, 1], [8190, 5001], 1000),
])
def test_garbage_in_unseen_slots_costs_nothing(name, new, ctx, window, dt):
    """NaN and infinities in every slot that no row sees (behind the lengths, before the
    windows, in pages of nobody) leave the bits and the time as they are.  (An infinity that
    a row sees asks for a walk over its keys one by one, which takes many times as long.)"""
    say("unseen garbage", name, dt)
    page, kv, hd, heads = 16, 2, 128, 8
    per = [-(-x // page) for x in ctx]
    order = torch.randperm(sum(per) + 3, generator=torch.Generator().manual_seed(1)).int()
    table = torch.full((len(ctx), max(per)), -1, dtype=torch.int32)
    seen = torch.zeros(sum(per) + 3, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
        lo = max(0, ctx[b] - new[b] - window + 1) if window else 0
        p = torch.arange(lo, ctx[b])
        seen[table[b, p // page].long(), p % page] = True
    g = torch.Generator("cuda").manual_seed(2)
    k = torch.randn(sum(per) + 3, kv, page, hd, device="cuda", generator=g).half()
    v = torch.randn(sum(per) + 3, kv, hd, page, device="cuda", generator=g).half()
    q = torch.randn(sum(new), heads * hd, device="cuda", generator=g).to(dt)
    cu = torch.tensor([0] + new).cumsum(0).int().cuda()
    batch = lmx.PagedBatch(cu, torch.tensor(ctx, dtype=torch.int32, device="cuda"), table.cuda(), n_tokens=sum(new),
                           max_new=max(new), max_ctx=max(ctx))
    ws = lmx.Workspace()
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda").half()

    def run(k, v):
        cache, times = lmx.PagedCache(k, v), []
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(5):
                out = lmx.paged_attention(q, cache, batch, n_heads=heads, window=window, workspace=ws)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b) / 5)
        return out, min(times)

    clean, fast = run(k, v)
    hide = ~seen.cuda()
    fill = bad[torch.arange(hide.numel(), device="cuda") % 3].view(hide.shape)
    k = torch.where(hide[:, None, :, None], fill[:, None, :, None], k)
    v = torch.where(hide[:, None, None, :], fill[:, None, None, :], v)
    got, slow = run(k, v)
    say(f"{fast * 1e3:.1f} us, with garbage {slow * 1e3:.1f}")
    assert torch.equal(got, clean)
    assert slow <= 1.5 * fast


def test_a_window_that_hides_nothing_gives_the_bits_of_none():
    kv, hd, n, page = 8, 64, 2500, 64
    entries = -(-n // page)
    cache = lmx.PagedCache(torch.randn(entries, kv, page, hd, device="cuda").half(),
                           torch.randn(entries, kv, hd, page, device="cuda").half())
    batch = lmx.PagedBatch(torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                           torch.tensor([n], dtype=torch.int32, device="cuda"),
                           torch.arange(entries, dtype=torch.int32, device="cuda")[None], n_tokens=n, max_new=n, max_ctx=n)
    q = torch.randn(n, kv * hd, device="cuda").half()
    want = lmx.paged_attention(q, cache, batch, n_heads=kv)
    for window in (n, n + 1, 1 << 20):
        assert torch.equal(lmx.paged_attention(q, cache, batch, n_heads=kv, window=window), want)
    assert not torch.equal(lmx.paged_attention(q, cache, batch, n_heads=kv, window=n - 1), want)


# ----------------------------------------------------------- bounds and paddings --
@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("new", [[1, 2, 1], [3, 0, 70]])
def test_rows_in_front_of_the_first_sequence(store, new):
    """cu may begin above 0: rows before it belong to nobody, the others are as without them."""
    lead, kv, hd, heads = 7, 2, 128, 4
    c = po.PagedCase(90, new=new, ctx=[40, 90, 700], page=16, kv=kv, hd=hd, store=store)
    n = c.tokens
    x = {w: gpu(rows(c, 91 + i, h).reshape(n, -1)) for i, (w, h) in enumerate((("q", heads), ("k", kv), ("v", kv)))}

    def padded(t):
        return torch.cat([torch.full((lead, t.shape[1]), float("nan"), dtype=t.dtype, device="cuda"), t])

    def run(pad):
        cache, batch = on_gpu(c)
        a = x
        if pad:
            a = {w: padded(t) for w, t in x.items()}
            batch = lmx.PagedBatch(batch.cu + lead, batch.ctx_lens, batch.page_table, n_tokens=n + lead,
                                   max_new=max(new), max_ctx=700)
        outs = [torch.full((a["q"].shape[0], w), 3.0, device="cuda") for w in (heads * hd, heads * hd, kv * hd, kv * hd)]
        lmx.paged_prologue(a["q"], a["k"], a["v"], cache, batch, n_heads=heads, q_out=outs[0])
        lmx.paged_attention(outs[0], cache, batch, n_heads=heads, out=outs[1])
        lmx.paged_read(cache, batch, k_out=outs[2])
        lmx.paged_read(cache, batch, v_out=outs[3])
        lmx.paged_append(a["v"], a["k"], cache, batch)
        return outs, [cache.k, cache.v]
    (outs, pools), (pad_outs, pad_pools) = run(False), run(True)
    for a, b in zip(outs, pad_outs):
        assert torch.equal(b[lead:], a) and torch.all(b[:lead] == 3)
    assert all(torch.equal(a, b) for a, b in zip(pools, pad_pools))


@pytest.mark.parametrize("store", ["f16", "i8"])
@pytest.mark.parametrize("new", [[1], [40], [64, 2, 1]])
@pytest.mark.parametrize("q16", [False, True])
def test_bounds_above_what_a_batch_brings(store, new, q16):
    """max_new, n_tokens and max_ctx as a captured graph keeps them, the batch far below:
    the plan is that of the bounds, the result the batch's."""
    c = po.PagedCase(94, new=new, ctx=[900, 70, 333][:len(new)], page=16, kv=2, hd=128, store=store, pad=300, extra_entries=400)
    cache, small = on_gpu(c)
    q = rows(c, 95, 8)
    if q16:
        q = q.astype(np.float16).astype(np.float32)
    dt = torch.float16 if q16 else torch.float32
    want, mag, prod, top = po.attend(c, q, heads=8)
    bound = po.attend_bound(c, mag, prod, top, max(c.ctx), f32=not q16)
    own = slice(0, c.rows)
    for most, ctx in ((max(new), 900), (100, 4000), (c.tokens, 7000)):
        batch = lmx.PagedBatch(small.cu, small.ctx_lens, small.page_table, n_tokens=c.tokens, max_new=most, max_ctx=ctx)
        out = torch.full((c.tokens, 8 * 128), 5.0, dtype=dt, device="cuda")
        lmx.paged_attention(gpu(q.reshape(c.tokens, -1)).to(dt), cache, batch, n_heads=8, out=out)
        got = out.double().cpu().numpy().reshape(c.tokens, 8, 128)
        assert np.all(np.abs(got[own] - want[own]) <= bound[own]), (most, ctx)
        assert np.all(got[c.rows:] == 5)


def test_a_graph_of_chunks_replays_with_shorter_ones():
    """One capture for up to 96 rows a sequence, replayed with 96, 5, 1 and no rows."""
    kv, hd, heads, page = 2, 128, 8, 16
    c = po.PagedCase(96, new=[96, 96], ctx=[1500, 400], page=page, kv=kv, hd=hd, store="i8")
    cache, batch = on_gpu(c)
    twin, _ = on_gpu(c)
    batch = lmx.PagedBatch(batch.cu, batch.ctx_lens, batch.page_table, n_tokens=192, max_new=96, max_ctx=1500)
    q, k, v = (gpu(rows(c, 97 + i, h).reshape(192, -1)) for i, h in enumerate((heads, kv, kv)))
    spaces = lmx.Workspace(), lmx.Workspace()

    def path(cache, ws, out):
        y = lmx.paged_prologue(q, k, v, cache, batch, n_heads=heads, q_dtype=torch.float16)
        lmx.paged_attention(y, cache, batch, n_heads=heads, workspace=ws, out=out)
    outs = [torch.zeros(192, heads * hd, device="cuda").half() for _ in range(2)]
    for cc, ws, out in zip((cache, twin), spaces, outs):
        path(cc, ws, out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        path(cache, spaces[0], outs[0])
    for cu, ctx in (([0, 96, 192], [1500, 400]), ([0, 5, 101], [1300, 400]), ([3, 4, 5], [1400, 7]), ([2, 2, 98], [0, 96]),
                    ([0, 0, 0], [5, 5])):
        batch.cu.copy_(torch.tensor(cu, dtype=torch.int32))
        batch.ctx_lens.copy_(torch.tensor(ctx, dtype=torch.int32))
        for out in outs:
            out.fill_(4)
        graph.replay()
        path(twin, spaces[1], outs[1])
        torch.cuda.synchronize()
        assert torch.equal(*outs) and torch.all(outs[0][:cu[0]] == 4) and torch.all(outs[0][cu[2]:] == 4)
        assert torch.all(torch.isfinite(outs[0]))
        assert torch.equal(cache.k, twin.k) and torch.equal(cache.v, twin.v)


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("new,ctx", [([2], [60]), ([2], [2000]), ([150], [150]), ([150], [2000])])
@pytest.mark.parametrize("hd", [64, 512])
def test_rows_of_no_weight_are_zero_whatever_the_values(new, ctx, hd, dt):
    """Every score -infinity, infinities and NaN among V: zeros, in one walk and in splits."""
    say("no weight", new, ctx, hd, dt)
    c = po.PagedCase(98, new=new, ctx=ctx, page=16, kv=1, hd=hd)
    q = rows(c, 99, 2)
    q[..., 7] = np.abs(q[..., 7]) + 0.5
    c.k[:, 0, :, 7] = -np.inf
    for p, x in ((1, np.inf), (40, -np.inf), (ctx[0] - 1, np.nan)):
        pg, s = c.place(0, p)
        c.v[pg, 0, 5 * p % hd, s] = x
    assert np.all(attend(c, q, dt, 2) == 0)
