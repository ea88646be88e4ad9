"""Timed cases of a step with drafted tokens over a paged KV cache: its page tables
and tree, its prologue, its attention, the verification of the drafts, and the
keeping of the accepted rows.

The cache is that of ``perf/operators.py``: pages of ``page`` positions per kv head,
K as ``[pages, kv_heads, page, head_dim]``, V as ``[pages, kv_heads, head_dim,
page]``, f16 or int8 with one f32 scale per row and head.  A request brings ``new``
rows, which take the slots behind its cached positions in row order.  Where they are
a tree of drafted tokens, ``parent[i]`` is the row (within the request's) that row i
continues, row 0 being the last accepted token; row i's position is its depth behind
the cached ones, and it sees the cache, itself and its ancestors (``seen``: 64 rows a
word, lowest bit first).

Kinds:

* ``plan``      requests leave and take pages, row offsets, lengths and slots are
                made, with trees also positions and ``seen``; then the step is
                withdrawn (the second call gives its pages back)
* ``prologue``  per-head RMS norm with gain and rotation of q and k at given
                positions, K and V into the pages
* ``attend``    attention of the trees' rows over the pages
* ``verify``    which drafted rows are accepted, and the next token
* ``keep``      the accepted rows' K and V to consecutive slots, in every layer

With ``own`` false ``run`` is the plain form in torch; with ``own`` true it calls
llmoxide_amd's entry points.
"""
import math
import random

import torch

own = False

DEV = "cuda"
RMS_EPS = 1e-6
ROPE_BASE = 1e6


def _shape(heads, kv_heads, head_dim):
    return dict(heads=heads, kv_heads=kv_heads, head_dim=head_dim)


SMALL = _shape(16, 8, 128)
QWEN8B = _shape(32, 8, 128)
GEMMA = _shape(16, 8, 256)


def _case(kind, *, seqs, new, lens=0, **kw):
    """``new`` is (least, most) rows a request; ``lens`` seeds lengths and trees."""
    return dict(kw, kind=kind, seqs=seqs, new_lo=new[0], new_hi=new[1], lens=lens)


def _paged(kind, shape, *, ctx, page, store="f16", io="f16", window=0, tree="tree", **kw):
    """``ctx`` is (least, most) length of a request, its new rows counted."""
    return _case(kind, **shape, ctx_lo=ctx[0], ctx_hi=ctx[1], page=page, store=store, io=io, window=window,
                 tree=tree, **kw)


def _verify(*, seqs, new, vocab, drafts, tree, io="f32", lens=0, **kw):
    return _case("verify", seqs=seqs, new=new, vocab=vocab, drafts=drafts, tree=tree, io=io, lens=lens, **kw)


def listed():
    return [
        # 16 conversations, each with a tree of 32 drafted tokens: latency
        _case("plan", seqs=16, new=(32, 32), ctx_lo=100, ctx_hi=8192, page=16, tree="tree", lens=1,
              name="plan_trees"),
        # a full server takes in prompts while some requests leave
        _case("plan", seqs=64, new=(1, 4096), ctx_lo=1, ctx_hi=16384, page=32, tree="none", lens=2,
              name="plan_prompts"),
        # the trees' prologue in one layer
        _paged("prologue", QWEN8B, seqs=16, new=(32, 32), ctx=(100, 8192), page=16, rot=128, layout="half",
               far=0, lens=3, name="prologue_trees"),
        # chunks of long documents on an 8-bit cache: interleaved pairs, half of the head,
        # frequencies and turns scaled for positions past those trained on
        _paged("prologue", GEMMA, seqs=6, new=(129, 1024), ctx=(1000, 4096), page=64, store="i8", rot=128,
               layout="pairs", far=100000, tree="chain", lens=4, name="prologue_far_i8"),
        # one conversation, a short chain of drafts: latency
        _paged("attend", SMALL, seqs=1, new=(6, 6), ctx=(518, 518), page=16, io="f32", tree="chain", lens=5,
               name="attend_chain"),
        # trees of 64 nodes on long conversations
        _paged("attend", QWEN8B, seqs=8, new=(64, 64), ctx=(1000, 8192), page=64, lens=6, name="attend_trees"),
        # a full server on 8-bit pages, small ragged trees
        _paged("attend", QWEN8B, seqs=32, new=(1, 16), ctx=(16, 8192), page=32, store="i8", lens=7,
               name="attend_step_i8"),
        # one conversation, a chain sampled from a draft model: latency
        _verify(seqs=1, new=(6, 6), vocab=32000, drafts="sampled", tree="chain", lens=8, name="verify_chain"),
        # 16 conversations, trees of a draft model's best tokens
        _verify(seqs=16, new=(32, 32), vocab=131072, drafts="best", tree="tree", lens=9, name="verify_trees"),
        # trees sampled from a draft model, an odd vocabulary
        _verify(seqs=8, new=(9, 24), vocab=100003, drafts="sampled", tree="tree", lens=10,
                name="verify_sampled_trees"),
        # the accepted rows of a step, all layers at once
        _paged("keep", QWEN8B, seqs=16, new=(32, 32), ctx=(100, 1024), page=16, layers=36, lens=11,
               name="keep_trees"),
        # one conversation's, in a small model
        _paged("keep", SMALL, seqs=1, new=(16, 16), ctx=(512, 512), page=64, layers=8, lens=12, name="keep_one"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "prologue", "attend", "attend", "verify", "verify", "keep"])
    lens = rng.randrange(1 << 20)
    tree = rng.choice(["tree", "tree", "chain"])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "plan":
        seqs = _log(rng, 1, 64)
        tree = rng.choice(["tree", "none"])
        most = _log(rng, 1, 64 if tree == "tree" else 4096)
        return _case("plan", seqs=seqs, new=(1, most), ctx_lo=1, ctx_hi=_log(rng, most + 1, 16384), page=page,
                     tree=tree, lens=lens)
    if kind == "verify":
        drafts = rng.choice(["best", "sampled"])
        most = _log(rng, 1, 32)
        seqs = _log(rng, 1, min(16, 512 // most))
        return _verify(seqs=seqs, new=(rng.randint(1, most), most), vocab=_log(rng, 1000, 131072), drafts=drafts,
                       tree=tree, io=rng.choice(["f32", "f32", "f16"]), lens=lens)
    kv = rng.choice([1, 2, 4, 8])
    hd = rng.choice([64, 128, 128, 256])
    shape = _shape(kv * rng.choice([1, 2, 3, 4, 5]), kv, hd)
    most = _log(rng, 1, 64)
    seqs = _log(rng, 1, max(1, min(32, 512 // most)))
    ctx_hi = _log(rng, most + 1, 8192)
    ctx = (rng.randint(1, ctx_hi), ctx_hi)
    store = rng.choice(["f16", "i8"])
    new = (rng.randint(1, most), most)
    if kind == "keep":
        return _paged("keep", shape, seqs=seqs, new=new, ctx=(min(ctx[0], 1024), min(ctx_hi, 1024)), page=page,
                      store=store, tree=tree, layers=rng.randint(1, 8 if store == "i8" else 36), lens=lens)
    io = rng.choice(["f32", "f16"])
    if kind == "attend":
        return _paged("attend", shape, seqs=seqs, new=new, ctx=ctx, page=page, store=store, io=io, tree=tree,
                      window=rng.choice([0, 0, rng.randint(most, 2048)]), lens=lens)
    return _paged("prologue", shape, seqs=seqs, new=new, ctx=ctx, page=page, store=store, io=io, tree=tree,
                  rot=rng.choice([hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)]),
                  layout=rng.choice(["half", "pairs"]), far=rng.choice([0, rng.randint(1, 1000000)]), lens=lens)


# ------------------------------------------------------------------ lengths --
def _lens(case):
    """(new rows, length with them) of each request."""
    r = random.Random(case["lens"])
    new, ctx = [], []
    for b in range(case["seqs"]):
        n = case["new_hi"] if b == 0 else r.randint(case["new_lo"], case["new_hi"])
        if case["kind"] == "plan" and case["tree"] == "none" and b % 3:
            n = 1  # beside the prompts, requests that decode
        new.append(n)
        if "ctx_hi" in case:
            ctx.append(max(n, case["ctx_hi"] if b == 0 else r.randint(case["ctx_lo"], case["ctx_hi"])))
    return new, ctx


def _parents(case):
    """The tree of each request, as lists: parents lie before their children."""
    r = random.Random(case["lens"] + 1)
    if case["tree"] == "chain":
        return [list(range(-1, n - 1)) for n in _lens(case)[0]]
    return [[-1] + [r.randrange(i) for i in range(1, n)] for n in _lens(case)[0]]


def _dtype(name):
    return {"f16": torch.float16, "f32": torch.float32, "i8": torch.int8}[name]


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def _offsets(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return cu


def _trees(case):
    """Parents of all rows, their depths and who sees whom, as a program has them
    on the host: words of 64 rows, lowest bit first, in two's complement."""
    parent, depth, seen, words = [], [], [], -(-case["new_hi"] // 64)
    for tree in _parents(case):
        d, s = [], []
        for i, p in enumerate(tree):
            d.append(d[p] + 1 if p >= 0 else 0)
            s.append((s[p] if p >= 0 else 0) | 1 << i)
        parent, depth, seen = parent + tree, depth + d, seen + s

    def word(bits, w):
        x = bits >> (64 * w) & (1 << 64) - 1
        return x - (1 << 64) if x >> 63 else x

    return _ints(parent), _ints(depth), _ints([[word(s, w) for w in range(words)] for s in seen], torch.int64)


# ------------------------------------------------------------------- inputs --
def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    return {"plan": _prepare_plan, "verify": _prepare_verify}.get(case["kind"], _prepare_paged)(case, g)


def _prepare_plan(case, g):
    new, ctx = _lens(case)
    page, n = case["page"], case["seqs"]
    stride = -(-max(ctx) // page)
    before = [c - k for c, k in zip(ctx, new)]
    held = [-(-c // page) for c in before]
    r = random.Random(case["lens"] + 2)
    if case["tree"] == "none":  # some requests leave in this step
        for b in range(1, n):
            if r.random() < 0.15:
                new[b] = 0
    after = [0 if k == 0 else c for k, c in zip(new, before)]
    pages = sum(-(-c // page) for c in ctx) + 8
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((n, stride), -1, dtype=torch.int32, device=DEV)
    at = _offsets(held)
    for b in range(n):
        table[b, :held[b]] = order[at[b]:at[b + 1]]
    free = torch.full((pages,), -1, dtype=torch.int32, device=DEV)
    free[:pages - at[-1]] = order[at[-1]:]
    s = dict(case=case, tokens=sum(new), max_new=max(new), max_ctx=max(ctx), table=table, free=free,
             held=_ints(held), n_free=_ints([pages - at[-1], 0]), lens=_ints(after), new=_ints(new),
             before=_ints(before), none=_ints([0] * n))
    if case["tree"] == "tree":
        s["parent"] = _trees(case)[0]
    if own:
        import llmoxide_amd as lmx
        s["tables"] = lmx.PageTables(table, s["held"], free, s["n_free"], page_size=page)
        s["step"], s["undone"] = (lmx.StepPlan.empty(s["tables"], n_tokens=s["tokens"]) for _ in range(2))
        s["batch"] = lmx.PagedBatch(s["step"].cu, s["step"].ctx_lens, table, n_tokens=s["tokens"],
                                    max_new=s["max_new"], max_ctx=s["max_ctx"])
    return s


def _prepare_paged(case, g):
    H, kv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    new, ctx = _lens(case)
    tokens, layers = sum(new), case.get("layers", 1)
    per = [-(-c // page) for c in ctx]
    pages, at = sum(per), _offsets(per)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(ctx), max(per)), -1, dtype=torch.int32, device=DEV)
    for b, n in enumerate(per):
        table[b, :n] = order[at[b]:at[b + 1]]
    s = dict(case=case, tokens=tokens, max_new=max(new), max_ctx=max(ctx), table=table, cu=_ints(_offsets(new)),
             ctx=_ints(ctx))

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    def pool(*shape):
        if case["store"] == "f16":
            return torch.randn((layers, *shape), generator=g, device=DEV, dtype=torch.float16)
        return (normal(layers, *shape) * 35).round().clamp(-127, 127).to(torch.int8)

    s["k"], s["v"] = pool(pages, kv, page, hd), pool(pages, kv, hd, page)
    s["k_scale"] = s["v_scale"] = None
    if case["store"] == "i8":
        # amax / 127 of rows whose amax is around 3.5, some rows louder
        s["k_scale"] = 0.0275 * torch.exp(0.3 * normal(layers, pages, kv, page))
        s["v_scale"] = 0.0275 * torch.exp(0.3 * normal(layers, pages, kv, page))
    s["parent"], depth, s["seen"] = _trees(case)
    seq = torch.repeat_interleave(torch.arange(len(new), device=DEV), _ints(new, torch.int64))
    s["pos"] = (s["ctx"] - _ints(new))[seq] + depth + case.get("far", 0)
    if case["kind"] == "attend":
        s["q"] = (1.5 * normal(tokens, H * hd)).to(_dtype(case["io"]))
    elif case["kind"] == "prologue":
        # the fused projection's rows: [q heads | k heads | v heads]
        s["qkv"] = 2 * normal(tokens, (H + 2 * kv) * hd)
        s["q_gain"], s["k_gain"] = 1 + 0.1 * normal(hd), 1 + 0.1 * normal(hd)
        s["factors"], s["turn_scale"] = _far_factors(case) if case["far"] else (None, 1.0)
    else:
        # a path from each tree's root: at each row, one of its children while there are any
        r = random.Random(int(torch.randint(1 << 30, (1,), generator=g, device=DEV)))
        paths = []
        for tree in _parents(case):
            path = [0]
            while path[-1] in tree and r.random() < 0.8:
                path.append(r.choice([i for i, p in enumerate(tree) if p == path[-1]]))
            paths.append(path)
        s["path"] = _ints([p + [-1] * (max(new) - len(p)) for p in paths])
        s["accepted"] = _ints([len(p) for p in paths])
    if own:
        import llmoxide_amd as lmx
        s["caches"] = [lmx.PagedCache(*(None if x is None else x[i] for x in (s["k"], s["v"], s["k_scale"], s["v_scale"])))
                       for i in range(layers)]
        s["batch"] = lmx.PagedBatch(s["cu"], s["ctx"], table, n_tokens=tokens, max_new=max(new), max_ctx=max(ctx))
        s["ws"] = lmx.Workspace()
    return s


def _far_factors(case):
    """Divisors of the angles that stretch the slow pairs 8 times and leave the fast
    ones, by how often a pair turns over 32768 positions, and the factor that goes
    with them."""
    half = case["rot"] // 2
    j = torch.arange(half, device=DEV, dtype=torch.float64)
    turns = 32768 / (2 * math.pi) * torch.exp(-j / half * math.log(ROPE_BASE))
    keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
    return (1 / (keep + (1 - keep) / 8)).float(), 0.1 * math.log(8) + 1


def _prepare_verify(case, g):
    new, _ = _lens(case)
    trees, V, tokens = _parents(case), case["vocab"], sum(new)
    cu = _offsets(new)
    dt = _dtype(case["io"])
    logits = 5 * torch.randn((tokens, V), generator=g, device=DEV)
    s = dict(case=case, tokens=tokens, max_new=max(new), cu=_ints(cu), p=torch.softmax(logits, 1).to(dt), q=None)
    up, rank, most = [], [], 0  # each row's parent among all rows, and its place among the parent's children
    for b, tree in enumerate(trees):
        count = [0] * len(tree)
        for p in tree:
            up.append(cu[b] + max(p, 0))
            rank.append(count[p] if p >= 0 else 0)
            if p >= 0:
                count[p] += 1
        most = max(most, *count)
    s["children"] = most
    up, rank = _ints(up, torch.int64), _ints(rank, torch.int64)
    if case["drafts"] == "sampled":
        s["q"] = torch.softmax(logits + torch.randn((tokens, V), generator=g, device=DEV), 1).to(dt)
        picks = torch.multinomial(s["q"].float(), max(most, 1), replacement=True, generator=g)
    else:
        picks = s["p"].float().topk(max(most, 1), 1).indices
    s["tokens_in"] = picks[up, rank].to(torch.int32)
    s["parent"] = None if case["tree"] == "chain" else _ints([p for t in trees for p in t])
    s["u"] = torch.rand(tokens, generator=g, device=DEV)
    s["r"] = torch.rand(len(new), generator=g, device=DEV)
    if own:
        import llmoxide_amd as lmx
        s["ws"] = lmx.Workspace()
    return s


# -------------------------------------------------------------- plain forms --
def _rows(s):
    """Request, row within it and slot position of each of the batch's rows."""
    new = s["cu"][1:] - s["cu"][:-1]
    row = torch.arange(s["tokens"], device=DEV)
    seq = torch.searchsorted(s["cu"][1:].long(), row, right=True)
    j = row - s["cu"][seq]
    return seq, j, (s["ctx"] - new)[seq] + j


def _plan_plain(s, lens, new):
    """Pages given back and taken, in place; offsets, lengths, slots and positions."""
    page, table, free, held, (n, E) = s["case"]["page"], s["table"], s["free"], s["held"], s["table"].shape
    total = lens + new
    need = (total + page - 1) // page
    e = torch.arange(E, device=DEV)
    back = (e >= need[:, None]) & (e < held[:, None]) & (table >= 0)
    # the last request's last entry first; what goes nowhere goes behind the list
    order = back.flatten().flip(0).cumsum(0).flip(0).view(n, E)
    room = torch.cat([free, free[:1]])
    room.scatter_(0, torch.where(back, s["n_free"][0] + order - 1, len(free)).flatten(), table.flatten())
    top = s["n_free"][0] + back.sum()
    had = torch.minimum(held, need)
    want = need - had
    first = want.cumsum(0) - want
    got = torch.minimum((top - first).clamp_min(0), want)
    new_entry = (e >= had[:, None]) & (e < (had + got)[:, None])
    k = (top - 1 - (first - had)[:, None] - e).clamp(0, len(free) - 1)
    table.copy_(torch.where(new_entry, room[k], torch.where(back, -1, table)))
    free.copy_(room[:-1])
    held.copy_(had + got)
    s["n_free"].copy_(torch.stack([top - got.sum(), (want - got).sum()]))
    cu = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0).to(torch.int32)])
    row = torch.arange(s["tokens"], device=DEV)
    seq = torch.searchsorted(cu[1:], row.to(torch.int32), right=True).clamp_max(n - 1)
    pos = lens[seq] + row - cu[seq]
    at = table[seq, (pos // page).clamp_max(E - 1)].long()
    mine = row < cu[-1]
    return (cu, total.to(torch.int32), torch.where(mine & (at >= 0), at * page + pos % page, -1),
            torch.where(mine, pos, -1).to(torch.int32))


def _tree_plain(s, cu, ctx):
    """Positions and ``seen`` of the rows from their parents."""
    n, M = s["case"]["seqs"], s["max_new"]
    seq, j, first = _rows(dict(s, cu=cu, ctx=ctx))
    sees = torch.zeros(n, M, M, device=DEV)
    sees[seq, j, s["parent"].clamp_min(0)] = 1  # a root: itself
    sees[seq, j, j] = 1
    for _ in range(max(1, (M - 1).bit_length())):
        sees = (torch.matmul(sees, sees) > 0).float()
    mine = sees[seq, j]
    words = -(-M // 64)
    bits = torch.nn.functional.pad(mine, (0, 64 * words - M)).long().view(-1, words, 64)
    return ((first - j + mine.sum(1) - 1).to(torch.int32),
            (bits << torch.arange(64, device=DEV)).sum(2))


def _quantised(x):
    """(ints, scale) of heads [..., head_dim]: the stored scale is f32, the ints
    are rounded in 64 bits, since some values lie next to a border."""
    scale = (x.double().abs().amax(-1) / 127).float()
    ints = torch.round(x.double() / scale.double().clamp_min(1e-300)[..., None])
    return ints.to(torch.int8), scale


def _normed_turned(x, gain, s):
    """x [tokens, heads, head_dim]: RMS norm with gain, then the rotation of its
    first ``rot`` dims at the rows' positions."""
    c = s["case"]
    half = c["rot"] // 2
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + RMS_EPS) * gain
    j = torch.arange(half, device=DEV, dtype=torch.float64)
    angle = s["pos"].double()[:, None] * torch.exp(-j / half * math.log(ROPE_BASE))  # far positions: 64 bits
    if s["factors"] is not None:
        angle = angle / s["factors"].double()
    cos, sin = ((f(angle) * s["turn_scale"]).float()[:, None] for f in (torch.cos, torch.sin))
    y, tail = x[..., :2 * half], x[..., 2 * half:]
    if c["layout"] == "pairs":
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, tail], -1)


def _prologue_plain(s):
    c = s["case"]
    q, k, v = (x.unflatten(1, (-1, c["head_dim"])) for x in _parts(s))
    q, k = _normed_turned(q, s["q_gain"], s), _normed_turned(k, s["k_gain"], s)
    seq, _, at = _rows(s)
    page, slot = s["table"][seq, at // c["page"]].long(), at % c["page"]
    if c["store"] == "i8":
        k, s["k_scale"][0, page, :, slot] = _quantised(k)
        v, s["v_scale"][0, page, :, slot] = _quantised(v)
    s["k"][0, page, :, slot] = k.to(s["k"].dtype)
    s["v"][0, page, :, :, slot] = v.to(s["v"].dtype)
    q = q.to(_dtype(c["io"])).flatten(1)
    if c["store"] == "f16":
        return q, s["k"], s["v"]
    k, v = s["k"][0, page, :, slot].float(), s["v"][0, page, :, :, slot].float()
    k, v = k * s["k_scale"][0, page, :, slot][..., None], v * s["v_scale"][0, page, :, slot][..., None]
    return q, k.to(torch.float16).flatten(1), v.to(torch.float16).flatten(1)


def _attend_plain(s):
    c = s["case"]
    H, kv, hd, page, n_seq = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["seqs"]
    group, most = H // kv, s["max_new"]
    table = s["table"].long().clamp_min(0)
    S = table.shape[1] * page

    def whole(pool, scale, slots_last):
        x = pool[0][table].float()  # [seqs, pages, kv, ...]
        x = x.transpose(-1, -2) if slots_last else x
        if scale is not None:
            x = x * scale[0][table][..., None]
        return x.transpose(1, 2).reshape(n_seq, kv, S, hd).contiguous()

    K, V = whole(s["k"], s["k_scale"], False), whole(s["v"], s["v_scale"], True)
    seq, j, _ = _rows(s)
    q = torch.zeros(n_seq, most, kv, group, hd, device=DEV)
    q[seq, j] = s["q"].float().view(-1, kv, group, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(n_seq, kv, group * most, hd).contiguous()
    scores = torch.matmul(q, K.transpose(-1, -2).contiguous()) * (1 / math.sqrt(hd))
    # the cache before the batch's rows, in a window by position; of the rows those whose bits are set
    key = torch.arange(S, device=DEV)
    first = (s["ctx"] - (s["cu"][1:] - s["cu"][:-1]))[seq][:, None]
    sees = key < first
    if c["window"]:
        sees = sees & (key > s["pos"][:, None] - c["window"])
    bits = (s["seen"][:, :, None] >> torch.arange(64, device=DEV) & 1).bool().flatten(1)
    place = key - first
    sees = sees | (place >= 0) & (place < most) & bits.gather(1, place.clamp(0, bits.shape[1] - 1))
    seen = torch.zeros(n_seq, most, S, dtype=torch.bool, device=DEV)
    seen[seq, j] = sees & (key < s["ctx"][seq][:, None])
    scores = scores.view(n_seq, kv, group, most, S).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(scores.sub_(top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n_seq, kv, group * most, S), V).view(n_seq, kv, group, most, hd) / total
    return o.permute(0, 3, 1, 2, 4)[seq, j].reshape(s["tokens"], H * hd).to(s["q"].dtype)


def _verify_plain(s):
    """A row's test depends on its parent's row and its earlier siblings alone (they
    were all refused where it is tested), so all rows are tested at once; those
    whose ancestors all passed, each the first among its siblings, are the path.
    Sums over the vocabulary, and what is held against a border, are in 64 bits."""
    V, n, M = s["case"]["vocab"], s["case"]["seqs"], s["max_new"]
    row = torch.arange(s["tokens"], device=DEV)
    seq = torch.searchsorted(s["cu"][1:].long(), row, right=True)
    j = row - s["cu"][seq]
    up = j - 1 if s["parent"] is None else s["parent"].long()
    here = torch.zeros(n, M, dtype=torch.bool, device=DEV)
    here[seq, j] = True

    def pad(x, fill):
        y = torch.full((n, M), fill, dtype=x.dtype, device=DEV)
        y[seq, j] = x
        return y

    parent, token = pad(up, -1), pad(s["tokens_in"].long(), -1)
    i = torch.arange(M, device=DEV)
    drafted = here & (parent >= 0)
    above = (s["cu"][:-1, None] + parent.clamp_min(0)).long()  # the parent's row in the batch
    older = drafted[:, :, None] & drafted[:, None, :] & (parent[:, :, None] == parent[:, None, :]) & (i[:, None] > i)
    rank = older.sum(2)
    p = s["p"][above, token.clamp_min(0)].double()
    u = pad(s["u"], 1.0).double()
    if s["q"] is None:
        twice = (older & (token[:, :, None] == token[:, None, :])).any(2)
        gone = torch.where(twice, 0.0, p)
        passed = drafted & ~twice & (u * (1 - torch.matmul(older.double(), gone[:, :, None])[..., 0]) < p)
    else:
        a, W = torch.zeros(s["tokens"], 1, device=DEV).double(), torch.ones(s["tokens"], 1, device=DEV).double()
        a_s, W_s = [a], [W]
        for _ in range(s["children"]):
            a = a + W
            W = (s["p"].double() - a * s["q"].double()).clamp_min_(0).sum(1, keepdim=True)
            a_s.append(a)
            W_s.append(W)
        a_s, W_s = torch.cat(a_s, 1), torch.cat(W_s, 1)
        q = s["q"][above, token.clamp_min(0)].double()
        w = (p - a_s[above, rank] * q).clamp_min(0)
        passed = drafted & (u * W_s[above, rank] * q < w)
    best = passed & ~(older & passed[:, None, :]).any(2)
    # the root, and the rows all of whose ancestors are such
    link = torch.zeros(n, M, M, device=DEV).double()
    link.scatter_(2, parent.clamp_min(0)[..., None], best[..., None].double())
    link[:, 0] = 0
    link[:, 0, 0] = 1
    for _ in range(max(1, (M - 1).bit_length())):
        link = torch.matmul(link, link)
    on = (link[:, :, 0] > 0) & here
    accepted = on.sum(1)
    path = torch.where(on, i, M).sort(1).values
    path = torch.where(path < M, path, -1)
    last = path.gather(1, (accepted - 1).clamp_min(0)[:, None])[:, 0]
    final = s["cu"][:-1] + last
    w = s["p"][final].double()
    mine = drafted & (parent == last[:, None])
    if s["q"] is None:
        w = torch.nn.functional.pad(w, (0, 1))
        w.scatter_(1, torch.where(mine, token, V), 0.0)
        w = w[:, :V]
    else:
        w = (w - a_s[final, mine.sum(1)][:, None] * s["q"][final].double()).clamp_min_(0)
    sums = w.cumsum(1)
    token = (sums <= s["r"].double()[:, None] * sums[:, -1:]).sum(1).clamp_max(V - 1)
    return path.to(torch.int32), accepted.to(torch.int32), token.to(torch.int32)


def _keep_plain(s):
    page = s["case"]["page"]
    n, M = s["path"].shape
    i = torch.arange(M, device=DEV)
    first = (s["ctx"] - (s["cu"][1:] - s["cu"][:-1]))[:, None]
    move = i < s["accepted"][:, None]
    # a row that does not move is its own source
    src, dst = first + torch.where(move, s["path"], 0), first + torch.where(move, i, 0)
    b = torch.arange(n, device=DEV)[:, None].expand(n, M)

    def place(pos):
        return s["table"][b, pos // page].long().flatten(), (pos % page).flatten()

    (ps, ss), (pd, sd) = place(src), place(dst)
    s["k"][:, pd, :, sd] = s["k"][:, ps, :, ss]
    s["v"][:, pd, :, :, sd] = s["v"][:, ps, :, :, ss]
    if s["k_scale"] is not None:
        s["k_scale"][:, pd, :, sd] = s["k_scale"][:, ps, :, ss]
        s["v_scale"][:, pd, :, sd] = s["v_scale"][:, ps, :, ss]
    return _pools(s)


def _pools(s):
    """The pools as answers: f16 pages as they are, 8-bit ones as their values."""
    if s["k_scale"] is None:
        return s["k"], s["v"]
    return s["k"] * s["k_scale"][..., None], s["v"] * s["v_scale"][..., None, :]


def _parts(s):
    """The q, k and v columns of the fused rows, as views."""
    c = s["case"]
    nq, nk = c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
    x = s["qkv"]
    return x[:, :nq], x[:, nq:nq + nk], x[:, nq + nk:]


# ---------------------------------------------------------------- both forms --
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "plan":
        step = _plan_plain(s, s["lens"], s["new"])
        if "parent" in s:
            step += _tree_plain(s, step[0], step[1])
        _plan_plain(s, s["before"], s["none"])
        return (*step, s["table"], s["held"], s["n_free"])
    return {"prologue": _prologue_plain, "attend": _attend_plain, "verify": _verify_plain, "keep": _keep_plain}[kind](s)


def _run_own(s):
    import llmoxide_amd as lmx
    c = s["case"]
    kind = c["kind"]
    if kind == "plan":
        step = lmx.spec_plan(s["tables"], s["lens"], s["new"], out=s["step"], trim=True)
        out = (step.cu, step.ctx_lens, step.slots, step.pos)
        if "parent" in s:
            tree = lmx.spec_tree(s["parent"], s["batch"])
            out += (tree.pos, tree.seen)
        lmx.spec_plan(s["tables"], s["before"], s["none"], out=s["undone"], trim=True)
        return (*out, s["table"], s["held"], s["n_free"])
    if kind == "verify":
        got = lmx.spec_verify(s["p"], s["tokens_in"], s["u"], s["r"], s["cu"], max_new=s["max_new"],
                              parent=s["parent"], q=s["q"], workspace=s["ws"])
        return got.path, got.accepted, got.token
    if kind == "keep":
        lmx.spec_keep(s["caches"], s["batch"], s["path"], s["accepted"])
        return _pools(s)
    cache, batch = s["caches"][0], s["batch"]
    if kind == "attend":
        return lmx.spec_attention(s["q"], cache, batch, s["seen"], n_heads=c["heads"], pos=s["pos"],
                                  window=c["window"], workspace=s["ws"])
    q, k, v = _parts(s)
    q = lmx.spec_prologue(q, k, v, cache, batch, pos=s["pos"], n_heads=c["heads"], n_rot=c["rot"],
                          interleaved=c["layout"] == "pairs", turn_scale=s["turn_scale"],
                          rope_factors=s["factors"], q_gain=s["q_gain"], k_gain=s["k_gain"], rms_eps=RMS_EPS,
                          rope_base=ROPE_BASE, q_dtype=_dtype(c["io"]))
    if c["store"] == "f16":
        return q, s["k"], s["v"]
    return (q, *lmx.paged_read(cache, batch, dtype=torch.float16))


# --------------------------------------------------------------- what it costs --
def work(case):
    new, ctx = _lens(case)
    tokens, n = sum(new), case["seqs"]
    if case["kind"] == "plan":
        pages = sum(-(-c // case["page"]) - -(-(c - k) // case["page"]) for k, c in zip(new, ctx))
        tree = tokens * (8 + 8 * -(-max(new) // 64)) if case["tree"] == "tree" else 0
        # lengths, offsets and counts of both calls; pages into the table and back; slots and positions
        return {"bytes": 2 * 28 * n + 24 * pages + 12 * tokens + tree, "flops": 10 * tokens}
    if case["kind"] == "verify":
        each = (2 if case["io"] == "f16" else 4) * (2 if case["drafts"] == "sampled" else 1)
        return {"bytes": n * case["vocab"] * each + tokens * (12 + each) + 4 * n * max(new), "flops": 4 * n * case["vocab"]}
    H, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    io = 2 if case["io"] == "f16" else 4
    held = 2 * kv * (hd * 2 if case["store"] == "f16" else hd + 4)  # K and V of one position
    if case["kind"] == "attend":
        w = case["window"] or max(ctx)
        keys = [min(c - k, w) for k, c in zip(new, ctx)]
        # of the rows themselves a row sees a few: its ancestors
        return {"bytes": 2 * tokens * H * hd * io + sum(m + k for m, k in zip(keys, new)) * held + 12 * tokens,
                "flops": 4 * hd * H * sum(k * (m + 4) for m, k in zip(keys, new))}
    if case["kind"] == "keep":
        moved = sum(max(1, int(math.log2(k + 1))) for k in new) * case["layers"]  # about a path's rows
        return {"bytes": 2 * moved * held + 8 * tokens, "flops": moved}
    back = tokens * (held + 2 * kv * hd * 2) if case["store"] == "i8" else 0
    return {"bytes": tokens * (H * hd * (4 + io) + 2 * kv * hd * 4 + held + 4) + back,
            "flops": 8 * (H + kv) * hd * tokens}


# ------------------------------------------------------------------ 64 bits --
def exact(case, seed):
    """The definitions, request by request, in 64 bits."""
    s = prepare(case, seed)
    return {"plan": _exact_plan, "verify": _exact_verify, "keep": _exact_keep, "attend": _exact_attend,
            "prologue": _exact_prologue}[case["kind"]](case, s)


def _exact_plan(case, s):
    page = case["page"]
    table, held = s["table"].tolist(), s["held"].tolist()
    free = s["free"].tolist()[:s["n_free"].tolist()[0]]

    def step(lens, new):
        need = [-(-(a + b) // page) for a, b in zip(lens, new)]
        for b in reversed(range(len(need))):
            while held[b] > need[b]:
                held[b] -= 1
                free.append(table[b][held[b]])
                table[b][held[b]] = -1
        for b in range(len(need)):
            while held[b] < need[b] and free:
                table[b][held[b]] = free.pop()
                held[b] += 1

    lens, new = s["lens"].tolist(), s["new"].tolist()
    step(lens, new)
    pos = [a + i for a, k in zip(lens, new) for i in range(k)]
    slots = [table[b][(a + i) // page] * page + (a + i) % page for b, (a, k) in enumerate(zip(lens, new)) for i in range(k)]
    out = [_ints(_offsets(new)), _ints([a + b for a, b in zip(lens, new)]), _ints(slots, torch.int64), _ints(pos)]
    if "parent" in s:
        _, depth, seen = _trees(case)
        out += [_ints([a for a, k in zip(lens, new) for _ in range(k)]) + depth, seen]
    step(s["before"].tolist(), s["none"].tolist())
    return (*out, _ints(table), _ints(held), _ints([len(free), 0]))  # no page is lacking


def _exact_verify(case, s):
    new, _ = _lens(case)
    cu, parents = _offsets(new), _parents(case)
    tok, u, r = s["tokens_in"].tolist(), s["u"].tolist(), s["r"].tolist()
    paths, counts, tokens = [], [], []
    for b, n in enumerate(new):
        at, path = 0, [0]
        p = s["p"][cu[b]].double()
        q = None if s["q"] is None else s["q"][cu[b]].double()
        w, W = p, 1.0  # what is left of the target's distribution, and its mass
        a = 0.0
        for i in range(1, n):
            if parents[b][i] != at:
                continue
            t, x = tok[cu[b] + i], u[cu[b] + i]
            if (x * W * float(q[t]) if q is not None else x * W) < float(w[t]):
                at = i
                path.append(i)
                p = w = s["p"][cu[b] + i].double()
                q = None if s["q"] is None else s["q"][cu[b] + i].double()
                W, a = 1.0, 0.0
            elif q is None:
                W -= float(w[t])
                w = w.clone()
                w[t] = 0
            else:
                a += W
                w = (p - a * q).clamp_min(0)
                W = float(w.sum())
        sums = w.cumsum(0)
        tokens.append(int((sums > r[b] * sums[-1]).nonzero()[0]))
        counts.append(len(path))
        paths.append(path + [-1] * (max(new) - len(path)))
    return _ints(paths), _ints(counts), _ints(tokens)


def _exact_keep(case, s):
    page, (new, ctx) = case["page"], _lens(case)
    table, paths, counts = s["table"].tolist(), s["path"].tolist(), s["accepted"].tolist()
    k, v = (x.double() for x in _pools(s)) if s["k_scale"] is not None else (s["k"].clone(), s["v"].clone())
    for b, (n, c) in enumerate(zip(new, ctx)):
        for j in range(counts[b]):  # a row's source never lies before it
            (p0, s0), (p1, s1) = ((table[b][x // page], x % page) for x in (c - n + paths[b][j], c - n + j))
            k[:, p1, :, s1] = k[:, p0, :, s0].clone()
            v[:, p1, :, :, s1] = v[:, p0, :, :, s0].clone()
    return k.double(), v.double()


def _held(case, s, b, lo, hi):
    """K and V of positions [lo, hi) as [kv, positions, hd]."""
    p = torch.arange(lo, hi, device=DEV)
    pg, sl = s["table"][b].long()[p // case["page"]], p % case["page"]
    out = []
    for x, scale in ((s["k"][0, pg, :, sl], s["k_scale"]), (s["v"][0, pg, :, :, sl], s["v_scale"])):
        x = x.double()
        out.append((x * scale[0, pg, :, sl].double()[..., None] if scale is not None else x).transpose(0, 1))
    return out


def _exact_attend(case, s):
    H, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    outs, at = [], 0
    for b, (n, c, tree) in enumerate(zip(*_lens(case), _parents(case))):
        first = c - n
        lo = max(0, first + 1 - case["window"]) if case["window"] else 0
        K, V = _held(case, s, b, lo, c)
        hidden = torch.ones(n, c - lo, dtype=torch.bool)
        depth = []
        for i, p in enumerate(tree):
            depth.append(depth[p] + 1 if p >= 0 else 0)
            hidden[i, :first - lo] = False
            if case["window"]:
                hidden[i, :max(0, first + depth[i] + 1 - case["window"] - lo)] = True
            while i >= 0:
                hidden[len(depth) - 1, first - lo + i] = False
                i = tree[i]
        hidden = hidden.to(DEV)
        q = s["q"][at:at + n].double().view(n, H, hd)
        at += n
        o = torch.empty(n, H, hd, dtype=torch.float64, device=DEV)
        for h in range(H):
            x = (q[:, h].contiguous() @ K[h // (H // kv)].t().contiguous()) / math.sqrt(hd)
            x = torch.where(hidden, torch.full_like(x, -math.inf), x)
            x = torch.exp(x - x.max(1, keepdim=True).values)
            o[:, h] = (x / x.sum(1, keepdim=True)) @ V[h // (H // kv)].contiguous()
        outs.append(o.reshape(n, H * hd))
    return torch.cat(outs)


def _exact_prologue(case, s):
    hd, page, half = case["head_dim"], case["page"], case["rot"] // 2
    q, k, v = (x.double().reshape(x.shape[0], -1, hd) for x in _parts(s))
    freq = torch.tensor([ROPE_BASE ** (-2.0 * i / case["rot"]) for i in range(half)], device=DEV, dtype=torch.float64)
    if s["factors"] is not None:
        freq = freq / s["factors"].double()
    pos = s["pos"].double()[:, None]
    turn = torch.polar(torch.full_like(pos, s["turn_scale"]) * torch.ones_like(freq), pos * freq)

    def turned(x, gain):
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + RMS_EPS) * gain.double()
        if case["layout"] == "pairs":
            z = torch.view_as_complex(x[..., :2 * half].unflatten(-1, (half, 2)).contiguous()) * turn[:, None]
            return torch.cat([torch.view_as_real(z).flatten(-2), x[..., 2 * half:]], -1)
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn[:, None]
        return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)

    q, k = turned(q, s["q_gain"]), turned(k, s["k_gain"])
    if case["store"] == "i8":
        back = []
        for x in (k, v):
            scale = (x.abs().amax(-1, keepdim=True) / 127).float().double()  # held in 32 bits
            back.append((torch.round(x / scale) * scale).flatten(1))
        return (q.flatten(1), *back)
    pools, at = [s["k"].double(), s["v"].double()], 0  # the pages' values before their rounding to f16
    for b, (n, c) in enumerate(zip(*_lens(case))):
        p = torch.arange(c - n, c, device=DEV)
        pg, sl = s["table"][b].long()[p // page], p % page
        pools[0][0, pg, :, sl] = k[at:at + n]
        pools[1][0, pg, :, :, sl] = v[at:at + n]
        at += n
    return (q.flatten(1), *pools)
