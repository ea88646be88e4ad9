"""Timed cases of the paged KV cache: its write, its read-back, the norm / rotate
/ store prologue in front of attention, and the attention over it.

A pool holds pages of ``page`` positions per kv head: K as ``[pages, kv_heads,
page, head_dim]``, V as ``[pages, kv_heads, head_dim, page]``, in f16 or in int8
with one f32 scale per row and head (``scale[pages, kv_heads, page]``; value =
int * scale, scale = amax / 127).  A batch is ragged: sequence b brings rows
``cu[b]:cu[b+1]``, its last ``new`` positions of ``ctx_lens[b]``, and
``page_table[b]`` names its pages.

Kinds:

* ``append``    rows of a fused [q | k | v] projection into the pages
* ``round``     the same into int8 pages, and the rows read back as f32
* ``read``      rows of the pages, as contiguous K and V
* ``prologue``  per-head RMS norm with gain and NeoX rotation of q and k, q out,
                K and V into the pages (int8 pages: read back as f16)
* ``attend``    attention of the batch's rows over the pages

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


def _case(kind, shape, *, seqs, new, ctx, page, store, io, lens=0, window=0, **kw):
    """``new`` and ``ctx`` are (least, most) over the sequences; ``lens`` seeds
    the lengths between.  ctx counts the new rows."""
    return dict(kw, kind=kind, **shape, seqs=seqs, new_lo=new[0], new_hi=new[1], ctx_lo=ctx[0],
                ctx_hi=ctx[1], page=page, store=store, io=io, lens=lens, window=window)


def listed():
    return [
        # one decode step of 32 conversations: a row each, at odd lengths
        _case("append", QWEN8B, seqs=32, new=(1, 1), ctx=(1, 4096), page=16, store="f16", io="f32",
              lens=1, name="append_step_f16"),
        # prompts of a batch written to an 8-bit cache, and checked by reading them back
        _case("round", QWEN8B, seqs=8, new=(37, 2048), ctx=(37, 4096), page=32, store="i8", io="f32",
              lens=2, name="round_prompts_i8"),
        # a long conversation leaves the 8-bit pool (hand-over to a contiguous f16 cache)
        _case("read", QWEN8B, seqs=1, new=(32768, 32768), ctx=(32768, 32768), page=64, store="i8",
              io="f16", lens=3, name="read_long_i8"),
        # the prologue of one decode step
        _case("prologue", QWEN8B, seqs=16, new=(1, 1), ctx=(100, 8192), page=16, store="f16", io="f32",
              lens=4, name="prologue_step_f16"),
        # the prologue of prompt chunks on an 8-bit cache, head_dim 256, q in f16
        _case("prologue", GEMMA, seqs=6, new=(129, 1024), ctx=(1000, 4096), page=64, store="i8",
              io="f16", lens=5, name="prologue_chunks_i8"),
        # one token early in a conversation: latency
        _case("attend", SMALL, seqs=1, new=(1, 1), ctx=(512, 512), page=16, store="f16", io="f32",
              lens=6, name="attend_one_short"),
        # one token of a long conversation
        _case("attend", QWEN8B, seqs=1, new=(1, 1), ctx=(32768, 32768), page=64, store="f16", io="f32",
              lens=7, name="attend_one_long"),
        # a decode step of a full server on 8-bit pages, ragged
        _case("attend", QWEN8B, seqs=32, new=(1, 1), ctx=(1, 16384), page=32, store="i8", io="f16",
              lens=8, name="attend_step_i8"),
        # a prompt chunk behind a cached prefix
        _case("attend", QWEN8B, seqs=1, new=(512, 512), ctx=(4608, 4608), page=64, store="f16", io="f16",
              lens=9, name="attend_chunk"),
        # a whole long prompt
        _case("attend", QWEN8B, seqs=1, new=(8192, 8192), ctx=(8192, 8192), page=64, store="f16",
              io="f16", lens=10, name="attend_prompt"),
        # chunks and single tokens in one batch, 8-bit pages, fp32 queries
        _case("attend", QWEN8B, seqs=9, new=(1, 700), ctx=(64, 5000), page=16, store="i8", io="f32",
              lens=11, name="attend_mixed_i8"),
        # sliding-window layer, head_dim 256
        _case("attend", GEMMA, seqs=2, new=(900, 2048), ctx=(900, 4096), page=128, store="f16", io="f16",
              lens=12, window=1024, name="attend_window"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


#: What a drawn attention case may cost: rows x heads x longest context.
MOST_SCORES = 8192 * 8192 * 32


def draw(rng):
    kind = rng.choice(["append", "round", "read", "prologue", "attend", "attend", "attend", "attend"])
    kv = rng.choice([1, 2, 4, 8])
    shape = _shape(kv * rng.choice([1, 2, 3, 4, 5, 8]), kv, rng.choice([64, 128, 128, 256]))
    page = rng.choice([16, 32, 64, 128, 256])
    store = rng.choice(["f16", "i8"])
    io = rng.choice(["f32", "f16"])
    seqs = _log(rng, 1, 48)
    ctx_hi = _log(rng, 16, 16384)
    ctx_lo = rng.randint(1, ctx_hi)
    window = 0
    if kind == "attend":
        form = rng.choice(["step", "chunk", "mixed"])
        window = rng.choice([0, 0, 0, rng.randint(1, 2048)])
        if form == "step":
            new = (1, 1)
        else:
            seqs = _log(rng, 1, 6 if form == "chunk" else 12)
            most = max(1, min(4096, MOST_SCORES // (seqs * shape["heads"] * ctx_hi)))
            new_hi = min(ctx_hi, rng.randint(1, most))
            new = (1 if form == "mixed" else max(1, new_hi // 2), new_hi)
    elif kind == "round" or kind == "read" or rng.random() < 0.5:
        seqs = _log(rng, 1, 8)
        new_hi = min(ctx_hi, _log(rng, 2, 4096))
        new = (1, new_hi)
    else:
        new = (1, 1)
    if kind == "round":
        store, io = "i8", "f32"
    return _case(kind, shape, seqs=seqs, new=new, ctx=(ctx_lo, ctx_hi), page=page, store=store, io=io,
                 lens=rng.randrange(1 << 20), window=window)


# ------------------------------------------------------------------ lengths --
def _lens(case):
    """(new rows, context length) of each sequence."""
    r = random.Random(case["lens"])
    new, ctx = [], []
    for b in range(case["seqs"]):
        # the longest is the first; a batch that mixes both starts with a chunk
        n = case["new_hi"] if b == 0 else r.randint(case["new_lo"], case["new_hi"])
        if case["new_lo"] == 1 < case["new_hi"] and b % 2:
            n = 1
        c = case["ctx_hi"] if b == 0 else r.randint(case["ctx_lo"], case["ctx_hi"])
        new.append(n)
        ctx.append(max(c, n))
    return new, ctx


def _dtype(name):
    return {"f16": torch.float16, "f32": torch.float32, "i8": torch.int8}[name]


# ------------------------------------------------------------------- inputs --
def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    H, kv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    new, ctx = _lens(case)
    tokens = sum(new)
    per = [-(-c // page) for c in ctx]
    pages, stride = sum(per), max(per)
    order = torch.randperm(pages, generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    table = torch.full((len(ctx), stride), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s = dict(case=case, tokens=tokens, max_new=max(new), max_ctx=max(ctx), table=table,
             cu=torch.tensor(cu, dtype=torch.int32, device=DEV),
             ctx=torch.tensor(ctx, dtype=torch.int32, device=DEV))

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    def pool(*shape):
        if case["store"] == "f16":
            return normal(*shape).to(torch.float16)
        return (normal(*shape) * 35).round().clamp(-127, 127).to(torch.int8)

    s["k"], s["v"] = pool(pages, kv, page, hd), pool(pages, kv, hd, page)
    s["k_scale"] = s["v_scale"] = None
    if case["store"] == "i8":
        # amax / 127 of rows whose amax is around 3.5, some rows louder
        s["k_scale"] = 0.0275 * torch.exp(0.3 * normal(pages, kv, page))
        s["v_scale"] = 0.0275 * torch.exp(0.3 * normal(pages, kv, page))
    if case["kind"] == "attend":
        s["q"] = (1.5 * normal(tokens, H * hd)).to(_dtype(case["io"]))
    elif case["kind"] != "read":
        # the fused projection's rows: [q heads | k heads | v heads]
        src = torch.float32 if case["kind"] == "prologue" else _dtype(case["io"])
        s["qkv"] = (2 * normal(tokens, (H + 2 * kv) * hd)).to(src)
        s["q_gain"], s["k_gain"] = 1 + 0.1 * normal(hd), 1 + 0.1 * normal(hd)
    if own:
        import llmoxide_amd as lmx
        s["cache"] = lmx.PagedCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        s["batch"] = lmx.PagedBatch(s["cu"], s["ctx"], s["table"], n_tokens=tokens,
                                    max_new=s["max_new"], max_ctx=s["max_ctx"])
        s["ws"] = lmx.Workspace()
    return s


def _parts(s):
    """The q, k and v columns of the fused rows, as views."""
    c = s["case"]
    nq, nk = c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
    x = s["qkv"]
    return x[:, :nq], x[:, nq:nq + nk], x[:, nq + nk:]


# --------------------------------------------------------------- plain form --
def _rows(s):
    """Sequence, position, page and slot of each of the batch's rows."""
    new = s["cu"][1:] - s["cu"][:-1]
    row = torch.arange(s["tokens"], device=DEV)
    seq = torch.searchsorted(s["cu"][1:].long(), row, right=True)
    pos = (s["ctx"] - new)[seq] + row - s["cu"][seq]
    page = s["table"][seq, pos // s["case"]["page"]].long()
    return seq, pos, page, pos % s["case"]["page"]


def _quantised(x):
    """(ints, scale) of heads [..., head_dim]: the stored scale is f32, the ints
    are rounded in 64 bits, since some values lie next to a border."""
    scale = (x.double().abs().amax(-1) / 127).float()
    ints = torch.round(x.double() / scale.double().clamp_min(1e-300)[..., None])
    return ints.to(torch.int8), scale


def _store(s, k, v):
    """Rows [tokens, kv_heads, head_dim] into the pool."""
    _, _, page, slot = _rows(s)
    if s["case"]["store"] == "i8":
        k, s["k_scale"][page, :, slot] = _quantised(k)
        v, s["v_scale"][page, :, slot] = _quantised(v)
    else:
        k, v = k.to(torch.float16), v.to(torch.float16)
    s["k"][page, :, slot] = k
    s["v"][page, :, :, slot] = v


def _load(s, dtype):
    """The batch's rows back as contiguous [tokens, kv_heads * head_dim]."""
    _, _, page, slot = _rows(s)
    k, v = s["k"][page, :, slot].float(), s["v"][page, :, :, slot].float()
    if s["case"]["store"] == "i8":
        k, v = k * s["k_scale"][page, :, slot][..., None], v * s["v_scale"][page, :, slot][..., None]
    return k.to(dtype).flatten(1), v.to(dtype).flatten(1)


def _normed_rotated(x, gain, pos):
    """x [tokens, heads, head_dim]: RMS norm with gain, then NeoX rotation."""
    hd = x.shape[-1]
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + RMS_EPS) * gain
    j = torch.arange(hd // 2, device=DEV, dtype=torch.float64)
    angle = pos.double()[:, None] * torch.exp(-2 * j / hd * math.log(ROPE_BASE))  # far positions: 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _attend_plain(s):
    c = s["case"]
    H, kv, hd, page, n_seq = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["seqs"]
    group, most = H // kv, s["max_new"]
    table = s["table"].long().clamp_min(0)
    S = table.shape[1] * page

    def whole(pool, scale, slots_last):
        x = pool[table].float()  # [seqs, pages, kv, ...]
        x = x.transpose(-1, -2) if slots_last else x
        if scale is not None:
            x = x * scale[table][..., None]
        return x.transpose(1, 2).reshape(n_seq, kv, S, hd).contiguous()

    K, V = whole(s["k"], s["k_scale"], False), whole(s["v"], s["v_scale"], True)
    seq, pos, _, _ = _rows(s)
    j = torch.arange(s["tokens"], device=DEV) - s["cu"][seq]
    q = torch.zeros(n_seq, most, kv, group, hd, device=DEV)
    q[seq, j] = s["q"].float().view(-1, kv, group, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(n_seq, kv, group * most, hd).contiguous()
    scores = torch.matmul(q, K.transpose(-1, -2).contiguous()) * (1 / math.sqrt(hd))
    at = (s["ctx"] - (s["cu"][1:] - s["cu"][:-1]))[:, None] + torch.arange(most, device=DEV)
    key = torch.arange(S, device=DEV)
    seen = (key <= at[..., None]) & (key < s["ctx"][:, None, None])
    if c["window"]:
        seen &= key > at[..., None] - c["window"]
    scores = scores.view(n_seq, kv, group, most, S).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(scores.sub_(top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n_seq, kv, group * most, S), V).view(n_seq, kv, group, most, hd) / total
    return o.permute(0, 3, 1, 2, 4)[seq, j].reshape(s["tokens"], H * hd).to(s["q"].dtype)


def _pool_out(s):
    """A pool as an answer: f16 pages as they are, 8-bit rows as their values."""
    if s["case"]["store"] == "f16":
        return s["k"], s["v"]
    return _load(s, torch.float16)


# ---------------------------------------------------------------- both forms --
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "attend":
        return _attend_plain(s)
    if c["kind"] == "read":
        return _load(s, _dtype(c["io"]))
    heads = [x.float().unflatten(1, (-1, c["head_dim"])) for x in _parts(s)]
    if c["kind"] == "prologue":
        _, pos, _, _ = _rows(s)
        q, k = (_normed_rotated(x, gain, pos) for x, gain in zip(heads, (s["q_gain"], s["k_gain"])))
        _store(s, k, heads[2])
        return (q.to(_dtype(c["io"])).flatten(1), *_pool_out(s))
    _store(s, heads[1], heads[2])
    return _load(s, torch.float32) if c["kind"] == "round" else _pool_out(s)


def _run_own(s):
    import llmoxide_amd as lmx
    c = s["case"]
    cache, batch = s["cache"], s["batch"]
    if c["kind"] == "attend":
        return lmx.paged_attention(s["q"], cache, batch, n_heads=c["heads"], window=c["window"],
                                   workspace=s["ws"])
    if c["kind"] == "read":
        return lmx.paged_read(cache, batch, dtype=_dtype(c["io"]))
    q, k, v = _parts(s)
    if c["kind"] == "prologue":
        q = lmx.paged_prologue(q, k, v, cache, batch, n_heads=c["heads"], q_gain=s["q_gain"],
                               k_gain=s["k_gain"], rms_eps=RMS_EPS, rope_base=ROPE_BASE,
                               q_dtype=_dtype(c["io"]))
        return (q, s["k"], s["v"]) if c["store"] == "f16" else (
            q, *lmx.paged_read(cache, batch, dtype=torch.float16))
    lmx.paged_append(k, v, cache, batch)
    if c["kind"] == "round":
        return lmx.paged_read(cache, batch, dtype=torch.float32)
    return (s["k"], s["v"]) if c["store"] == "f16" else lmx.paged_read(cache, batch, dtype=torch.float16)


# --------------------------------------------------------------- what it costs --
def work(case):
    H, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    new, ctx = _lens(case)
    tokens = sum(new)
    io = 2 if case["io"] == "f16" else 4
    held = 2 * kv * (hd * 2 if case["store"] == "f16" else hd + 4)  # K and V of one position
    rows = 2 * kv * hd
    if case["kind"] == "attend":
        w = case["window"] or max(ctx)
        span = sum(c - max(0, c - n + 1 - w) for n, c in zip(new, ctx))
        pairs = sum(min(c - n + i + 1, w) for n, c in zip(new, ctx) for i in range(n))
        return {"bytes": 2 * tokens * H * hd * io + span * held, "flops": 4 * hd * H * pairs}
    if case["kind"] == "read":
        return {"bytes": tokens * (held + rows * io), "flops": rows * tokens}
    if case["kind"] == "prologue":
        q = tokens * H * hd * (4 + io)
        back = tokens * (held + rows * 2) if case["store"] == "i8" else 0
        return {"bytes": q + tokens * (rows * 4 + held) + back, "flops": 8 * (H + kv) * hd * tokens}
    back = 4 if case["kind"] == "round" else 2 if case["store"] == "i8" else 0
    return {"bytes": tokens * (rows * io + held) + (tokens * (held + rows * back) if back else 0),
            "flops": 4 * rows * tokens}


# ------------------------------------------------------------------ 64 bits --
def exact(case, seed):
    """The definition, sequence by sequence and head by head, in 64 bits."""
    s = prepare(case, seed)
    H, kv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    new, ctx = _lens(case)
    eight = case["store"] == "i8"

    def places(b, lo, hi):
        p = torch.arange(lo, hi, device=DEV)
        return s["table"][b].long()[p // page], p % page

    def held(b, lo, hi):
        """K and V of positions [lo, hi) as [kv, positions, hd]."""
        pg, sl = places(b, lo, hi)
        out = []
        for x, scale in ((s["k"][pg, :, sl], s["k_scale"]), (s["v"][pg, :, :, sl], s["v_scale"])):
            x = x.double()
            out.append((x * scale[pg, :, sl].double()[..., None] if eight else x).transpose(0, 1))
        return out

    if case["kind"] == "attend":
        outs, at = [], 0
        for b, (n, c) in enumerate(zip(new, ctx)):
            lo = max(0, c - n + 1 - case["window"]) if case["window"] else 0
            K, V = held(b, lo, c)
            q = s["q"][at:at + n].double().view(n, H, hd)
            at += n
            pos = torch.arange(c - n, c, device=DEV)[:, None]
            key = torch.arange(lo, c, device=DEV)[None]
            hidden = key > pos
            if case["window"]:
                hidden |= key <= pos - case["window"]
            o = torch.empty(n, H, hd, dtype=torch.float64, device=DEV)
            for h in range(H):
                x = (q[:, h].contiguous() @ K[h // (H // kv)].t().contiguous()) / math.sqrt(hd)
                x = torch.where(hidden, torch.full_like(x, -math.inf), x)
                x = torch.exp(x - x.max(1, keepdim=True).values)
                o[:, h] = (x / x.sum(1, keepdim=True)) @ V[h // (H // kv)].contiguous()
            outs.append(o.reshape(n, H * hd))
        return torch.cat(outs)

    if case["kind"] == "read":
        got = [held(b, c - n, c) for b, (n, c) in enumerate(zip(new, ctx))]
        return tuple(torch.cat([x[i].transpose(0, 1).reshape(-1, kv * hd) for x in got]) for i in (0, 1))

    q, k, v = (x.double().reshape(x.shape[0], -1, hd) for x in _parts(s))
    if case["kind"] == "prologue":
        pos = torch.cat([torch.arange(c - n, c, device=DEV) for n, c in zip(new, ctx)]).double()
        freq = torch.tensor([ROPE_BASE ** (-2.0 * i / hd) for i in range(hd // 2)], device=DEV,
                            dtype=torch.float64)
        turn = torch.polar(torch.ones_like(pos)[:, None] * torch.ones_like(freq), pos[:, None] * freq)

        def turned(x, gain):
            x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + RMS_EPS) * gain.double()
            z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * turn[:, None]
            return torch.cat([z.real, z.imag], -1)

        q, k = turned(q, s["q_gain"]), turned(k, s["k_gain"])

    if not eight:  # the pages' values before their rounding to f16
        pools = [s["k"].double(), s["v"].double()]
        at = 0
        for b, (n, c) in enumerate(zip(new, ctx)):
            pg, sl = places(b, c - n, c)
            pools[0][pg, :, sl] = k[at:at + n]
            pools[1][pg, :, :, sl] = v[at:at + n]
            at += n
        back = pools
    else:
        back = []
        for x in (k, v):
            scale = (x.abs().amax(-1, keepdim=True) / 127).float().double()  # held in 32 bits
            back.append((torch.round(x / scale) * scale).flatten(1))
    return (q.flatten(1), *back) if case["kind"] == "prologue" else tuple(back)
