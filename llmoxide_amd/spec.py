"""Steps with drafted tokens over the paged KV cache (include/lmx/spec.h): pages and
row maps from the requests' lengths, trees, the prologue at their positions,
attention by their masks, verification of the drafts and the keeping of what was
accepted.

=====================  ======================================================
this module            what it does
=====================  ======================================================
``spec_plan``          page table, row offsets, lengths and slots of a step
``spec_tree``          positions of a tree's rows, and who sees whom
``spec_prologue``      ``paged_prologue`` at given positions, either order of
                       pairs, with scaled turns
``spec_attention``     ``paged_attention`` of rows that see each other by a mask
``spec_verify``        which drafts the target accepts, and the next token
``spec_keep``          the accepted rows to consecutive slots, in all layers
=====================  ======================================================

The reference decodes one token at a time (docs/limitations.md:21).  A request's
rows are its last accepted token, whose K and V the cache lacks, and drafted tokens
behind it; ``parent`` names the row that each continues.  One step of a loop::

    step = spec_plan(tables, lens, new_rows, out=step, trim=True)
    tree = spec_tree(parent, batch, out=tree)             # batch of step and tables
    for layer in layers:
        q = spec_prologue(..., layer.cache, batch, pos=tree.pos)
        o = spec_attention(q, layer.cache, batch, tree.seen)
    got = spec_verify(p, tokens, u, r, step.cu, max_new=..., parent=parent, lens=lens)
    spec_keep([layer.cache for layer in layers], batch, got.path, got.accepted)

All of it is read on the device, so the loop can be one captured graph.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Sequence

from . import F32, Workspace, _allocated, _check, _need_cuda, _ptr, _stream, _torch, lib
from . import paged as _paged
from .paged import BatchDesc, PagedAttnDesc, PagedBatch, PagedCache, PagedPrologueDesc, PoolDesc, _new_out, _rows

#: Most rows of a request in a tree, an attention, a verification and a keeping.
MAX_ROWS = 1024

_U32, _VP = ctypes.c_uint32, ctypes.c_void_p


class SpecPlanDesc(ctypes.Structure):
    """lmxs_plan_desc."""
    _fields_ = [("n_seq", _U32), ("n_tokens", _U32), ("page_size", _U32), ("table_stride", _U32), ("n_pages", _U32),
                ("trim", _U32)]


class SpecRope(ctypes.Structure):
    """lmxs_rope."""
    _fields_ = [("interleaved", _U32), ("turn_scale", ctypes.c_float)]


class SpecVerifyDesc(ctypes.Structure):
    """lmxs_verify_desc."""
    _fields_ = [("n_seq", _U32), ("n_tokens", _U32), ("max_new", _U32), ("vocab", _U32), ("p_stride", _U32),
                ("q_stride", _U32), ("greedy", _U32)]


_PP, _PB = ctypes.POINTER(PoolDesc), ctypes.POINTER(BatchDesc)
_PR, _PA = ctypes.POINTER(PagedPrologueDesc), ctypes.POINTER(PagedAttnDesc)
_PS, _PO, _PV = ctypes.POINTER(SpecPlanDesc), ctypes.POINTER(SpecRope), ctypes.POINTER(SpecVerifyDesc)
_I, _SZ = ctypes.c_int, ctypes.c_size_t
# Every symbol include/lmx/spec.h declares.
SIGNATURES = {
    "lmxs_plan": (_I, [_PS] + [_VP] * 11),
    "lmxs_tree": (_I, [_PB, _VP, _U32, _U32, _VP, _VP, _VP]),
    "lmxs_prologue": (_I, [_PP, _PB, _PR, _PO] + [_VP] * 8 + [_I, _VP]),
    "lmxs_attn_workspace_bytes": (_SZ, [_PP, _PB, _PA]),
    "lmxs_attn": (_I, [_PP, _PB, _PA, _VP, _U32, _VP, _VP, _I, _VP, _VP, _SZ, _VP]),
    "lmxs_verify_workspace_bytes": (_SZ, [_PV]),
    "lmxs_verify": (_I, [_PV] + [_VP] * 5 + [_I] + [_VP] * 7 + [_SZ, _VP]),
    "lmxs_keep": (_I, [ctypes.POINTER(_VP), _U32, _PB, _VP, _U32, _VP, _VP]),
}

_lib = None


def spec_lib() -> ctypes.CDLL:
    """The library with lmx/spec.h's signatures set; raises if it is missing."""
    global _lib
    if _lib is None:
        L = lib()
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _lib = L
    return _lib


_i32 = None


def _ints(what: str, t, size, at: int) -> None:
    """``t``: int32, contiguous, on device ``at``, of ``size`` elements (None: any)."""
    global _i32
    if _i32 is None:
        _i32 = _torch().int32
    if t.dtype != _i32:
        raise TypeError(f"{what} is int32")
    if t.get_device() != at or at < 0:
        raise ValueError(f"{what} must be on the GPU, on the device of the call's other tensors")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    if size is not None and t.numel() != size:
        raise ValueError(f"{what} has {size} elements, not {t.numel()}")


def _fresh(like, shape, stream):
    """``_new_out`` of ``like``'s type and device (1.1 us; by torch.empty, which is told
    both, 1.6)."""
    return like.new_empty(shape) if stream is None else _allocated(lambda: like.new_empty(shape), stream)


class _Held:
    """Tensors that a call writes, checked when they are put together; the calls read
    their addresses from ``ptrs``.  Unpacks to the tensors."""
    __slots__ = ("ts", "ptrs", "device", "at")

    def __init__(self, *ts):
        first = next(t for t in ts if t is not None)
        self.ts, self.ptrs = ts, tuple(_ptr(t) for t in ts)
        self.device, self.at = first.device, first.get_device()

    def __iter__(self):
        return iter(self.ts)

    @classmethod
    def _made(cls, device, at, *ts):
        """Of tensors that a call allocated itself: nothing to check."""
        self = object.__new__(cls)
        self.ts, self.ptrs, self.device, self.at = ts, tuple([t.data_ptr() for t in ts]), device, at
        return self


# ------------------------------------------------------------------- pages --
class PageTables:
    """Who has which page: int32 device tensors ``page_table`` [n_seq, entries],
    ``held`` [n_seq] (entries in use), ``free_pages`` [n_pages] (the first
    ``n_free[0]`` of them are free) and ``n_free`` [2] (free pages; entries that the
    last plan lacked)."""

    def __init__(self, page_table, held, free_pages, n_free, *, page_size: int):
        if page_table.dim() != 2:
            raise ValueError("page_table is [n_seq, entries]")
        n_seq, at = page_table.shape[0], page_table.get_device()
        _ints("page_table", page_table, None, at)
        _ints("held", held, n_seq, at)
        _ints("free_pages", free_pages, None, at)
        _ints("n_free", n_free, 2, at)
        self.page_table, self.held, self.free_pages, self.n_free = page_table, held, free_pages, n_free
        self.n_seq, self.entries, self.n_pages, self.page_size = n_seq, page_table.shape[1], free_pages.numel(), page_size
        self.device, self.at = page_table.device, at
        self.ptrs = tuple(t.data_ptr() for t in (page_table, held, free_pages, n_free))

    @classmethod
    def empty(cls, n_pages: int, *, page_size: int, n_seq: int, entries: int, device=None) -> "PageTables":
        """Tables of requests that hold nothing; page 0 is handed out first."""
        torch = _torch()
        device = device or torch.device("cuda")

        def full(shape, x):
            return torch.full(shape, x, dtype=torch.int32, device=device)

        free = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=device)
        n_free = full((2,), 0)
        n_free[0] = n_pages
        return cls(full((n_seq, entries), -1), full((n_seq,), 0), free, n_free, page_size=page_size)


class StepPlan(_Held):
    """What a plan writes: int32 ``cu`` [n_seq + 1] and ``ctx_lens`` [n_seq] (a
    PagedBatch's), ``slots`` int64 [n_tokens] (page * page_size + slot, or -1) and
    ``pos`` int32 [n_tokens]; each of the last two may be None."""
    __slots__ = ("n_seq", "n_tokens")

    def __init__(self, cu, ctx_lens, slots=None, pos=None):
        super().__init__(cu, ctx_lens, slots, pos)
        self.n_seq = ctx_lens.numel()
        _ints("ctx_lens", ctx_lens, None, self.at)
        _ints("cu", cu, self.n_seq + 1, self.at)
        self.n_tokens = next((t.numel() for t in (slots, pos) if t is not None), None)
        if pos is not None:
            _ints("pos", pos, self.n_tokens, self.at)
        if slots is not None:
            _need_cuda(slots)
            if slots.dtype != _torch().int64 or slots.get_device() != self.at:
                raise TypeError("slots is int64, on the device of cu")

    cu, ctx_lens, slots, pos = (property(lambda self, i=i: self.ts[i]) for i in range(4))

    @classmethod
    def empty(cls, tables: PageTables, *, n_tokens: int, rows: bool = True, stream=None) -> "StepPlan":
        """Tensors for a plan to write; without ``rows`` slots and pos are left out."""
        torch = _torch()

        def new(n, dtype=torch.int32):
            return _new_out((n,), dtype, tables.device, stream)

        return cls(new(tables.n_seq + 1), new(tables.n_seq), new(n_tokens, torch.int64) if rows else None,
                   new(n_tokens) if rows else None)


@functools.lru_cache(maxsize=256)
def _plan_desc(*fields):
    d = SpecPlanDesc(*fields)
    return d, ctypes.byref(d)


def spec_plan(tables: PageTables, lens, new_rows, *, n_tokens: Optional[int] = None, trim: bool = False,
              out: Optional[StepPlan] = None, stream=None) -> StepPlan:
    """The step's pages and row maps: requests with ``lens`` [n_seq] positions cached
    and ``new_rows`` [n_seq] to come take from the free list the pages that they
    lack, in order; with ``trim`` those beyond what a request needs go back first
    (all of one with length 0 and no rows).  Pages that the list lacks are left out,
    counted in ``tables.n_free[1]`` and asked for again by the next plan.  Where a
    request's row of the table ends before its length does, ``ctx_lens`` says so, and
    the rows behind are in no page.
    ``n_tokens`` is the rows of the batch (``out``'s maps have as many)."""
    if n_tokens is None:
        n_tokens = out and out.n_tokens
        if n_tokens is None:
            raise ValueError("n_tokens, or an out with maps, must be given")
    if out is None:
        out = StepPlan.empty(tables, n_tokens=n_tokens, stream=stream)
    elif out.n_seq != tables.n_seq or out.n_tokens not in (None, n_tokens):
        raise ValueError("out is of other requests or rows")
    at = tables.at
    _ints("lens", lens, tables.n_seq, at)
    _ints("new_rows", new_rows, tables.n_seq, at)
    _paged._place(tables, out, stream=stream)
    d = _plan_desc(tables.n_seq, n_tokens, tables.page_size, tables.entries, tables.n_pages, 1 if trim else 0)[1]
    _check("lmxs_plan", spec_lib().lmxs_plan(d, lens.data_ptr(), new_rows.data_ptr(), *tables.ptrs, *out.ptrs,
                                             _stream(stream)))
    return out


# ------------------------------------------------------------------- trees --
class SpecTree(_Held):
    """``pos`` int32 [n_tokens] and ``seen`` int64 [n_tokens, words]: bit j of row i's
    words (64 rows a word, lowest first) says that it sees row j of its request."""
    __slots__ = ("words",)

    def __init__(self, pos, seen):
        super().__init__(pos, seen)
        self.words = _words(seen, pos.numel())
        _ints("pos", pos, None, self.at)
        if seen.get_device() != self.at:
            raise ValueError("pos and seen are on one device")

    pos, seen = (property(lambda self, i=i: self.ts[i]) for i in range(2))


def spec_tree(parent, batch: PagedBatch, *, window: int = 0, out: Optional[SpecTree] = None, stream=None) -> SpecTree:
    """Positions and sight of the batch's rows from ``parent`` int32 [n_tokens], the
    row of the request that each continues (earlier than its own; -1: a root).  With
    ``window`` > 0 ancestors that far behind are not seen.  Rows of no request are
    left as they are."""
    n_tokens, at = batch.n_tokens, batch.device.index
    _ints("parent", parent, n_tokens, at)
    if out is None:
        words = -(-batch.max_new // 64)
        out = SpecTree._made(batch.device, at, _fresh(parent, n_tokens, stream),
                             _new_out((n_tokens, words), _torch().int64, batch.device, stream))
        out.words = words
    elif out.pos.numel() != n_tokens:
        raise ValueError("out is of other rows")
    _paged._place(batch, out, stream=stream)
    pos, seen = out.ptrs
    _check("lmxs_tree", spec_lib().lmxs_tree(batch.ref, parent.data_ptr(), out.words, window, pos, seen, _stream(stream)))
    return out


def _words(seen, n_tokens: int) -> int:
    """Words a row of a mask."""
    _need_cuda(seen)
    if seen.dtype != _torch().int64 or seen.dim() != 2 or seen.shape[0] != n_tokens:
        raise ValueError(f"seen is int64 [{n_tokens}, words]")
    return seen.shape[1]


# ---------------------------------------------------- prologue and attention --
@functools.lru_cache(maxsize=256)
def _rope_desc(interleaved: int, turn_scale: float):
    d = SpecRope(interleaved, turn_scale)
    return d, ctypes.byref(d)


def rope_scaling(n_rot: int, *, kind: str, factor: float, rope_base: float = 1e6, trained_ctx: int = 0,
                 fast: float = 32.0, slow: float = 1.0):
    """(rope_factors [n_rot / 2] as a list, turn_scale) that stretch a rotation
    trained on ``trained_ctx`` positions ``factor`` times, for ``spec_prologue``
    (and, with turn_scale 1, ``paged_prologue``):

    * ``linear``  every angle divided by ``factor``
    * ``bands``   pairs that turn more than ``fast`` times in trained_ctx positions
                  keep their angle, those below ``slow`` turns are divided, and in
                  between 1 / divisor goes linearly in the turns
    * ``yarn``    the same with the divisor's reciprocal linear in the pair's index
                  between the two borders, and sine and cosine times
                  0.1 ln(factor) + 1
    """
    if kind not in ("linear", "bands", "yarn"):
        raise ValueError(f"unknown scaling {kind!r}")
    if n_rot < 2 or n_rot % 2 or not factor > 0 or not rope_base > 1:
        raise ValueError("n_rot is even, factor positive and rope_base above 1")
    half = n_rot // 2
    if kind == "linear":
        return [float(factor)] * half, 1.0
    if trained_ctx < 1 or not fast > slow > 0:
        raise ValueError("trained_ctx is positive, and fast above slow above 0")

    def pair(turns):  # index, as a real number, of the pair that turns so often
        return half * math.log(trained_ctx / (2 * math.pi * turns)) / math.log(rope_base)

    out = []
    lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), n_rot - 1)
    for j in range(half):
        if kind == "yarn":
            keep = 1 - min(max((j - lo) / max(hi - lo, 0.001), 0.0), 1.0)
        else:
            turns = trained_ctx / (2 * math.pi) * rope_base ** (-j / half)
            keep = min(max((turns - slow) / (fast - slow), 0.0), 1.0)
        out.append(1 / (keep + (1 - keep) / factor))
    return out, 0.1 * math.log(factor) + 1 if kind == "yarn" and factor > 1 else 1.0


def spec_prologue(q, k, v, cache: PagedCache, batch: PagedBatch, *, n_heads: int, pos=None,
                  n_rot: Optional[int] = None, interleaved: bool = False, turn_scale: float = 1.0,
                  v_norm: bool = False, rms_eps: float = 1e-6, rope_base: float = 1e6, q_gain=None, k_gain=None,
                  rope_factors=None, q_head_stride: Optional[int] = None, q_dtype=None, q_out=None, stream=None):
    """``paged_prologue`` with the rows' positions ``pos`` int32 [n_tokens] apart from
    their slots (None: the slots'), pairs of neighbouring dims where ``interleaved``
    (else half a rotation apart), and sine and cosine times ``turn_scale``."""
    torch = _torch()
    hd = cache.head_dim
    head = q_head_stride or hd
    # the last head's columns behind its head_dim need not exist
    width = q.shape[-1] if q.dim() == 2 else -1
    if not (n_heads - 1) * head + hd <= width <= n_heads * head:
        raise ValueError(f"q is [{batch.n_tokens}, {n_heads * head}], not {list(q.shape)}")
    _rows(q, batch.n_tokens, width, "q")
    if k is None or v is None:
        raise ValueError("k and v must be given")
    dt, kv_stride = _paged._kv_rows(k, v, cache, batch)
    if dt != F32 or q.dtype != torch.float32:
        raise TypeError("q, k and v are float32")
    n_rot = hd if n_rot is None else n_rot
    for g, n in ((q_gain, hd), (k_gain, hd), (rope_factors, n_rot // 2)):
        if g is not None and (g.dtype != torch.float32 or g.numel() < n or not g.is_contiguous()):
            raise ValueError("gains are contiguous float32 [head_dim], factors [n_rot / 2]")
    if pos is not None:
        _ints("pos", pos, batch.n_tokens, cache.at)
    if q_out is None:
        shape = batch.n_tokens, n_heads * hd
        q_out = _fresh(q, shape, stream) if q_dtype is None else _new_out(shape, q_dtype, cache.device, stream)
    elif q_dtype is not None and q_out.dtype != q_dtype:
        raise TypeError("q_dtype differs from q_out's")
    if _rows(q_out, batch.n_tokens, n_heads * hd, "q_out"):
        raise ValueError("q_out must be contiguous")
    _paged._place(cache, batch, q, k, v, q_gain, k_gain, rope_factors, q_out, stream=stream)
    d = _paged._prologue_desc(n_heads, n_rot, int(bool(v_norm)), head, q.stride(0) if batch.n_tokens > 1 else 0,
                              kv_stride, float(rms_eps), float(rope_base))[1]
    r = _rope_desc(int(bool(interleaved)), float(turn_scale))[1]
    _check("lmxs_prologue", spec_lib().lmxs_prologue(
        cache.ref, batch.ref, d, r, _ptr(pos), q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(q_gain), _ptr(k_gain),
        _ptr(rope_factors), q_out.data_ptr(), _paged._dt_of(q_out.dtype), _stream(stream)))
    return q_out


def spec_attention(q, cache: PagedCache, batch: PagedBatch, seen, *, n_heads: int, pos=None, window: int = 0,
                   scale: Optional[float] = None, q_head_stride: Optional[int] = None, out=None,
                   workspace: Optional[Workspace] = None, stream=None):
    """``paged_attention`` of rows that see each other by a mask: each the positions
    before its request's rows (with ``window`` > 0 those above its ``pos`` less the
    window) and the request's rows whose bits are set in its ``seen`` int64
    [n_tokens, words]; one that sees nothing gets zeros.  Types and workspaces are
    ``paged_attention``'s, and its precision, but that with f16 ``q`` the softmax's
    weights always have 22 bits, as with f32."""
    hd = cache.head_dim
    head = q_head_stride or hd
    width = q.shape[-1] if q.dim() == 2 else -1
    if not (n_heads - 1) * head + hd <= width <= n_heads * head:
        raise ValueError(f"q is [{batch.n_tokens}, {n_heads * head}], not {list(q.shape)}")
    _rows(q, batch.n_tokens, width, "q")
    dt = _paged._dt_of(q.dtype)
    words = _words(seen, batch.n_tokens)
    if pos is not None:
        _ints("pos", pos, batch.n_tokens, cache.at)
    if out is None:
        out = _fresh(q, (batch.n_tokens, n_heads * hd), stream)
    elif out.dtype != q.dtype or _rows(out, batch.n_tokens, n_heads * hd, "out"):
        raise ValueError("out is contiguous and of q's dtype")
    _paged._place(cache, batch, q, seen, out, stream=stream, workspace=workspace)
    d = _paged._attn_desc(n_heads, window, head, q.stride(0) if batch.n_tokens > 1 else 0,
                          1.0 / math.sqrt(hd) if scale is None else float(scale))[1]
    L = spec_lib()
    ws_ptr, ws_bytes = _space(L.lmxs_attn_workspace_bytes(cache.ref, batch.ref, d), workspace, cache.device, stream)
    _check("lmxs_attn", L.lmxs_attn(cache.ref, batch.ref, d, seen.data_ptr(), words, _ptr(pos), q.data_ptr(), dt,
                                    out.data_ptr(), _ptr_of(ws_ptr), ws_bytes, _stream(stream)))
    return out


def _space(need: int, workspace: Optional[Workspace], device, stream):
    """(pointer or tensor held for this call, bytes) of ``need`` bytes of workspace;
    nothing need be cleared."""
    if not need:
        return None, 0
    if workspace is None:
        return _new_out((need,), _torch().uint8, device, stream), need
    if need > workspace.nbytes:
        workspace.ensure(need, stream)
    return workspace.base, workspace.nbytes


def _ptr_of(x):
    return x if x is None or isinstance(x, int) else x.data_ptr()


# ------------------------------------------------------------ verification --
class Verified(_Held):
    """int32 ``path`` [n_seq, max_new] (accepted rows within the request, 0 first, then
    -1), ``accepted`` [n_seq] (their number) and ``token`` [n_seq]."""
    __slots__ = ()

    def __init__(self, path, accepted, token):
        super().__init__(path, accepted, token)
        if path.dim() != 2:
            raise ValueError("path is [n_seq, max_new]")
        _ints("path", path, None, self.at)
        _ints("accepted", accepted, path.shape[0], self.at)
        _ints("token", token, path.shape[0], self.at)

    path, accepted, token = (property(lambda self, i=i: self.ts[i]) for i in range(3))

    @classmethod
    def empty(cls, n_seq: int, max_new: int, device, stream=None) -> "Verified":
        """Tensors for a verification to write."""
        return cls._parts(_new_out((n_seq * (max_new + 2),), _torch().int32, device, stream), n_seq, max_new)

    @classmethod
    def _parts(cls, held, n_seq: int, max_new: int) -> "Verified":
        """The three as parts of one allocation (which takes half the time of three)."""
        path, accepted, token = held.split_with_sizes((n_seq * max_new, n_seq, n_seq))
        return cls._made(held.device, held.get_device(), path.view(n_seq, max_new), accepted, token)


@functools.lru_cache(maxsize=256)
def _verify_desc(*fields):
    d = SpecVerifyDesc(*fields)
    return d, ctypes.byref(d), spec_lib().lmxs_verify_workspace_bytes(ctypes.byref(d))


def spec_verify(p, tokens, u, r, cu, *, max_new: int, parent=None, q=None, lens=None, greedy: bool = False,
                out: Optional[Verified] = None, workspace: Optional[Workspace] = None, stream=None) -> Verified:
    """Which drafted rows the target accepts, and the token behind them, distributed as
    the target's own samples.  ``p`` [n_tokens, vocab] (f32 or f16) is the target's
    distribution behind each row, ``tokens`` int32 [n_tokens] the rows' tokens, ``cu``
    the step's row offsets; ``parent`` as ``spec_tree``'s (None: chains).  ``q``
    [n_tokens, vocab] is what each row's children were drawn from; None: they were
    chosen.  ``u`` f32 [n_tokens] decides each row's test, ``r`` f32 [n_seq] the last
    token, both uniform in [0, 1).  With ``greedy`` a child passes if it is the
    largest p's index (p may be logits; u, r and q are not read, u and r may be
    None).  ``lens`` int32 [n_seq], where given, has the accepted rows added."""
    torch = _torch()
    dt = _paged._dt_of(p.dtype)
    if p.dim() != 2:
        raise ValueError("p is [n_tokens, vocab]")
    n_tokens, vocab = p.shape
    n_seq = cu.numel() - 1
    p_stride, q_stride = _rows(p, n_tokens, vocab, "p"), 0
    if q is not None:
        if q.dtype != p.dtype:
            raise TypeError("q is of p's dtype")
        q_stride = _rows(q, n_tokens, vocab, "q")
    at = p.get_device()
    _ints("cu", cu, None, at)
    _ints("tokens", tokens, n_tokens, at)
    if parent is not None:
        _ints("parent", parent, n_tokens, at)
    if lens is not None:
        _ints("lens", lens, n_seq, at)
    if not greedy or u is not None or r is not None:
        for t, n, what in ((u, n_tokens, "u"), (r, n_seq, "r")):
            if t is None or t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
                raise ValueError(f"{what} is contiguous float32 [{n}]")
    if out is None:
        out = Verified._parts(_fresh(cu, n_seq * (max_new + 2), stream), n_seq, max_new)
    elif out.path.shape != (n_seq, max_new):
        raise ValueError("out is of other requests or rows")
    _paged._place(out, out, p, q, u, r, stream=stream, workspace=workspace)
    _, d, need = _verify_desc(n_seq, n_tokens, max_new, vocab, p_stride, q_stride, 1 if greedy else 0)
    ws_ptr, ws_bytes = _space(need, workspace, p.device, stream)
    _check("lmxs_verify", spec_lib().lmxs_verify(
        d, cu.data_ptr(), tokens.data_ptr(), _ptr(parent), p.data_ptr(), _ptr(q), dt, _ptr(u), _ptr(r), *out.ptrs,
        _ptr(lens), _ptr_of(ws_ptr), ws_bytes, _stream(stream)))
    return out


def spec_keep(caches: Sequence[PagedCache], batch: PagedBatch, path, accepted, *, stream=None) -> None:
    """Moves the accepted rows' K and V to the slots behind the cached positions, in
    all ``caches`` (layers of one geometry, whose pages and scales are each its own
    memory) at once: row ``path[b][j]`` of request b to where its row j is.  ``batch`` is
    the step's, ``path`` and ``accepted`` are ``spec_verify``'s."""
    if not caches:
        raise ValueError("caches is empty")
    first = caches[0]
    at, n_seq = first.at, batch.n_seq
    _ints("path", path, None, at)
    _ints("accepted", accepted, n_seq, at)
    if path.dim() != 2 or path.shape[0] != n_seq:
        raise ValueError(f"path is [{n_seq}, entries]")
    _paged._place(first, batch, stream=stream)
    for c in caches:
        if c.at != at:
            raise ValueError("the caches are on one device")
    pools = (_VP * len(caches))(*[c.address for c in caches])
    _check("lmxs_keep", spec_lib().lmxs_keep(pools, len(caches), batch.ref, path.data_ptr(), path.shape[1],
                                             accepted.data_ptr(), _stream(stream)))
