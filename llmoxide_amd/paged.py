"""The paged KV cache (include/lmx/paged.h): writing it, reading it back, the
prologue in front of it and attention over it, for ragged batches of prompt
chunks and single tokens.

=====================  ======================================================
this module            what it is the paged, ragged form of
=====================  ======================================================
``paged_append``       ``write_cache`` (ops.wgsl:323-346), into f16 or 8 bits
``paged_read``         (new) the written rows back, as contiguous K and V
``paged_prologue``     per-head ``rms_norm`` + ``rope`` on Q and K, K/V store
                       (ops.wgsl:49-91, 186-218, 269-306, 323-346)
``paged_attention``    ``scores_pass``/``softmax_pass``/``weighted_v``
                       (attn.wgsl:84-232; cpu.rs:342-387)
=====================  ======================================================

A :class:`PagedCache` holds the pages of one layer, a :class:`PagedBatch` says
which rows a call brings and where they live.  Both are made once and kept: a
call reads the lengths and the page table on the device, so a captured graph
replays with what these tensors hold then.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional

from . import F16, F32, Workspace, _check, _need_cuda, _ptr, _stream, _torch, lib

STORE_F16, STORE_I8 = 1, 2

_U32, _VP = ctypes.c_uint32, ctypes.c_void_p


class PoolDesc(ctypes.Structure):
    """lmxp_pool."""
    _fields_ = [("n_pages", _U32), ("page_size", _U32), ("n_kv_heads", _U32), ("head_dim", _U32),
                ("store", _U32), ("k", _VP), ("v", _VP), ("k_scale", _VP), ("v_scale", _VP)]


class BatchDesc(ctypes.Structure):
    """lmxp_batch."""
    _fields_ = [("n_seq", _U32), ("n_tokens", _U32), ("max_new", _U32), ("max_ctx", _U32),
                ("table_stride", _U32), ("cu", _VP), ("ctx_lens", _VP), ("page_table", _VP)]


class PagedPrologueDesc(ctypes.Structure):
    """lmxp_prologue_desc."""
    _fields_ = [("n_heads", _U32), ("n_rot", _U32), ("v_norm", _U32), ("q_head_stride", _U32),
                ("q_row_stride", _U32), ("kv_row_stride", _U32), ("rms_eps", ctypes.c_float),
                ("rope_base", ctypes.c_float)]


class PagedAttnDesc(ctypes.Structure):
    """lmxp_attn_desc."""
    _fields_ = [("n_heads", _U32), ("window", _U32), ("q_head_stride", _U32), ("q_row_stride", _U32),
                ("scale", ctypes.c_float)]


_PP, _PB = ctypes.POINTER(PoolDesc), ctypes.POINTER(BatchDesc)
_PR, _PA = ctypes.POINTER(PagedPrologueDesc), ctypes.POINTER(PagedAttnDesc)
_I = ctypes.c_int
# Every symbol include/lmx/paged.h declares.
SIGNATURES = {
    "lmxp_append": (_I, [_PP, _PB, _VP, _VP, _I, _U32, _VP]),
    "lmxp_read": (_I, [_PP, _PB, _VP, _VP, _I, _U32, _VP]),
    "lmxp_prologue": (_I, [_PP, _PB, _PR, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _I, _VP]),
    "lmxp_attn_workspace_bytes": (ctypes.c_size_t, [_PP, _PB, _PA]),
    "lmxp_attn": (_I, [_PP, _PB, _PA, _VP, _I, _VP, _VP, ctypes.c_size_t, _VP]),
}

_lib = None


def paged_lib() -> ctypes.CDLL:
    """The library with lmx/paged.h's signatures set; raises if it is missing."""
    global _lib
    if _lib is None:
        L = lib()
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _lib = L
    return _lib


_dts = None


def _dt_of(dtype) -> int:
    global _dts
    if _dts is None:
        torch = _torch()
        _dts = {torch.float32: F32, torch.float16: F16}
    dt = _dts.get(dtype)
    if dt is None:
        raise TypeError(f"unsupported dtype {dtype}")
    return dt


class PagedCache:
    """One layer's pages: ``k`` [n_pages, n_kv_heads, page_size, head_dim] and
    ``v`` [n_pages, n_kv_heads, head_dim, page_size] (V is kept transposed), f16,
    or int8 with f32 ``k_scale``, ``v_scale`` [n_pages, n_kv_heads, page_size]."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        torch = _torch()
        _need_cuda(k, v, k_scale, v_scale)
        if k.dim() != 4 or v.shape != (k.shape[0], k.shape[1], k.shape[3], k.shape[2]):
            raise ValueError("k is [pages, kv_heads, page, head_dim], v [pages, kv_heads, head_dim, page]")
        if k.dtype != v.dtype or k.dtype not in (torch.float16, torch.int8):
            raise TypeError(f"pages are float16 or int8, not {k.dtype} and {v.dtype}")
        if (k.dtype == torch.int8) != (k_scale is not None) or (k_scale is None) != (v_scale is None):
            raise ValueError("int8 pages have a k_scale and a v_scale, float16 pages neither")
        for s in (k_scale, v_scale):
            if s is not None and (s.dtype != torch.float32 or s.shape != k.shape[:3]):
                raise ValueError("scales are float32 [pages, kv_heads, page]")
        for t in (v, k_scale, v_scale):
            if t is not None and t.device != k.device:
                raise ValueError("a cache's tensors are on one device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.device = k.device
        self.dtype = k.dtype
        store = STORE_I8 if k.dtype == torch.int8 else STORE_F16
        self.desc = PoolDesc(self.n_pages, self.page_size, self.n_kv_heads, self.head_dim, store,
                             _ptr(k), _ptr(v), _ptr(k_scale), _ptr(v_scale))
        self.ref = ctypes.byref(self.desc)

    @classmethod
    def empty(cls, n_pages: int, *, page_size: int, n_kv_heads: int, head_dim: int, dtype=None,
              device=None) -> "PagedCache":
        """Fresh pages of ``dtype`` (float16 unless int8 is asked for); what they
        hold before they are written is unspecified."""
        torch = _torch()
        dtype = dtype or torch.float16
        device = device or torch.device("cuda")
        k = torch.empty((n_pages, n_kv_heads, page_size, head_dim), dtype=dtype, device=device)
        v = torch.empty((n_pages, n_kv_heads, head_dim, page_size), dtype=dtype, device=device)
        scales = [torch.empty((n_pages, n_kv_heads, page_size), dtype=torch.float32, device=device)
                  for _ in range(2)] if dtype == torch.int8 else [None, None]
        return cls(k, v, *scales)


class PagedBatch:
    """A batch's rows: int32 device tensors ``cu`` [n_seq + 1] (sequence b brings
    rows cu[b]:cu[b+1]), ``ctx_lens`` [n_seq] (lengths, the new rows counted) and
    ``page_table`` [n_seq, entries]; entries that are no page (-1) hide their
    positions.  ``n_tokens`` is the rows of the batch's tensors, ``max_new`` and
    ``max_ctx`` are bounds of the rows and the length of a sequence."""

    def __init__(self, cu, ctx_lens, page_table, *, n_tokens: int, max_new: int, max_ctx: int):
        torch = _torch()
        _need_cuda(cu, ctx_lens, page_table)
        for t in (cu, ctx_lens, page_table):
            if t.dtype != torch.int32:
                raise TypeError("cu, ctx_lens and page_table are int32")
            if t.device != cu.device:
                raise ValueError("a batch's tensors are on one device")
        n_seq = ctx_lens.numel()
        if cu.numel() != n_seq + 1 or page_table.dim() != 2 or page_table.shape[0] != n_seq:
            raise ValueError("cu is [n_seq + 1], ctx_lens [n_seq], page_table [n_seq, entries]")
        self.cu, self.ctx_lens, self.page_table = cu, ctx_lens, page_table
        self.n_seq, self.n_tokens, self.max_new, self.max_ctx = n_seq, n_tokens, max_new, max_ctx
        self.device = cu.device
        self.desc = BatchDesc(n_seq, n_tokens, max_new, max_ctx, page_table.shape[1], _ptr(cu),
                              _ptr(ctx_lens), _ptr(page_table))
        self.ref = ctypes.byref(self.desc)


_current_device = None


def _place(cache: PagedCache, batch: PagedBatch, *ts, stream=None, workspace=None) -> None:
    """All on the current device: the stream a call takes is that device's."""
    global _current_device
    if _current_device is None:
        torch = _torch()
        _current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
    at = cache.device.index
    if batch.device.index != at or at != _current_device():
        raise ValueError("cache and batch must be on the current device")
    for t in ts:
        if t is not None and t.get_device() != at:  # -1: the CPU's
            raise ValueError("tensors must be on the cache's device")
    if stream is not None and getattr(stream, "device_index", at) != at:
        raise ValueError("the stream must be one of the cache's device")
    if workspace is not None:
        if workspace.buf is not None:
            held = workspace.buf.get_device()
        else:  # where it will be allocated; no index: the current device
            held = None if workspace.device is None else _torch().device(workspace.device).index
        if held is not None and held != at:
            raise ValueError("the workspace must be on the cache's device")


@functools.lru_cache(maxsize=256)
def _attn_desc(n_heads: int, window: int, head: int, row: int, scale: float):
    """(structure, reference) of an attention call's scalars."""
    d = PagedAttnDesc(n_heads, window, head, row, scale)
    return d, ctypes.byref(d)


@functools.lru_cache(maxsize=256)
def _prologue_desc(*fields):
    """The same of a prologue call's."""
    d = PagedPrologueDesc(*fields)
    return d, ctypes.byref(d)


def _rows(t, n_tokens: int, width: int, what: str) -> int:
    """Row stride of a [n_tokens, width] tensor whose rows may be columns of a
    wider one (0: dense)."""
    if t.shape != (n_tokens, width):
        raise ValueError(f"{what} is [{n_tokens}, {width}], not {list(t.shape)}")
    row, col = t.stride()
    if col != 1:
        raise ValueError(f"{what}'s rows must be contiguous")
    if n_tokens == 1 or row == width:
        return 0
    if not width < row < 1 << 32:
        raise ValueError(f"{what}'s rows must not share memory, nor lie 2^32 elements apart")
    return row


def _kv_rows(k, v, cache: PagedCache, batch: PagedBatch, names=("k", "v")):
    """(dtype code, row stride) of a pair of which either may be None."""
    width = cache.n_kv_heads * cache.head_dim
    some = k if k is not None else v
    if some is None:
        raise ValueError(f"{names[0]} or {names[1]} must be given")
    stride = _rows(some, batch.n_tokens, width, names[0] if k is not None else names[1])
    if k is not None and v is not None and (_rows(v, batch.n_tokens, width, names[1]) != stride or v.dtype != k.dtype):
        raise ValueError(f"{names[0]} and {names[1]} have one dtype and one row stride")
    return _dt_of(some.dtype), stride


def paged_append(k, v, cache: PagedCache, batch: PagedBatch, *, stream=None) -> None:
    """Write the batch's rows ``k``, ``v`` [n_tokens, n_kv_heads * head_dim] (f32 or
    f16; columns of a wider tensor will do) into their pages.  Either may be None."""
    dt, stride = _kv_rows(k, v, cache, batch)
    _place(cache, batch, k, v, stream=stream)
    _check("lmxp_append", paged_lib().lmxp_append(cache.ref, batch.ref, _ptr(k), _ptr(v), dt, stride,
                                                  _stream(stream)))


def _new_out(shape, dtype, device, stream):
    """A result allocated here; one that another stream fills is marked as used there."""
    torch = _torch()
    out = torch.empty(shape, dtype=dtype, device=device)
    if stream is not None and stream != torch.cuda.current_stream():
        out.record_stream(stream)
    return out


def paged_read(cache: PagedCache, batch: PagedBatch, *, dtype=None, k_out=None, v_out=None, stream=None):
    """The batch's rows back from the pages: (k, v), each [n_tokens, n_kv_heads *
    head_dim] of ``dtype`` (float32 unless float16 is asked for).  Without outputs
    given both are allocated; rows of no sequence are left as they are there."""
    torch = _torch()
    if k_out is None and v_out is None:
        shape = (batch.n_tokens, cache.n_kv_heads * cache.head_dim)
        k_out = _new_out(shape, dtype or torch.float32, cache.device, stream)
        v_out = _new_out(shape, dtype or torch.float32, cache.device, stream)
    elif dtype is not None and any(t is not None and t.dtype != dtype for t in (k_out, v_out)):
        raise TypeError("dtype differs from the outputs'")
    dt, stride = _kv_rows(k_out, v_out, cache, batch, ("k_out", "v_out"))
    _place(cache, batch, k_out, v_out, stream=stream)
    _check("lmxp_read", paged_lib().lmxp_read(cache.ref, batch.ref, _ptr(k_out), _ptr(v_out), dt, stride,
                                              _stream(stream)))
    return k_out, v_out


def paged_prologue(q, k, v, cache: PagedCache, batch: PagedBatch, *, n_heads: int,
                   n_rot: Optional[int] = None, v_norm: bool = False, rms_eps: float = 1e-6,
                   rope_base: float = 1e6, q_gain=None, k_gain=None, rope_factors=None,
                   q_head_stride: Optional[int] = None, q_dtype=None, q_out=None, stream=None):
    """Per-head RMS norm (gain), NeoX rotation over ``n_rot`` dims at each row's
    position, and the store of K and V into their pages, in one launch.  ``q``
    [n_tokens, n_heads * q_head_stride], ``k``, ``v`` [n_tokens, n_kv_heads * head_dim]
    are f32 rows (columns of a wider tensor will do); returns q_out [n_tokens,
    n_heads * head_dim] of ``q_dtype`` (float32 unless float16 is asked for)."""
    torch = _torch()
    hd = cache.head_dim
    head = q_head_stride or hd
    # the last head's columns behind its head_dim need not exist
    width = q.shape[-1] if q.dim() == 2 else -1
    if not (n_heads - 1) * head + hd <= width <= n_heads * head:
        raise ValueError(f"q is [{batch.n_tokens}, {n_heads * head}], not {list(q.shape)}")
    _rows(q, batch.n_tokens, width, "q")
    dt, kv_stride = _kv_rows(k, v, cache, batch)
    if k is None or v is None or dt != F32 or q.dtype != torch.float32:
        raise TypeError("q, k and v are float32")
    n_rot = hd if n_rot is None else n_rot
    for g, n in ((q_gain, hd), (k_gain, hd), (rope_factors, n_rot // 2)):
        if g is not None and (g.dtype != torch.float32 or g.numel() < n or not g.is_contiguous()):
            raise ValueError("gains are contiguous float32 [head_dim], factors [n_rot / 2]")
    if q_out is None:
        q_out = _new_out((batch.n_tokens, n_heads * hd), q_dtype or torch.float32, cache.device, stream)
    elif q_dtype is not None and q_out.dtype != q_dtype:
        raise TypeError("q_dtype differs from q_out's")
    if _rows(q_out, batch.n_tokens, n_heads * hd, "q_out"):
        raise ValueError("q_out must be contiguous")
    _place(cache, batch, q, k, v, q_gain, k_gain, rope_factors, q_out, stream=stream)
    dref = _prologue_desc(n_heads, n_rot, int(bool(v_norm)), head, q.stride(0) if batch.n_tokens > 1 else 0,
                          kv_stride, float(rms_eps), float(rope_base))[1]
    _check("lmxp_prologue", paged_lib().lmxp_prologue(
        cache.ref, batch.ref, dref, q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(q_gain), _ptr(k_gain),
        _ptr(rope_factors), q_out.data_ptr(), _dt_of(q_out.dtype), _stream(stream)))
    return q_out


def paged_attention(q, cache: PagedCache, batch: PagedBatch, *, n_heads: int, window: int = 0,
                    scale: Optional[float] = None, q_head_stride: Optional[int] = None, out=None,
                    workspace: Optional[Workspace] = None, stream=None):
    """Causal GQA attention of the batch's rows ``q`` [n_tokens, n_heads * head_dim]
    (f32 or f16; columns of a wider tensor will do) over the pages, where their own
    K and V already are.  Returns out [n_tokens, n_heads * head_dim] of q's dtype;
    ``window`` > 0 limits a row to its last ``window`` positions.  Rows of no
    sequence are left as they are.  With f16 ``q`` the softmax's weights have 11
    bits where a sequence brings many rows (new rows times heads / kv heads above 32
    to 128), 22 elsewhere and always with f32 ``q``.  A ``workspace`` that served a batch serves all
    whose ``n_seq``, ``n_tokens``, ``max_new`` and ``max_ctx`` are no larger without
    growing (and moving, which a captured graph would not notice)."""
    hd = cache.head_dim
    head = q_head_stride or hd
    width = q.shape[-1] if q.dim() == 2 else -1
    if not (n_heads - 1) * head + hd <= width <= n_heads * head:
        raise ValueError(f"q is [{batch.n_tokens}, {n_heads * head}], not {list(q.shape)}")
    _rows(q, batch.n_tokens, width, "q")
    dt = _dt_of(q.dtype)
    if out is None:
        out = _new_out((batch.n_tokens, n_heads * hd), q.dtype, cache.device, stream)
    elif out.dtype != q.dtype or _rows(out, batch.n_tokens, n_heads * hd, "out"):
        raise ValueError("out is contiguous and of q's dtype")
    _place(cache, batch, q, out, stream=stream, workspace=workspace)
    dref = _attn_desc(n_heads, window, head, q.stride(0) if batch.n_tokens > 1 else 0,
                      1.0 / math.sqrt(hd) if scale is None else float(scale))[1]
    L = paged_lib()
    need = L.lmxp_attn_workspace_bytes(cache.ref, batch.ref, dref)
    ws_ptr, ws_bytes = None, 0
    if need and workspace is None:
        held = _new_out((need,), _torch().uint8, cache.device, stream)  # for this call; nothing need be cleared
        ws_ptr, ws_bytes = held.data_ptr(), need
    elif need:
        if need > workspace.nbytes:
            workspace.ensure(need, stream)
        ws_ptr, ws_bytes = workspace.base, workspace.nbytes
    _check("lmxp_attn", L.lmxp_attn(cache.ref, batch.ref, dref, q.data_ptr(), dt, out.data_ptr(), ws_ptr, ws_bytes,
                                    _stream(stream)))
    return out
