"""Paged KV cache operators (the ``pc_kv_*`` and ``pc_attn_*`` entry points of
include/picchio_b200.h) on torch CUDA tensors.

For programs that keep their own caches: pages of a fixed number of positions
that requests take and give back, one K and one V tensor per layer.  A serving
step is :func:`kv_tables` once, then per layer :func:`kv_store` and
:meth:`Attention.paged` (or :meth:`Attention.packed` while a batch of whole
prompts is read).  Every call runs on torch's current stream of the tensors'
device unless ``stream`` is given, and waits for nothing.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

from .api import _check, lib

DT_F32, DT_F16, DT_BF16 = 0, 1, 2


class _Pages(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("ks0", C.c_int64), ("ks1", C.c_int64), ("ks2", C.c_int64),
                ("vs0", C.c_int64), ("vs1", C.c_int64), ("vs2", C.c_int64),
                ("dtype", C.c_int), ("n_pages", C.c_int), ("page_size", C.c_int), ("n_kv_heads", C.c_int),
                ("head_dim", C.c_int)]


class _Step(C.Structure):
    _fields_ = [("n_requests", C.c_int), ("max_pages", C.c_int), ("page_size", C.c_int), ("n_tokens", C.c_int),
                ("free_cap", C.c_int)] + [(n, C.c_void_p) for n in (
                    "kv_len", "new_len", "n_free", "page_table", "free_pages", "kv_end", "cu_new", "served",
                    "n_free_out", "pos", "slot")]


class _Call(C.Structure):
    _fields_ = [("q", C.c_void_p), ("qs0", C.c_int64), ("qs1", C.c_int64), ("out", C.c_void_p), ("os0", C.c_int64),
                ("os1", C.c_int64),
                ("dtype", C.c_int), ("n_heads", C.c_int), ("n_kv_heads", C.c_int), ("head_dim", C.c_int),
                ("n_rows", C.c_int), ("n_requests", C.c_int), ("cu_new", C.c_void_p), ("sinks", C.c_void_p),
                ("window", C.c_int), ("scale", C.c_float)]


class StepTables(NamedTuple):
    """What :func:`kv_tables` returns; int32 except ``slots`` (int64)."""
    kv_len: object     # [B] lengths after the step
    cu_new: object     # [B + 1] prefix sums of the served new positions
    served: object     # [B] 1: the request got what it needs
    n_free: object     # [1] free pages left
    positions: object  # [n_tokens] position of each row in its request, -1: no row
    slots: object      # [n_tokens] its slot in the cache, -1: no row


_L = None
_dt = {}
_Two = C.c_int64 * 2


def _entry():
    global _L
    if _L is None:
        import torch
        L = lib()
        vp, i64p = C.c_void_p, C.POINTER(C.c_int64)
        L.pc_kv_tables.argtypes = [C.c_int, C.POINTER(_Step), vp]
        L.pc_kv_store.argtypes = [C.c_int, C.POINTER(_Pages), vp, i64p, vp, i64p, C.c_int, vp, C.c_int, vp]
        L.pc_attn_create.argtypes = [C.c_int, C.POINTER(vp)]
        L.pc_attn_free.argtypes = [vp]
        L.pc_attn_free.restype = None
        L.pc_attn_paged.argtypes = [vp, C.POINTER(_Call), C.POINTER(_Pages), vp, C.c_int, vp, vp]
        L.pc_attn_packed.argtypes = [vp, C.POINTER(_Call), vp, i64p, vp, i64p, vp]
        L.pc_attn_check.argtypes = [vp, vp]
        for n in ("pc_kv_tables", "pc_kv_store", "pc_attn_create", "pc_attn_paged", "pc_attn_packed",
                  "pc_attn_check"):
            getattr(L, n).restype = C.c_int
        _dt.update({torch.float32: DT_F32, torch.float16: DT_F16, torch.bfloat16: DT_BF16, "i32": torch.int32,
                    "i64": torch.int64, "empty": torch.empty,
                    # the current stream's handle without a Stream object (5 us less a call), where torch has it
                    "stream": getattr(torch._C, "_cuda_getCurrentRawStream", None)
                    or (lambda i: torch.cuda.current_stream(i).cuda_stream)})
        _L = L
    return _L


def _stream(dev, stream):
    if stream is not None:
        return getattr(stream, "cuda_stream", stream)
    return _dt["stream"](dev.index)


def _type(t, name):
    d = _dt.get(t.dtype)
    if d is None:
        raise ValueError(f"{name}: float32, float16 or bfloat16 expected, got {t.dtype}")
    return d


def _ints(t, name, dev, n=None, dtype="i32"):
    """Pointer of a contiguous integer tensor on `dev` (of n elements, if given)."""
    if t.dtype != _dt[dtype] or not t.is_contiguous() or t.device != dev or (n is not None and t.numel() != n):
        raise ValueError(f"{name}: a contiguous {_dt[dtype]} tensor{'' if n is None else f' of {n} elements'} on {dev} expected")
    return t.data_ptr()


def _heads3(t, name, dev):
    """(shape, strides) of a [rows, heads, head_dim] tensor with contiguous head_dim."""
    shape, st = t.shape, t.stride()
    if len(shape) != 3 or t.device != dev or (st[2] != 1 and shape[2] != 1):
        raise ValueError(f"{name}: a [rows, heads, head_dim] tensor on {dev} with contiguous head_dim expected")
    return shape, st


def _pages(k_pages, v_pages) -> _Pages:
    shape = k_pages.shape
    ks, vs = k_pages.stride(), v_pages.stride()
    if len(shape) != 4 or v_pages.shape != shape or v_pages.dtype != k_pages.dtype or v_pages.device != k_pages.device \
            or not k_pages.is_cuda or ks[3] != 1 or vs[3] != 1:
        raise ValueError("k_pages, v_pages: two CUDA tensors [pages, page_size, kv_heads, head_dim] of one type with "
                         "contiguous head_dim expected")
    return _Pages(k_pages.data_ptr(), v_pages.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                  _type(k_pages, "k_pages"), shape[0], shape[1], shape[2], shape[3])


def kv_tables(kv_len, new_len, page_table, free_pages, n_free, *, page_size: int, n_tokens: int, stream=None) -> StepTables:
    """The tables of one serving step from the requests' lengths (pc_kv_tables).

    ``kv_len``, ``new_len`` [B], ``page_table`` [B, max_pages], ``free_pages``
    [capacity] and ``n_free`` [1] are int32 CUDA tensors; ``new_len[b] < 0``
    ends request b.  ``page_table`` and ``free_pages`` are updated in place;
    the next step's ``kv_len`` and ``n_free`` are returned.  ``n_tokens`` is
    the number of rows of the step's token tensors.
    """
    L = _entry()
    dev = kv_len.device
    B = kv_len.numel()
    if page_table.dim() != 2 or page_table.shape[0] != B or n_tokens < 0:
        raise ValueError("page_table: [requests, max_pages] expected, and n_tokens >= 0")
    # one allocation: cu_new, kv_end, served, n_free, positions
    empty = _dt["empty"]
    buf = empty(3 * B + 2 + n_tokens, dtype=_dt["i32"], device=dev)
    slots = empty(n_tokens, dtype=_dt["i64"], device=dev)
    cu, end, served, left, pos = buf.split_with_sizes((B + 1, B, B, 1, n_tokens))
    out = StepTables(end, cu, served, left, pos, slots)
    base = buf.data_ptr()
    s = _Step(B, page_table.shape[1], page_size, n_tokens, free_pages.numel(), _ints(kv_len, "kv_len", dev),
              _ints(new_len, "new_len", dev, B), _ints(n_free, "n_free", dev, 1),
              _ints(page_table, "page_table", dev), _ints(free_pages, "free_pages", dev), base + 4 * (B + 1), base,
              base + 4 * (2 * B + 1), base + 4 * (3 * B + 1), base + 4 * (3 * B + 2), slots.data_ptr())
    _check(L.pc_kv_tables(dev.index, C.byref(s), _stream(dev, stream)))
    return out


def kv_store(k_pages, v_pages, k, v, slots, stream=None) -> None:
    """Writes new K and V rows [n, kv_heads, head_dim] to their slots of the
    cache [pages, page_size, kv_heads, head_dim] (pc_kv_store), rounded to its
    type; rows with a slot outside the cache (-1) are skipped."""
    L = _entry()
    p = _pages(k_pages, v_pages)
    dev, n = k_pages.device, slots.numel()
    shape, ks = _heads3(k, "k", dev)
    vshape, vs = _heads3(v, "v", dev)
    if shape != vshape or k.dtype != v.dtype or shape != (n, p.n_kv_heads, p.head_dim):
        raise ValueError(f"k and v: two tensors [{n}, {p.n_kv_heads}, {p.head_dim}] of one type expected")
    _check(L.pc_kv_store(dev.index, C.byref(p), k.data_ptr(), _Two(ks[0], ks[1]), v.data_ptr(), _Two(vs[0], vs[1]),
                         _type(k, "k"), _ints(slots, "slots", dev, dtype="i64"), n, _stream(dev, stream)))


class Attention:
    """The workspace of the attention calls on one GPU (pc_attn); calls on one
    handle run one after another, so use one per stream."""

    def __init__(self, device: int = 0):
        h = C.c_void_p()
        _check(_entry().pc_attn_create(device, C.byref(h)))
        self._h, self.device = h, device

    def _call(self, q, cu_new, sinks, window, scale, kv_heads, out):
        dev = q.device
        if dev.type != "cuda" or dev.index != self.device:
            raise ValueError(f"q: a tensor on cuda:{self.device} expected")
        shape, qs = _heads3(q, "q", dev)
        T, H, D = shape
        if out is None:
            out = _dt["empty"](shape, dtype=q.dtype, device=dev)
            os = (H * D, D)
        else:
            oshape, os = _heads3(out, "out", dev)
            if oshape != shape or out.dtype != q.dtype:
                raise ValueError("out: a tensor like q expected")
        sp = None
        if sinks is not None:
            if _dt.get(sinks.dtype) != DT_F32 or sinks.numel() != H or not sinks.is_contiguous() or sinks.device != dev:
                raise ValueError(f"sinks: a contiguous float32 tensor of {H} elements on {dev} expected")
            sp = sinks.data_ptr()
        return _Call(q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1], _type(q, "q"), H, kv_heads, D, T,
                     cu_new.numel() - 1, _ints(cu_new, "cu_new", dev), sp, int(window),
                     D ** -0.5 if scale is None else scale), out

    def paged(self, q, k_pages, v_pages, page_table, cu_new, kv_len, *, sinks=None, window: int = 0, scale=None,
              out=None, stream=None):
        """Attention of each request's new rows over its pages (pc_attn_paged).

        ``q`` [rows, heads, head_dim], rows ``cu_new[b] : cu_new[b + 1]`` of
        request b; ``k_pages``, ``v_pages`` [pages, page_size, kv_heads,
        head_dim]; ``page_table`` [B, max_pages], ``cu_new`` [B + 1],
        ``kv_len`` [B] int32: positions in the cache, the new rows' included.
        """
        p = _pages(k_pages, v_pages)
        c, out = self._call(q, cu_new, sinks, window, scale, p.n_kv_heads, out)
        dev = q.device
        if page_table.dim() != 2 or page_table.shape[0] != c.n_requests or k_pages.device != dev:
            raise ValueError("page_table: [requests, max_pages] expected, on one device with q and the pages")
        _check(_L.pc_attn_paged(self._h, C.byref(c), C.byref(p), _ints(page_table, "page_table", dev),
                                page_table.shape[1], _ints(kv_len, "kv_len", dev, c.n_requests), _stream(dev, stream)))
        return out

    def packed(self, q, k, v, cu_new, *, sinks=None, window: int = 0, scale=None, out=None, stream=None):
        """Attention over whole prompts packed into one tensor (pc_attn_packed):
        ``q`` [rows, heads, head_dim], ``k``, ``v`` [rows, kv_heads, head_dim],
        rows ``cu_new[b] : cu_new[b + 1]`` of prompt b."""
        c, out = self._call(q, cu_new, sinks, window, scale, k.shape[1], out)
        dev = q.device
        shape, ks = _heads3(k, "k", dev)
        vshape, vs = _heads3(v, "v", dev)
        if shape != vshape or k.dtype != q.dtype or v.dtype != q.dtype or shape[0] != c.n_rows or shape[2] != c.head_dim:
            raise ValueError("k and v: [rows, kv_heads, head_dim] of q's rows, head_dim and type expected")
        _check(_L.pc_attn_packed(self._h, C.byref(c), k.data_ptr(), _Two(ks[0], ks[1]), v.data_ptr(), _Two(vs[0], vs[1]),
                                 _stream(dev, stream)))
        return out

    def check(self, stream=None):
        """pc_attn_check: waits for the stream and raises if an earlier call
        on this handle reported a device-side failure."""
        import torch
        _check(_L.pc_attn_check(self._h, _stream(torch.device("cuda", self.device), stream)))

    def close(self):
        if getattr(self, "_h", None):
            _L.pc_attn_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
