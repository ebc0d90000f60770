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
import math
import struct
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


# The same as bytes, which are made in a quarter of a ctypes structure's time:
# the smallest calls are as long as their Python side.
_pages_bytes, _step_bytes, _call_bytes = (struct.Struct("@" + f) for f in ("2P6q5i0P", "5i11P", "P2qP2q6i2Pif0P"))
_two_bytes = struct.Struct("@2q").pack
assert [f.size for f in (_pages_bytes, _step_bytes, _call_bytes)] == [C.sizeof(t) for t in (_Pages, _Step, _Call)]


class StepTables(NamedTuple):
    """What :func:`kv_tables` returns; int32 except ``slots`` (int64)."""
    kv_len: object     # [B] lengths after the step
    cu_new: object     # [B + 1] prefix sums of the served new positions
    served: object     # [B] 1: the request got what it needs
    n_free: object     # [1] free pages left
    positions: object  # [n_tokens] position of each row in its request, -1: no row
    slots: object      # [n_tokens] its slot in the cache, -1: no row


_L = None
_dt = {}           # torch dtype -> PC_DT_*
_i32 = _i64 = None  # torch.int32, torch.int64
_raw_stream = None  # device index -> handle of torch's current stream


def _entry():
    global _L, _i32, _i64, _raw_stream
    if _L is None:
        import torch
        L = lib()
        vp = C.c_void_p  # structures and strides go as bytes
        L.pc_kv_tables.argtypes = [C.c_int, vp, vp]
        L.pc_kv_store.argtypes = [C.c_int, vp, vp, vp, vp, vp, C.c_int, vp, C.c_int, vp]
        L.pc_attn_create.argtypes = [C.c_int, C.POINTER(vp)]
        L.pc_attn_free.argtypes = [vp]
        L.pc_attn_free.restype = None
        L.pc_attn_paged.argtypes = [vp, vp, vp, vp, C.c_int, vp, vp]
        L.pc_attn_packed.argtypes = [vp, vp, vp, vp, vp, vp, vp]
        L.pc_attn_check.argtypes = [vp, vp]
        for n in ("pc_kv_tables", "pc_kv_store", "pc_attn_create", "pc_attn_paged", "pc_attn_packed",
                  "pc_attn_check"):
            getattr(L, n).restype = C.c_int
        _dt.update({torch.float32: DT_F32, torch.float16: DT_F16, torch.bfloat16: DT_BF16})
        _i32, _i64 = torch.int32, torch.int64
        # the current stream's handle without a Stream object (5 us less a call), where torch has it
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
            (lambda i: torch.cuda.current_stream(i).cuda_stream)
        _L = L
    return _L


def _stream(dev, stream):
    """The stream of a call on device `dev`: torch's current one unless given."""
    return _raw_stream(dev) if stream is None else getattr(stream, "cuda_stream", stream)


def _made(t, stream):
    """A tensor made for a call on `stream`: torch does not hand its memory
    out again before that stream is done with it."""
    if stream is not None:
        import torch
        t.record_stream(stream if hasattr(stream, "cuda_stream") else torch.cuda.ExternalStream(stream, t.device))
    return t


def _int(x):
    """x as a C int; what one does not hold is out of every range the library takes."""
    return min(max(int(x), -1), 0x7fffffff)


def _type(t, name):
    d = _dt.get(t.dtype)
    if d is None:
        raise ValueError(f"{name}: float32, float16 or bfloat16 expected, got {t.dtype}")
    return d


def _ints(t, name, dev, n, dtype):
    """Pointer of a contiguous integer tensor of n elements on device `dev`."""
    if t.dtype is not dtype or t.get_device() != dev or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous {dtype} tensor of {n} elements on cuda:{dev} expected")
    return t.data_ptr()


def _heads3(t, name, dev):
    """(shape, strides) of a [rows, heads, head_dim] tensor with contiguous head_dim."""
    shape, st = t.shape, t.stride()
    if len(shape) != 3 or t.get_device() != dev or (st[2] != 1 and shape[2] != 1):
        raise ValueError(f"{name}: a [rows, heads, head_dim] tensor on cuda:{dev} with contiguous head_dim expected")
    return shape, st


def _pages(k_pages, v_pages, dev):
    """(bytes of the pc_kv_pages, KV heads, head_dim)"""
    shape = k_pages.shape
    ks, vs = k_pages.stride(), v_pages.stride()
    if len(shape) != 4 or v_pages.shape != shape or v_pages.dtype is not k_pages.dtype or k_pages.get_device() != dev \
            or v_pages.get_device() != dev or ks[3] != 1 or vs[3] != 1:
        raise ValueError(f"k_pages, v_pages: two tensors [pages, page_size, kv_heads, head_dim] of one type on cuda:{dev} "
                         "with contiguous head_dim expected")
    n, page, heads, dim = shape
    return _pages_bytes.pack(k_pages.data_ptr(), v_pages.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                             _type(k_pages, "k_pages"), n, page, heads, dim), heads, dim


def kv_tables(kv_len, new_len, page_table, free_pages, n_free, *, page_size: int, n_tokens: int, stream=None) -> StepTables:
    """The tables of one serving step from the requests' lengths (pc_kv_tables).

    ``kv_len``, ``new_len`` [B], ``page_table`` [B, max_pages], ``free_pages``
    [capacity] and ``n_free`` [1] are int32 CUDA tensors; ``new_len[b] < 0``
    ends request b.  ``page_table`` and ``free_pages`` are updated in place;
    the next step's ``kv_len`` and ``n_free`` are returned.  ``n_tokens`` is
    the number of rows of the step's token tensors.
    """
    L = _entry()
    dev, B, width = kv_len.get_device(), kv_len.numel(), page_table.shape[-1]
    if dev < 0 or page_table.shape != (B, width) or not 0 <= n_tokens <= 1 << 28:
        raise ValueError("kv_len on a CUDA device, page_table [requests, max_pages] and n_tokens from 0 to 2^28 expected")
    cap = free_pages.numel()
    if not (kv_len.dtype is new_len.dtype is page_table.dtype is free_pages.dtype is n_free.dtype is _i32
            and new_len.get_device() == page_table.get_device() == free_pages.get_device() == n_free.get_device() == dev
            and new_len.numel() == B and n_free.numel() == 1 and kv_len.is_contiguous() and new_len.is_contiguous()
            and page_table.is_contiguous() and free_pages.is_contiguous()):
        raise ValueError(f"kv_len, new_len [{B}], page_table, free_pages, n_free [1]: contiguous int32 tensors on cuda:{dev} expected")
    # one allocation: cu_new, kv_end, served, n_free, positions
    buf = _made(kv_len.new_empty(3 * B + 2 + n_tokens), stream)
    slots = _made(kv_len.new_empty(n_tokens, dtype=_i64), stream)
    base = buf.data_ptr()
    end = base + 4 * (B + 1)
    served = end + 4 * B
    s = _step_bytes.pack(B, width, _int(page_size), n_tokens, cap, kv_len.data_ptr(), new_len.data_ptr(), n_free.data_ptr(),
                         page_table.data_ptr(), free_pages.data_ptr(), end, base, served, served + 4 * B,
                         served + 4 * B + 4, slots.data_ptr())
    _check(L.pc_kv_tables(dev, s, _stream(dev, stream)))
    cu, end, served, left, pos = buf.split_with_sizes((B + 1, B, B, 1, n_tokens))
    return StepTables(end, cu, served, left, pos, slots)


def kv_store(k_pages, v_pages, k, v, slots, stream=None) -> None:
    """Writes new K and V rows [n, kv_heads, head_dim] to their slots of the
    cache [pages, page_size, kv_heads, head_dim] (pc_kv_store), rounded to its
    type; rows with a slot outside the cache (-1) are skipped."""
    L = _entry()
    dev, n = k.get_device(), slots.numel()
    if dev < 0:
        raise ValueError("k: a CUDA tensor expected")
    p, heads, dim = _pages(k_pages, v_pages, dev)
    shape, ks = _heads3(k, "k", dev)
    vshape, vs = _heads3(v, "v", dev)
    if shape != vshape or k.dtype is not v.dtype or shape != (n, heads, dim):
        raise ValueError(f"k and v: two tensors [{n}, {heads}, {dim}] of one type expected")
    _check(L.pc_kv_store(dev, p, k.data_ptr(), _two_bytes(ks[0], ks[1]), v.data_ptr(), _two_bytes(vs[0], vs[1]),
                         _type(k, "k"), _ints(slots, "slots", dev, n, _i64), n, _stream(dev, stream)))


class Attention:
    """The workspace of the attention calls on one GPU (pc_attn).

    Calls on one handle run one after another: a call on another stream than
    the last one's first makes its stream wait for that one, so programs that
    use several streams want a handle for each.  (A stream given as a bare
    handle has to live until then.)  A graph's replays are not seen here: they
    and other calls on the handle are the caller's to keep apart.
    """

    def __init__(self, device: int = 0):
        h = C.c_void_p()
        _check(_entry().pc_attn_create(device, C.byref(h)))
        self._h, self.device = h, device
        self._last = self._last_given = None  # the last call's stream, and the object it was given as

    def _on(self, stream):
        """The stream of a call, behind the calls before it."""
        st = _stream(self.device, stream)
        if st != self._last:
            self._follow(st, stream)
        return st

    def _follow(self, st, stream):
        import torch

        def of(handle):
            return torch.cuda.ExternalStream(handle, device=self.device) if handle else torch.cuda.default_stream(self.device)

        def capturing(s):
            with torch.cuda.stream(s):
                return torch.cuda.is_current_stream_capturing()

        new = of(st)
        if capturing(new):
            return  # only records; it cannot wait for what is outside its graph
        if self._last is not None:
            old = of(self._last)
            if not capturing(old):
                new.wait_stream(old)
        self._last, self._last_given = st, stream

    def _call(self, q, cu_new, sinks, window, scale, kv_heads, out, stream):
        """(bytes of the pc_attn_call, out, requests)"""
        dev = self.device
        shape, qs = _heads3(q, "q", dev)
        T, H, D = shape
        if out is None:
            out = _made(q.new_empty(shape), stream)
            os = (H * D, D)
        else:
            oshape, os = _heads3(out, "out", dev)
            if oshape != shape or out.dtype is not q.dtype:
                raise ValueError("out: a tensor like q expected")
        sp = 0
        if sinks is not None:
            if _dt.get(sinks.dtype) != DT_F32 or sinks.numel() != H or sinks.get_device() != dev or not sinks.is_contiguous():
                raise ValueError(f"sinks: a contiguous float32 tensor of {H} elements on cuda:{dev} expected")
            sp = sinks.data_ptr()
        n = cu_new.numel()
        return _call_bytes.pack(q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1], _type(q, "q"), H, kv_heads, D, T,
                                n - 1, _ints(cu_new, "cu_new", dev, n, _i32), sp, _int(window),
                                D ** -0.5 if scale is None else scale if -3e38 < scale < 3e38 else math.inf), out, n - 1

    def paged(self, q, k_pages, v_pages, page_table, cu_new, kv_len, *, sinks=None, window: int = 0, scale=None,
              out=None, stream=None):
        """Attention of each request's new rows over its pages (pc_attn_paged).

        ``q`` [rows, heads, head_dim], rows ``cu_new[b] : cu_new[b + 1]`` of
        request b; ``k_pages``, ``v_pages`` [pages, page_size, kv_heads,
        head_dim]; ``page_table`` [B, max_pages], ``cu_new`` [B + 1],
        ``kv_len`` [B] int32: positions in the cache, the new rows' included.
        Rows from ``cu_new[-1]`` on (padding of the step's tensors) are not
        written: in a tensor made by the call they hold anything, NaN too;
        give a zeroed ``out`` where they go on into other operators.
        """
        dev = self.device
        p, heads, _ = _pages(k_pages, v_pages, dev)
        c, out, B = self._call(q, cu_new, sinks, window, scale, heads, out, stream)
        width = page_table.shape[-1]
        if page_table.shape != (B, width):
            raise ValueError(f"page_table: [{B}, max_pages] expected")
        _check(_L.pc_attn_paged(self._h, c, p, _ints(page_table, "page_table", dev, B * width, _i32), width,
                                _ints(kv_len, "kv_len", dev, B, _i32), self._on(stream)))
        return out

    def packed(self, q, k, v, cu_new, *, sinks=None, window: int = 0, scale=None, out=None, stream=None):
        """Attention over whole prompts packed into one tensor (pc_attn_packed):
        ``q`` [rows, heads, head_dim], ``k``, ``v`` [rows, kv_heads, head_dim],
        rows ``cu_new[b] : cu_new[b + 1]`` of prompt b; as with :meth:`paged`,
        rows from ``cu_new[-1]`` on are not written."""
        dev = self.device
        shape, ks = _heads3(k, "k", dev)
        vshape, vs = _heads3(v, "v", dev)
        c, out, _ = self._call(q, cu_new, sinks, window, scale, shape[1], out, stream)
        T, _, D = q.shape
        if shape != vshape or k.dtype is not q.dtype or v.dtype is not q.dtype or shape[0] != T or shape[2] != D:
            raise ValueError("k and v: [rows, kv_heads, head_dim] of q's rows, head_dim and type expected")
        _check(_L.pc_attn_packed(self._h, c, k.data_ptr(), _two_bytes(ks[0], ks[1]), v.data_ptr(),
                                 _two_bytes(vs[0], vs[1]), self._on(stream)))
        return out

    def check(self, stream=None):
        """pc_attn_check: waits for the stream and raises if an earlier call
        on this handle reported a device-side failure."""
        _check(_L.pc_attn_check(self._h, _stream(self.device, stream)))

    def close(self):
        if getattr(self, "_h", None):
            _L.pc_attn_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
