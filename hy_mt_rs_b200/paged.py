"""A KV cache of pages and the operators over it (include/hyq.h, hyq_paged_*
and hyq_pages_*): RoPE + q/k norm + append, attention of ragged chunks of new
tokens, and reserving, freeing, forking and compacting the pages on the device.

A layer's keys and values are tensors [pages, kv_heads, page_size, head_dim]
(float32 or float16; any strides with a contiguous last dimension, so a
permuted [pages, page_size, kv_heads, head_dim] tensor works too).  A batch of
new tokens is ragged: rows row_start[s] .. row_start[s + 1] - 1 of the
activations belong to sequence s, at positions pos[s] ..; its pages are row
slot[s] of the table (row s without slots).  Indexes are device int32 tensors.
Every call runs on the current torch CUDA stream.
"""
import ctypes as C

import torch

from ._native import HyqError, check, lib
from .quant import _need_cuda, _ptr, _stream

__all__ = ["PagedCache", "rope_append", "attention", "attention_workspace"]

_KV_TYPES = {torch.float32: 0, torch.float16: 1}   # HYQ_KV_F32, HYQ_KV_F16


class _Kv(C.Structure):
    """hyq_paged_kv (include/hyq.h)."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("dtype", C.c_int), ("kv_heads", C.c_int),
                ("head_dim", C.c_int), ("page_size", C.c_int), ("pages", C.c_int64), ("page_stride", C.c_int64),
                ("head_stride", C.c_int64), ("row_stride", C.c_int64), ("table", C.c_void_p), ("slots", C.c_int64),
                ("table_width", C.c_int64)]


class _Batch(C.Structure):
    """hyq_paged_batch (include/hyq.h)."""
    _fields_ = [("slot", C.c_void_p), ("row_start", C.c_void_p), ("pos", C.c_void_p), ("seqs", C.c_int64),
                ("tokens", C.c_int64), ("max_new", C.c_int64), ("max_len", C.c_int64)]


class _Pages(C.Structure):
    """hyq_pages (include/hyq.h)."""
    _fields_ = [("table", C.c_void_p), ("length", C.c_void_p), ("refs", C.c_void_p), ("shortage", C.c_void_p),
                ("slots", C.c_int64), ("table_width", C.c_int64), ("pages", C.c_int64), ("page_size", C.c_int)]


class _Pool(C.Structure):
    """hyq_page_pool (include/hyq.h)."""
    _fields_ = [("base", C.c_void_p), ("planes", C.c_int64), ("plane_stride", C.c_int64), ("page_stride", C.c_int64),
                ("page_bytes", C.c_int64)]


def _kv(k_pages, v_pages, table):
    for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _KV_TYPES:
            raise HyqError(-1, f"{name}: expected a CUDA float32 or float16 tensor")
        if t.dim() != 4 or t.stride(3) != 1:
            raise HyqError(-2, f"{name}: expected [pages, kv_heads, page_size, head_dim], contiguous in head_dim")
    if k_pages.shape != v_pages.shape or k_pages.stride() != v_pages.stride() or k_pages.dtype != v_pages.dtype:
        raise HyqError(-2, "k_pages and v_pages differ in shape, strides or type")
    _need_cuda(table, "table", torch.int32)
    if table.dim() != 2:
        raise HyqError(-2, "table: expected [slots, table_width]")
    pages, heads, page, dim = k_pages.shape
    return _Kv(k_pages.data_ptr(), v_pages.data_ptr(), _KV_TYPES[k_pages.dtype], heads, dim, page, pages,
               k_pages.stride(0), k_pages.stride(1), k_pages.stride(2), table.data_ptr(), table.shape[0], table.shape[1])


def _batch(row_start, pos, slot, tokens, max_new, max_len):
    _need_cuda(row_start, "row_start", torch.int32)
    _need_cuda(pos, "pos", torch.int32)
    seqs = pos.numel()
    if row_start.numel() != seqs + 1:
        raise HyqError(-2, "row_start takes one more entry than pos")
    if slot is not None:
        _need_cuda(slot, "slot", torch.int32)
        if slot.numel() != seqs:
            raise HyqError(-2, "slot takes one entry per sequence")
    return _Batch(None if slot is None else slot.data_ptr(), row_start.data_ptr(), pos.data_ptr(), seqs, tokens,
                  max_new, max_len)


def _heads(t, name):
    """[tokens, heads, head_dim] float32 activations whose heads are contiguous."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.float32:
        raise HyqError(-1, f"{name}: expected a CUDA float32 tensor")
    if t.dim() != 3 or t.stride(2) != 1 or t.stride(1) != t.shape[2]:
        raise HyqError(-2, f"{name}: expected [tokens, heads, head_dim] with contiguous heads")
    return max(t.stride(0), t.shape[1] * t.shape[2])


def rope_append(q, k, v, k_pages, v_pages, table, row_start, pos, cos, sin, q_norm=None, k_norm=None, eps=1e-5,
                norm_first=False, slot=None, out=None):
    """hyq_paged_rope_append: rotate and normalise the heads of q [tokens,
    heads, head_dim] and k [tokens, kv_heads, head_dim] at their positions,
    write k and v into the pages, return the rotated queries (into `out` when
    given; q itself is allowed).  cos and sin are [positions, head_dim / 2]
    (hyq_rope_table); norm_first normalises before the rotation."""
    kv = _kv(k_pages, v_pages, table)
    qs, ks, vs = _heads(q, "q"), _heads(k, "k"), _heads(v, "v")
    out = torch.empty(q.shape, device=q.device) if out is None else out
    os = _heads(out, "out")
    if q.shape[2] != kv.head_dim or out.shape != q.shape or k.shape != (q.shape[0], kv.kv_heads, kv.head_dim) \
            or v.shape != k.shape:
        raise HyqError(-2, "rope_append: shapes of q, k, v and out")
    for t, name, shape in ((cos, "cos", None), (sin, "sin", None), (q_norm, "q_norm", (kv.head_dim,)),
                           (k_norm, "k_norm", (kv.head_dim,))):
        if t is None and shape:
            continue
        _need_cuda(t, name, torch.float32)
        if t.shape != shape if shape else t.dim() != 2 or t.shape != cos.shape or t.shape[1] * 2 != kv.head_dim:
            raise HyqError(-2, f"rope_append: shape of {name}")
    # every position of a sequence is below the table's reach, so max_new and
    # max_len (attention's bounds) are not needed here
    b = _batch(row_start, pos, slot, q.shape[0], 0, 0)
    opt = lambda t: C.c_void_p(None) if t is None else _ptr(t)  # noqa: E731
    check(lib.hyq_paged_rope_append(C.byref(kv), C.byref(b), _ptr(q), qs, q.shape[1], _ptr(k), ks, _ptr(v), vs,
                                    _ptr(cos), _ptr(sin), cos.shape[0], opt(q_norm), opt(k_norm), eps,
                                    1 if norm_first else 0, _ptr(out), os, _stream(q.device)))
    return out


def attention_workspace(heads, head_dim, device):
    """A zeroed workspace for attention() calls with these heads (any batch);
    calls that share one must not overlap in time."""
    n = C.c_size_t()
    check(lib.hyq_paged_attention_workspace_bytes(heads, head_dim, C.byref(n)))
    return torch.zeros(n.value, dtype=torch.uint8, device=device)


def attention(q, k_pages, v_pages, table, row_start, pos, max_new, max_len=None, slot=None, out=None, workspace=None):
    """hyq_paged_attention: causal grouped-query attention of the rotated
    queries q [tokens, heads, head_dim] over the pages, which hold the new
    tokens' keys and values already; [tokens, heads, head_dim] (into `out`
    when given).  max_new and max_len bound any sequence's new tokens and its
    length after them (max_len: the table's reach by default).  workspace:
    attention_workspace(...), made here when not given."""
    kv = _kv(k_pages, v_pages, table)
    qs = _heads(q, "q")
    out = torch.empty(q.shape, device=q.device) if out is None else out
    os = _heads(out, "out")
    if q.shape[2] != kv.head_dim or out.shape != q.shape:
        raise HyqError(-2, "attention: shapes of q and out")
    if max_len is None:
        max_len = kv.table_width * kv.page_size
    b = _batch(row_start, pos, slot, q.shape[0], max_new, max_len)
    if workspace is None:
        workspace = attention_workspace(q.shape[1], kv.head_dim, q.device)
    _need_cuda(workspace, "workspace", torch.uint8)
    need = C.c_size_t()
    check(lib.hyq_paged_attention_workspace_bytes(q.shape[1], kv.head_dim, C.byref(need)))
    if workspace.numel() < need.value:
        raise HyqError(-2, f"attention: the workspace takes {need.value} bytes")
    check(lib.hyq_paged_attention(C.byref(kv), C.byref(b), _ptr(q), qs, q.shape[1], _ptr(out), os, _ptr(workspace),
                                  _stream(q.device)))
    return out


class PagedCache:
    """Pages of every layer's keys and values, and the device tables that say
    which sequence holds which: `pool` [layers, 2, pages, kv_heads, page_size,
    head_dim] (layer(i) gives its keys and values), `table` [slots,
    table_width] (-1: unused), `length` [slots] and `refs` [pages].

    A slot is a sequence.  reserve() before each step makes room for its new
    tokens and returns the positions they start at; fork() shares a sequence's
    pages with another slot; free() gives them back; compact() moves the live
    pages to the front of the pool.  Nothing synchronises with the host:
    `shortage` holds the number of pages the last reserve or fork lacked (it
    then changed nothing, or left the forks empty)."""

    def __init__(self, layers, kv_heads, head_dim, pages, page_size, slots, table_width, device, dtype=torch.float16):
        z = lambda *n: torch.zeros(*n, dtype=torch.int32, device=device)  # noqa: E731
        self._init(torch.zeros(layers, 2, pages, kv_heads, page_size, head_dim, dtype=dtype, device=device),
                   z(slots, table_width) - 1, z(slots), z(pages))

    @classmethod
    def over(cls, pool, table, length, refs):
        """A cache over tensors the caller has (all contiguous, and consistent
        with each other)."""
        cache = cls.__new__(cls)
        cache._init(pool, table, length, refs)
        return cache

    def _init(self, pool, table, length, refs):
        if not isinstance(pool, torch.Tensor) or pool.dtype not in _KV_TYPES:
            raise HyqError(-1, "pool: expected a CUDA float32 or float16 tensor")
        _need_cuda(pool, "pool")
        for t, name in ((table, "table"), (length, "length"), (refs, "refs")):
            _need_cuda(t, name, torch.int32)
        if pool.dim() != 6 or pool.shape[1] != 2 or table.dim() != 2 or length.numel() != table.shape[0] \
                or refs.numel() != pool.shape[2]:
            raise HyqError(-2, "PagedCache: shapes of pool, table, length and refs")
        self.pool, self.table, self.length, self.refs = pool, table, length, refs
        self.page_size, self.pages, self.slots = pool.shape[4], pool.shape[2], table.shape[0]
        self.shortage = torch.zeros(1, dtype=torch.int32, device=pool.device)
        n = C.c_size_t()
        check(lib.hyq_pages_workspace_bytes(self.pages, C.byref(n)))
        self._ws = torch.empty(n.value, dtype=torch.uint8, device=pool.device)
        self._pages = _Pages(table.data_ptr(), length.data_ptr(), refs.data_ptr(), self.shortage.data_ptr(),
                             table.shape[0], table.shape[1], self.pages, self.page_size)
        page = pool[0, 0, 0].numel() * pool.element_size()
        self._pool = _Pool(pool.data_ptr(), 2 * pool.shape[0], page * self.pages, page, page)

    def layer(self, i):
        """(k_pages, v_pages) of a layer."""
        return self.pool[i, 0], self.pool[i, 1]

    def _slots(self, *arrays):
        for t in arrays:
            _need_cuda(t, "slots", torch.int32)
            if t.numel() != arrays[0].numel():
                raise HyqError(-2, "PagedCache: arrays of one call differ in length")
        return arrays[0].numel()

    def reserve(self, slot, extra, pos=None):
        """Grow sequence slot[i] by extra[i] positions; their first positions
        (int32, into `pos` when given)."""
        n = self._slots(slot, extra)
        pos = torch.empty(n, dtype=torch.int32, device=slot.device) if pos is None else pos
        self._slots(slot, pos)
        check(lib.hyq_pages_reserve(C.byref(self._pages), _ptr(slot), _ptr(extra), n, _ptr(pos), _ptr(self._ws),
                                    _stream(slot.device)))
        return pos

    def free(self, slot):
        """Give the sequences' pages back."""
        n = self._slots(slot)
        check(lib.hyq_pages_free(C.byref(self._pages), _ptr(slot), n, _stream(slot.device)))

    def fork(self, src, dst):
        """Sequence dst[i] becomes a copy of src[i]: full pages shared, the
        partial page copied in every layer."""
        n = self._slots(src, dst)
        check(lib.hyq_pages_fork(C.byref(self._pages), C.byref(self._pool), _ptr(src), _ptr(dst), n, _ptr(self._ws),
                                 _stream(src.device)))

    def compact(self):
        """Move the live pages to the front of the pool, in every layer."""
        check(lib.hyq_pages_compact(C.byref(self._pages), C.byref(self._pool), _ptr(self._ws),
                                    _stream(self.pool.device)))
