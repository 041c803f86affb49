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
import functools
import struct

import torch

from ._native import HyqError, check, lib
from .quant import _need_cuda, _ptr

__all__ = ["PagedCache", "rope_append", "attention", "attention_workspace"]

_KV_TYPES = {torch.float32: 0, torch.float16: 1}   # HYQ_KV_F32, HYQ_KV_F16

# The structures of include/hyq.h as packed bytes (a call at a decode step's
# sizes takes a few microseconds on the device: the host side counts).
_KV = struct.Struct("PPiiiiqqqqPqq")     # hyq_paged_kv
_BATCH = struct.Struct("PPPqqqq")        # hyq_paged_batch
_PAGES = struct.Struct("PPPPqqqi4x")     # hyq_pages
_POOL = struct.Struct("Pqqqq")           # hyq_page_pool

_current_stream = torch._C._cuda_getCurrentRawStream


def _check_int(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.int32 or not t.is_contiguous():
        _need_cuda(t, name, torch.int32)


def _check_f32(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.float32 or not t.is_contiguous():
        _need_cuda(t, name, torch.float32)


def _kv(k_pages, v_pages, table):
    """hyq_paged_kv of a layer's pages; (packed, kv_heads, page_size, head_dim, table_width)."""
    for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _KV_TYPES:
            raise HyqError(-1, f"{name}: expected a CUDA float32 or float16 tensor")
    shape, strides, dtype = k_pages.shape, k_pages.stride(), k_pages.dtype
    if len(shape) != 4 or strides[3] != 1:
        raise HyqError(-2, "k_pages: expected [pages, kv_heads, page_size, head_dim], contiguous in head_dim")
    if shape != v_pages.shape or strides != v_pages.stride() or dtype != v_pages.dtype:
        raise HyqError(-2, "k_pages and v_pages differ in shape, strides or type")
    _check_int(table, "table")
    rows = table.shape
    if len(rows) != 2:
        raise HyqError(-2, "table: expected [slots, table_width]")
    pages, heads, page, dim = shape
    return (_KV.pack(k_pages.data_ptr(), v_pages.data_ptr(), _KV_TYPES[dtype], heads, dim, page, pages, strides[0],
                     strides[1], strides[2], table.data_ptr(), rows[0], rows[1]), heads, page, dim, rows[1])


def _batch(row_start, pos, slot, tokens, max_new, max_len):
    _check_int(row_start, "row_start")
    _check_int(pos, "pos")
    seqs = pos.numel()
    if row_start.numel() != seqs + 1:
        raise HyqError(-2, "row_start takes one more entry than pos")
    if slot is not None:
        _check_int(slot, "slot")
        if slot.numel() != seqs:
            raise HyqError(-2, "slot takes one entry per sequence")
    if max_new < 0 or max_len < 0:
        raise HyqError(-2, "max_new and max_len are not negative")
    return _BATCH.pack(0 if slot is None else slot.data_ptr(), row_start.data_ptr(), pos.data_ptr(), seqs, tokens,
                       max_new, max_len)


def _heads(t, name):
    """Shape and row stride of [tokens, heads, head_dim] float32 activations
    whose heads are contiguous."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.float32:
        raise HyqError(-1, f"{name}: expected a CUDA float32 tensor")
    shape, strides = t.shape, t.stride()
    if len(shape) != 3 or strides[2] != 1 or (strides[1] != shape[2] and shape[1] > 1):
        raise HyqError(-2, f"{name}: expected [tokens, heads, head_dim] with contiguous heads")
    return shape, (strides[0] if shape[0] > 1 else shape[1] * shape[2])


def rope_append(q, k, v, k_pages, v_pages, table, row_start, pos, cos, sin, q_norm=None, k_norm=None, eps=1e-5,
                norm_first=False, slot=None, out=None):
    """hyq_paged_rope_append: rotate and normalise the heads of q [tokens,
    heads, head_dim] and k [tokens, kv_heads, head_dim] at their positions,
    write k and v into the pages, return the rotated queries (into `out` when
    given; q itself is allowed).  cos and sin are [positions, head_dim / 2]
    (hyq_rope_table); norm_first normalises before the rotation."""
    kv, kv_heads, _, dim, _ = _kv(k_pages, v_pages, table)
    (shape, qs), (k_shape, ks), (v_shape, vs) = _heads(q, "q"), _heads(k, "k"), _heads(v, "v")
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=q.device)
    out_shape, os = _heads(out, "out")
    if shape[2] != dim or out_shape != shape or k_shape != (shape[0], kv_heads, dim) or v_shape != k_shape:
        raise HyqError(-2, "rope_append: shapes of q, k, v and out")
    _check_f32(cos, "cos")
    _check_f32(sin, "sin")
    rows = cos.shape
    if len(rows) != 2 or rows != sin.shape or rows[1] * 2 != dim:
        raise HyqError(-2, "rope_append: cos and sin are [positions, head_dim / 2]")
    for w, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if w is not None:
            _check_f32(w, name)
            if w.shape != (dim,):
                raise HyqError(-2, f"rope_append: shape of {name}")
    # (positions are checked against the table's reach on the device; max_new
    # and max_len bound attention's work only)
    batch = _batch(row_start, pos, slot, shape[0], 0, 0)
    check(lib.hyq_paged_rope_append(kv, batch, q.data_ptr(), qs, shape[1], k.data_ptr(), ks, v.data_ptr(), vs,
                                    cos.data_ptr(), sin.data_ptr(), rows[0], None if q_norm is None else q_norm.data_ptr(),
                                    None if k_norm is None else k_norm.data_ptr(), eps, 1 if norm_first else 0,
                                    out.data_ptr(), os, _current_stream(q.get_device())))
    return out


@functools.lru_cache(maxsize=None)
def _workspace_bytes(heads, head_dim):
    n = C.c_size_t()
    check(lib.hyq_paged_attention_workspace_bytes(heads, head_dim, C.byref(n)))
    return n.value


def attention_workspace(heads, head_dim, device):
    """A zeroed workspace for attention() calls with these heads (any batch);
    calls that share one must not overlap in time."""
    return torch.zeros(_workspace_bytes(heads, head_dim), dtype=torch.uint8, device=device)


def attention(q, k_pages, v_pages, table, row_start, pos, max_new, max_len=None, slot=None, out=None, workspace=None):
    """hyq_paged_attention: causal grouped-query attention of the rotated
    queries q [tokens, heads, head_dim] over the pages, which hold the new
    tokens' keys and values already; [tokens, heads, head_dim] (into `out`
    when given).  max_new and max_len bound any sequence's new tokens and its
    length after them (max_len: the table's reach by default).  workspace:
    attention_workspace(...), made here when not given."""
    kv, _, page, dim, width = _kv(k_pages, v_pages, table)
    shape, qs = _heads(q, "q")
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=q.device)
    out_shape, os = _heads(out, "out")
    if shape[2] != dim or out_shape != shape:
        raise HyqError(-2, "attention: shapes of q and out")
    batch = _batch(row_start, pos, slot, shape[0], max_new, width * page if max_len is None else max_len)
    if workspace is None:
        workspace = attention_workspace(shape[1], dim, q.device)
    elif not isinstance(workspace, torch.Tensor) or not workspace.is_cuda or workspace.dtype != torch.uint8 \
            or not workspace.is_contiguous():
        _need_cuda(workspace, "workspace", torch.uint8)
    if workspace.numel() < _workspace_bytes(shape[1], dim):
        raise HyqError(-2, f"attention: the workspace takes {_workspace_bytes(shape[1], dim)} bytes")
    check(lib.hyq_paged_attention(kv, batch, q.data_ptr(), qs, shape[1], out.data_ptr(), os, workspace.data_ptr(),
                                  _current_stream(q.get_device())))
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
        self._pages = _PAGES.pack(table.data_ptr(), length.data_ptr(), refs.data_ptr(), self.shortage.data_ptr(),
                                  table.shape[0], table.shape[1], self.pages, self.page_size)
        page = pool[0, 0, 0].numel() * pool.element_size()
        self._pool = _POOL.pack(pool.data_ptr(), 2 * pool.shape[0], page * self.pages, page, page)

    def layer(self, i):
        """(k_pages, v_pages) of a layer."""
        return self.pool[i, 0], self.pool[i, 1]

    def _slots(self, *arrays):
        n = arrays[0].numel() if isinstance(arrays[0], torch.Tensor) else 0
        for t in arrays:
            _check_int(t, "slots")
            if t.numel() != n:
                raise HyqError(-2, "PagedCache: arrays of one call differ in length")
        return n

    def reserve(self, slot, extra, pos=None):
        """Grow sequence slot[i] by extra[i] positions; their first positions
        (int32, into `pos` when given)."""
        if pos is None:
            pos = torch.empty(slot.shape, dtype=torch.int32, device=slot.device)
        n = self._slots(slot, extra, pos)
        check(lib.hyq_pages_reserve(self._pages, slot.data_ptr(), extra.data_ptr(), n, pos.data_ptr(), _ptr(self._ws),
                                    _current_stream(slot.get_device())))
        return pos

    def free(self, slot):
        """Give the sequences' pages back."""
        n = self._slots(slot)
        check(lib.hyq_pages_free(self._pages, slot.data_ptr(), n, _current_stream(slot.get_device())))

    def fork(self, src, dst):
        """Sequence dst[i] becomes a copy of src[i]: full pages shared, the
        partial page copied in every layer."""
        n = self._slots(src, dst)
        check(lib.hyq_pages_fork(self._pages, self._pool, src.data_ptr(), dst.data_ptr(), n, _ptr(self._ws),
                                 _current_stream(src.get_device())))

    def compact(self):
        """Move the live pages to the front of the pool, in every layer."""
        check(lib.hyq_pages_compact(self._pages, self._pool, _ptr(self._ws), _current_stream(self.pool.get_device())))
