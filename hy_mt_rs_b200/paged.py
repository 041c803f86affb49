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

from ._native import HyqError, check, lib, load_ops
from .quant import _need_cuda, _ptr

__all__ = ["PagedCache", "REFUSED", "rope_append", "attention", "attention_workspace"]

REFUSED = 2147483647    # HYQ_PAGES_REFUSED

_ops = load_ops()
_KV_TYPES = (torch.float32, torch.float16)
_PAGES = struct.Struct("PPPPqqqi4x")     # hyq_pages
_POOL = struct.Struct("Pqqqq")           # hyq_page_pool
_ZEROED = 4096                           # HYQ_PAGED_ATTENTION_ZEROED
_current_stream = torch._C._cuda_getCurrentRawStream


def rope_append(q, k, v, k_pages, v_pages, table, row_start, pos, cos, sin, q_norm=None, k_norm=None, eps=1e-5,
                norm_first=False, slot=None, out=None):
    """hyq_paged_rope_append: rotate and normalise the heads of q [tokens,
    heads, head_dim] and k [tokens, kv_heads, head_dim] at their positions,
    write k and v into the pages, return the rotated queries (into `out` when
    given; q itself is allowed).  cos and sin are [positions, head_dim / 2]
    (hyq_rope_table); norm_first normalises before the rotation."""
    return _ops.rope_append(q, k, v, k_pages, v_pages, table, row_start, pos, cos, sin, q_norm, k_norm, eps, norm_first,
                            slot, out)


@functools.lru_cache(maxsize=None)
def _workspace_bytes(heads, head_dim):
    n = C.c_size_t()
    check(lib.hyq_paged_attention_workspace_bytes(heads, head_dim, C.byref(n)))
    return n.value


def attention_workspace(heads, head_dim, device):
    """A workspace for attention() calls with these heads (any batch), zero where
    the calls need it; calls that share one must not overlap in time."""
    workspace = torch.empty(_workspace_bytes(heads, head_dim), dtype=torch.uint8, device=device)
    workspace[:_ZEROED].zero_()
    return workspace


def attention(q, k_pages, v_pages, table, row_start, pos, max_new, max_len=None, slot=None, out=None, workspace=None):
    """hyq_paged_attention: causal grouped-query attention of the rotated
    queries q [tokens, heads, head_dim] over the pages, which hold the new
    tokens' keys and values already; [tokens, heads, head_dim] (into `out`
    when given).  max_new and max_len bound any sequence's new tokens and its
    length after them (max_len: the table's reach by default).  workspace:
    attention_workspace(...), made here when not given."""
    if workspace is None:
        if not isinstance(q, torch.Tensor) or q.dim() != 3:
            raise HyqError(-2, "q: expected [tokens, heads, head_dim] with contiguous heads")
        workspace = attention_workspace(q.shape[1], q.shape[2], q.device)
    return _ops.attention(q, k_pages, v_pages, table, row_start, pos, max_new, -1 if max_len is None else max_len, slot,
                          out, workspace)


def _check_int(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.int32 or not t.is_contiguous():
        _need_cuda(t, name, torch.int32)


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
    then changed nothing, or left the forks empty), or REFUSED after one with a
    slot that is repeated or out of range, or that would pass its table row
    (nothing changed; a reserve's positions are -1, which rope_append and
    attention skip).  `changes` counts the calls that changed lengths."""

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
            self._same_device(t, pool, name)
        if pool.dim() != 6 or pool.shape[1] != 2 or table.dim() != 2 or length.numel() != table.shape[0] \
                or refs.numel() != pool.shape[2]:
            raise HyqError(-2, "PagedCache: shapes of pool, table, length and refs")
        self.pool, self.table, self.length, self.refs = pool, table, length, refs
        self.page_size, self.pages, self.slots = pool.shape[4], pool.shape[2], table.shape[0]
        self.changes = 0
        self.shortage = torch.zeros(1, dtype=torch.int32, device=pool.device)
        n = C.c_size_t()
        check(lib.hyq_pages_workspace_bytes(self.pages, C.byref(n)))
        self._ws = torch.empty(n.value, dtype=torch.uint8, device=pool.device)
        self._pages = _PAGES.pack(table.data_ptr(), length.data_ptr(), refs.data_ptr(), self.shortage.data_ptr(),
                                  table.shape[0], table.shape[1], self.pages, self.page_size)
        page = pool[0, 0, 0].numel() * pool.element_size()
        self._pool = _POOL.pack(pool.data_ptr(), 2 * pool.shape[0], page * self.pages, page, page)

    @staticmethod
    def _same_device(t, like, name):
        if t.device != like.device:
            raise HyqError(-1, f"{name}: on another device")

    def layer(self, i):
        """(k_pages, v_pages) of a layer."""
        return self.pool[i, 0], self.pool[i, 1]

    def _slots(self, *arrays):
        n = arrays[0].numel() if isinstance(arrays[0], torch.Tensor) else 0
        for t in arrays:
            _check_int(t, "slots")
            self._same_device(t, self.pool, "slots")
            if t.numel() != n:
                raise HyqError(-2, "PagedCache: arrays of one call differ in length")
        return n

    def reserve(self, slot, extra, pos=None):
        """Grow sequence slot[i] by extra[i] positions; their first positions
        (int32, into `pos` when given)."""
        n = self._slots(slot, extra)
        if pos is None:
            pos = torch.empty(slot.shape, dtype=torch.int32, device=slot.device)
        self._slots(slot, pos)
        self.changes += 1
        check(lib.hyq_pages_reserve(self._pages, slot.data_ptr(), extra.data_ptr(), n, pos.data_ptr(), _ptr(self._ws),
                                    _current_stream(slot.get_device())))
        return pos

    def free(self, slot):
        """Give the sequences' pages back."""
        n = self._slots(slot)
        self.changes += 1
        check(lib.hyq_pages_free(self._pages, slot.data_ptr(), n, _current_stream(slot.get_device())))

    def fork(self, src, dst):
        """Sequence dst[i] becomes a copy of src[i]: full pages shared, the
        partial page copied in every layer."""
        n = self._slots(src, dst)
        self.changes += 1
        check(lib.hyq_pages_fork(self._pages, self._pool, src.data_ptr(), dst.data_ptr(), n, _ptr(self._ws),
                                 _current_stream(src.get_device())))

    def compact(self):
        """Move the live pages to the front of the pool, in every layer."""
        check(lib.hyq_pages_compact(self._pages, self._pool, _ptr(self._ws), _current_stream(self.pool.get_device())))
