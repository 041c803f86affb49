"""Host checks of the paged-cache and sampling entry points: bad arguments are
refused with a negative code and a reason before any GPU work."""
import ctypes as C
import struct

import pytest

INVALID, SHAPE, ALIGN = -1, -2, -3
PTR = 0x10000     # never read: every call here is refused on the host, or has nothing to do


_KV = struct.Struct("PPiiiiqqqqPqq")     # hyq_paged_kv
_BATCH = struct.Struct("PPPqqqq")        # hyq_paged_batch


def _kv(**kw):
    d = dict(k=PTR, v=PTR, dtype=1, kv_heads=2, head_dim=128, page_size=16, pages=10, page_stride=2 * 16 * 128,
             head_stride=16 * 128, row_stride=128, table=PTR, slots=4, table_width=8)
    d.update(kw)
    return _KV.pack(*(v or 0 for v in d.values()))


def _batch(**kw):
    d = dict(slot=None, row_start=PTR, pos=PTR, seqs=2, tokens=3, max_new=2, max_len=100)
    d.update(kw)
    return _BATCH.pack(*(v or 0 for v in d.values()))


KV = [(dict(k=None), INVALID), (dict(v=None), INVALID), (dict(table=None), INVALID), (dict(dtype=2), INVALID),
      (dict(kv_heads=0), SHAPE), (dict(kv_heads=3), SHAPE), (dict(head_dim=0), SHAPE), (dict(head_dim=258), SHAPE),
      (dict(page_size=0), SHAPE), (dict(pages=0), SHAPE), (dict(pages=1 << 40), SHAPE), (dict(slots=0), SHAPE),
      (dict(slots=1), SHAPE), (dict(table_width=0), SHAPE), (dict(table_width=1 << 40), SHAPE), (dict(row_stride=64), SHAPE),
      (dict(head_stride=1), SHAPE), (dict(page_stride=0), SHAPE), (dict(k=PTR + 1), ALIGN), (dict(table=PTR + 2), ALIGN),
      (dict(dtype=0, v=PTR + 2), ALIGN)]
BATCH = [(dict(row_start=None), INVALID), (dict(pos=None), INVALID), (dict(seqs=-1), SHAPE), (dict(tokens=-1), SHAPE),
         (dict(tokens=1 << 33), SHAPE), (dict(max_new=-1), SHAPE), (dict(max_len=1), SHAPE), (dict(max_len=129), SHAPE),
         (dict(pos=PTR + 1), ALIGN), (dict(slot=PTR + 2), ALIGN)]


def _attention(kv, b, q=PTR, q_stride=512, heads=4, out=PTR, out_stride=512, ws=PTR):
    from hy_mt_rs_b200._native import lib
    return lib.hyq_paged_attention(kv, b, q, q_stride, heads, out, out_stride, ws, None)


def _append(kv, b, q=PTR, q_stride=512, heads=4, k=PTR, k_stride=256, v=PTR, v_stride=256, cos=PTR, sin=PTR, positions=64,
            out=PTR, out_stride=512):
    from hy_mt_rs_b200._native import lib
    return lib.hyq_paged_rope_append(kv, b, q, q_stride, heads, k, k_stride, v,
                                     v_stride, cos, sin, positions, None, None, 1e-5, 0, out, out_stride, None)


@pytest.mark.parametrize("call", [_attention, _append])
def test_cache_and_batch_checks(call):
    from hy_mt_rs_b200._native import last_error
    assert call(None, _batch()) == INVALID
    assert call(_kv(), None) == INVALID
    for kw, code in KV:
        assert call(_kv(**kw), _batch()) == code, kw
        assert "paged_" in last_error()
    for kw, code in BATCH:
        assert call(_kv(), _batch(**kw)) == code, kw
    assert call(_kv(), _batch(), heads=0) == SHAPE
    assert call(_kv(), _batch(), heads=5) == SHAPE
    assert call(_kv(), _batch(), heads=34) == SHAPE      # 17 query heads per kv head


def test_attention_workspace_bytes():
    from hy_mt_rs_b200._native import lib
    n = C.c_size_t()
    assert lib.hyq_paged_attention_workspace_bytes(16, 128, C.byref(n)) == 0 and n.value >= 16
    assert lib.hyq_paged_attention_workspace_bytes(16, 128, None) == INVALID
    assert lib.hyq_paged_attention_workspace_bytes(0, 128, C.byref(n)) == SHAPE
    assert lib.hyq_paged_attention_workspace_bytes(16, 257, C.byref(n)) == SHAPE


def _pages(**kw):
    from hy_mt_rs_b200.paged import _PAGES
    d = dict(table=PTR, length=PTR, refs=PTR, shortage=PTR, slots=4, table_width=8, pages=10, page_size=16)
    d.update(kw)
    return _PAGES.pack(*(v or 0 for v in d.values()))


def _pool(**kw):
    from hy_mt_rs_b200.paged import _POOL
    d = dict(base=PTR, planes=4, plane_stride=10 * 4096, page_stride=4096, page_bytes=4096)
    d.update(kw)
    return _POOL.pack(*(v or 0 for v in d.values()))


def test_pages_checks():
    from hy_mt_rs_b200._native import lib
    calls = [lambda p, n=1, a=PTR: lib.hyq_pages_reserve(p, a, PTR, n, None, PTR, None),
             lambda p, n=1, a=PTR: lib.hyq_pages_free(p, a, n, None),
             lambda p, n=1, a=PTR: lib.hyq_pages_fork(p, _pool(), a, PTR, n, PTR, None)]
    bad = [(dict(table=None), INVALID), (dict(length=None), INVALID), (dict(refs=None), INVALID), (dict(shortage=None), INVALID),
           (dict(slots=0), SHAPE), (dict(table_width=0), SHAPE), (dict(pages=0), SHAPE), (dict(page_size=0), SHAPE),
           (dict(table_width=1 << 31), SHAPE), (dict(pages=1 << 31), SHAPE), (dict(refs=PTR + 1), ALIGN)]
    for kw, code in bad:
        for call in calls:
            assert call(_pages(**kw)) == code, kw
        assert lib.hyq_pages_compact(_pages(**kw), _pool(), PTR, None) == code
    pool = [(dict(base=None), INVALID), (dict(planes=0), SHAPE), (dict(page_bytes=0), SHAPE), (dict(page_stride=16), SHAPE),
            (dict(plane_stride=16), SHAPE), (dict(base=PTR + 8), ALIGN), (dict(page_bytes=4088), ALIGN),
            (dict(plane_stride=40968), ALIGN)]
    # the status word needs a device: without one the table check already fails
    import torch
    if torch.cuda.is_available():
        for call in calls:
            assert call(_pages(), n=-1) == SHAPE
            assert call(_pages(), n=1025) == SHAPE
            assert call(_pages(), a=None) == INVALID
            assert call(_pages(), a=PTR + 2) == ALIGN
        for kw, code in pool:
            assert lib.hyq_pages_compact(_pages(), _pool(**kw), PTR, None) == code, kw
    n = C.c_size_t()
    assert lib.hyq_pages_workspace_bytes(10, C.byref(n)) == 0 and n.value >= 120
    assert lib.hyq_pages_workspace_bytes(0, C.byref(n)) == SHAPE
    assert lib.hyq_pages_workspace_bytes(10, None) == INVALID


def test_sample_checks():
    from hy_mt_rs_b200._native import last_error, lib

    def call(logits=PTR, n=100, stride=100, rows=2, u=PTR, token=PTR, k=None):
        return lib.hyq_sample(logits, n, stride, rows, None, k, None, None, u, token, None, None)

    assert call(logits=None) == INVALID and "sample" in last_error()
    assert call(u=None) == INVALID and call(token=None) == INVALID
    assert call(n=0) == SHAPE and call(n=1 << 23, stride=1 << 23) == SHAPE and call(stride=99) == SHAPE
    assert call(rows=-1) == SHAPE and call(rows=1 << 31) == SHAPE
    assert call(logits=PTR + 2) == ALIGN and call(k=PTR + 1) == ALIGN
    assert call(rows=0) == 0      # nothing to do


def test_python_entry_points_refuse():
    """Tensors of the wrong kind raise HyqError before any call."""
    import torch
    from hy_mt_rs_b200 import paged, sampling
    from hy_mt_rs_b200._native import HyqError

    cpu = torch.zeros(2, 4, 128)
    ints = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(HyqError):
        paged.attention(cpu, cpu, cpu, ints, ints, ints, 1, workspace=ints)
    with pytest.raises(HyqError):
        paged.attention(None, cpu, cpu, ints, ints, ints, 1)
    with pytest.raises(HyqError):
        paged.rope_append(cpu, cpu, cpu, cpu, cpu, ints, ints, ints, cpu, cpu)
    with pytest.raises(HyqError):
        sampling.sample(cpu[0], ints)
    with pytest.raises(HyqError):
        sampling.sample(None, None, 0.5)
    with pytest.raises(HyqError):
        paged.PagedCache.over(cpu, ints, ints, ints)
    with pytest.raises(TypeError):
        paged._ops.sample(cpu)
