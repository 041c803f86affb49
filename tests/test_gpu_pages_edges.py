"""Refused page calls: what they return and what a step that goes on with it
does."""
import pytest

from test_gpu_paged import _int

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("slots,extra", [([0, 1, 2], [1, 1, 1]), ([0, 2, 0], [1, 1, 1]), ([0, 2, 4], [1, 1, 1]),
                                         ([0, -1, 2], [1, 1, 1]), ([0, 2, 3], [1, -1, 1])])
def test_refused_reserve_stops_the_step(cuda, slots, extra):
    """One sequence past its table row, repeated, out of range or shrinking:
    every position comes back -1, `shortage` says REFUSED, and an append and
    an attention at those positions leave the pages and the rows alone."""
    import torch
    from hy_mt_rs_b200 import paged, quant
    cache = paged.PagedCache(1, 2, 64, 16, 4, 4, 3, cuda)
    cache.reserve(_int([0, 1, 2], cuda), _int([5, 12, 3], cuda))
    cache.pool.normal_()
    pool, state = cache.pool.clone(), [t.clone() for t in (cache.table, cache.length, cache.refs)]
    kp, vp = cache.layer(0)
    cos = torch.ones(12, 32, device=cuda)
    q, k, v = (torch.randn(3, n, 64, device=cuda) for n in (4, 2, 2))
    pos = _int([2, 3, 1], cuda)         # what an earlier step left in this memory
    got = cache.reserve(_int(slots, cuda), _int(extra, cuda), pos=pos)
    assert got.tolist() == [-1, -1, -1] and cache.shortage.item() == paged.REFUSED
    slot, starts = _int(slots, cuda), _int([0, 1, 2, 3], cuda)
    out = torch.full_like(q, 7.0)
    paged.rope_append(q, k, v, kp, vp, cache.table, starts, pos, cos, cos, slot=slot, out=out)
    paged.attention(q, kp, vp, cache.table, starts, pos, 1, slot=slot, out=out)
    assert (out == 7).all() and torch.equal(cache.pool, pool)
    for a, b in zip(state, (cache.table, cache.length, cache.refs)):
        assert torch.equal(a, b)
    assert quant.device_status() == 8
    pos = cache.reserve(_int([0, 2, 3], cuda), _int([1, 1, 1], cuda))
    assert pos.tolist() == [5, 3, 0] and cache.shortage.item() == 0 and quant.device_status() == 0


def test_refused_fork_says_so(cuda):
    from hy_mt_rs_b200 import paged, quant
    cache = paged.PagedCache(1, 1, 8, 16, 4, 4, 3, cuda)
    cache.reserve(_int([0], cuda), _int([5], cuda))
    for src, dst in (([0], [0]), ([0, 0], [1, 1]), ([9], [2]), ([0], [4])):
        cache.fork(_int(src, cuda), _int(dst, cuda))
        assert cache.shortage.item() == paged.REFUSED and quant.device_status() == 8
    cache.fork(_int([0], cuda), _int([1], cuda))
    assert cache.shortage.item() == 0 and quant.device_status() == 0


def test_reserve_of_more_than_2_to_the_31_pages(cuda):
    """1,024 sequences that ask for 2^21 + 1 pages each: short, and nothing
    grows.  (The table is 8.6 GB, of which the call reads nothing.)"""
    import torch
    from hy_mt_rs_b200 import paged, quant
    width, pages = (1 << 21) + 1, 64
    z = lambda *n: torch.zeros(*n, dtype=torch.int32, device=cuda)  # noqa: E731
    table = torch.empty(1024, width, dtype=torch.int32, device=cuda)
    cache = paged.PagedCache.over(torch.zeros(1, 2, pages, 1, 1, 8, dtype=torch.float16, device=cuda), table, z(1024), z(pages))
    slot = torch.arange(1024, dtype=torch.int32, device=cuda)
    pos = cache.reserve(slot, torch.full_like(slot, width))
    assert (pos == 0).all() and cache.shortage.item() == paged.REFUSED - 1 - pages
    assert (cache.length == 0).all() and (cache.refs == 0).all()
    cache.reserve(slot[:3], torch.full_like(slot[:3], 21))
    assert cache.shortage.item() == 0 and cache.refs.sum().item() == 63
    assert table[:3, :21].flatten().tolist() == list(range(63))
    assert quant.device_status() == 0
