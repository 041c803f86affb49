"""GPU parity of paged.attention_shared (groups of sequences with a prefix in
common) with a 64-bit softmax over each sequence's whole table row, for every
cache type."""
import math
import random

import pytest

from test_gpu_paged import _int, _reference
from test_gpu_paged import _close as _close_plain
from test_gpu_paged8 import _close as _close_coded
from test_gpu_paged8 import _quantise, _values

pytestmark = pytest.mark.gpu

KINDS = ["f32", "f16", "i8", "f8"]


def _make(dev, groups, heads, kvh, dim, page, kind, seed=0, own_pages=(), layout="hnd"):
    """groups: [(prefix, [(positions behind it, new tokens), ..]), ..].  Full pages of
    a prefix are shared (own_pages: copies in pages of their own, for those
    sequences), the partial one is copied."""
    import torch
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    seqs = [(p, behind, new, i) for i, (p, members) in enumerate(groups) for behind, new in members]
    counts = [-(-(p + behind + new) // page) for p, behind, new, _ in seqs]
    pages = sum(counts) + 5
    # a table so wide that the call's bound on the prefixes makes them worth their own kernels
    row = 2 * kvh * {"f32": 4 * dim, "f16": 2 * dim}.get(kind, dim + 4)
    width = max(max(counts) + 1, -(-150000000 // (max(1, len(seqs) - len(groups)) * row * page)) + 1)
    held = list(range(pages))
    rng.shuffle(held)
    shape = (pages, kvh, page, dim) if layout == "hnd" else (pages, page, kvh, dim)
    pools = [torch.randn(*shape, generator=g, device=dev) for _ in range(2)]
    if layout != "hnd":
        pools = [x.permute(0, 2, 1, 3) for x in pools]
    table = torch.full((len(seqs), width), -1, dtype=torch.int32)
    at, first = 0, {}
    for s, ((p, behind, new, i), c) in enumerate(zip(seqs, counts)):
        mine = held[at:at + c]
        at += c
        if i in first:
            parent = table[first[i]].tolist()
            for j in range(-(-p // page)):
                if j < p // page and s not in own_pages:
                    mine[j] = parent[j]
                else:
                    for x in pools:
                        x[mine[j], :, :min(page, p - j * page)] = x[parent[j], :, :min(page, p - j * page)]
        else:
            first[i] = s
        table[s, :c] = torch.tensor(mine, dtype=torch.int32)
    new = [n for _, _, n, _ in seqs]
    ctx = [p + behind for p, behind, _, _ in seqs]
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    q = torch.randn(max(1, starts[-1]), heads, dim, generator=g, device=dev)[:starts[-1]]
    q = q * (1 + torch.arange(heads, device=dev) % 3)[:, None]
    counts = [len(m) for _, m in groups]
    s = dict(q=q, table=table.to(dev), row_start=_int(starts, dev), pos=_int(ctx, dev), new=new, ctx=ctx, starts=starts, page=page,
             slots=list(range(len(new))), slot=None, kv={}, kind=kind, group_start=_int([sum(counts[:i]) for i in range(len(counts) + 1)], dev),
             shared=_int([p for p, _ in groups], dev))
    for name, x in zip(("k", "v"), pools):
        if kind in ("i8", "f8"):
            codes, scale = (t.to(dev) for t in _quantise(x, kind))
            s[name + "_pages"], s["kv"][name + "_scale"], s[name] = codes, scale, _values(codes, scale)
        else:
            s[name] = s[name + "_pages"] = x.half() if kind == "f16" else x
    return s


def _attend(s, **kw):
    from hy_mt_rs_b200 import paged
    return paged.attention_shared(s["q"], s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos"], s["group_start"],
                                  s["shared"], max(s["new"] + [1]), **{"slot": s["slot"], **s["kv"], **kw})


def _close(got, s):
    (_close_coded if s["kv"] else _close_plain)(got, s)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,dim", [(16, 4, 128), (32, 8, 128), (16, 2, 128), (8, 8, 64), (12, 4, 64), (16, 1, 128), (6, 2, 80),
                                           (4, 2, 256)])
def test_shapes(cuda, heads, kvh, dim, kind):
    """Prefixes at and around the ends of pages and tiles; a group of one, an empty
    group, prefixes of nothing and of one position."""
    few = 16 * kvh // heads
    s = _make(cuda, [(300, [(0, 1), (17, min(2, few)), (130, 1)]), (128, [(5, 1)]), (77, []), (0, [(40, 1), (3, 1)]),
                     (1, [(0, 1), (0, 1)]), (640, [(64 * i, 1) for i in range(9)])], heads, kvh, dim, 32, kind, seed=dim + heads)
    _close(_attend(s), s)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [1, 7, 16, 48, 64, 100, 128, 256])
def test_page_sizes(cuda, page, kind):
    s = _make(cuda, [(515, [(i, 1) for i in range(6)]), (257, [(3, 3), (90, 1)])], 8, 2, 128, page, kind, seed=page)
    _close(_attend(s), s)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("prefix", [15, 127, 128, 129, 1000, 6000])
@pytest.mark.parametrize("per", [2, 33, 70])
def test_many_sequences_long_prefixes(cuda, per, prefix, kind):
    """Rows of one to three row tiles; prefixes cut over many CTAs."""
    s = _make(cuda, [(prefix, [((i * 37) % 200, 1) for i in range(per)])], 16, 4, 128, 64, kind, seed=per + prefix)
    _close(_attend(s), s)


@pytest.mark.parametrize("kind", KINDS)
def test_layout_slots_copies_outputs(cuda, kind):
    """Permuted pages, slots in another order, a sequence with copies of the prefix's
    pages, an output with a stride, rows behind the last sequence left alone; the
    call is reproducible, and attention() agrees."""
    import torch
    from hy_mt_rs_b200 import paged
    s = _make(cuda, [(200, [(9, 1), (0, 2), (50, 1)]), (333, [(1, 1), (70, 4)])], 16, 4, 128, 16, kind, seed=3, own_pages=(2,),
              layout="hnd" if kind in ("i8", "f8") else "nhd")
    order = [3, 0, 4, 1, 2]
    table = torch.empty_like(s["table"])
    table[order] = s["table"]
    s.update(table=table, slot=_int(order, cuda), slots=order)
    t = s["q"].shape[0]
    wide = torch.full((t + 3, 20, 128), 5.0, device=cuda)
    s["q"] = torch.cat([s["q"], torch.ones(3, 16, 128, device=cuda)])
    got = _attend(s, out=wide[:, :16])
    assert (wide[t:] == 5).all() and (wide[:, 16:] == 5).all()
    again = _attend(s)
    s["q"] = s["q"][:t]
    assert torch.equal(again[:t], got[:t])
    _close(got[:t], s)
    plain = paged.attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos"], 4, slot=s["slot"], **s["kv"])
    _close(plain, s)


@pytest.mark.parametrize("kind", KINDS)
def test_small_prefixes_are_attention(cuda, kind):
    """A call whose prefixes are not worth it gives attention()'s bits."""
    import torch
    from hy_mt_rs_b200 import paged
    s = _make(cuda, [(200, [(9, 1), (0, 2), (50, 1)]), (333, [(1, 1), (70, 4)])], 16, 4, 128, 16, kind, seed=3)
    plain = paged.attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos"], 4, 500, **s["kv"])
    assert torch.equal(_attend(s, max_len=500, max_shared=333), plain)
    assert not torch.equal(_attend(s), plain)     # the other tests' way


@pytest.mark.parametrize("kind", KINDS)
def test_bad_groups_are_taken_alone(cuda, kind):
    """A prefix longer than what a sequence holds, starts that do not ascend or
    pass the batch: the same outputs without the prefix, and the device status."""
    from hy_mt_rs_b200 import quant
    groups = [(140, [(9, 1), (0, 1), (50, 1)]), (200, [(1, 1), (70, 2)])]
    for shared, start in (([141, 200], [0, 3, 5]), ([-1, 200], [0, 3, 5]), ([140, 200], [0, 3, 6]), ([140, 200], [0, 6, 5]),
                          ([140, 200], [-1, 3, 5]), ([140, 2 ** 31 - 1], [0, 3, 5])):
        s = _make(cuda, groups, 8, 2, 128, 32, kind, seed=4)
        s.update(shared=_int(shared, cuda), group_start=_int(start, cuda))
        got = _attend(s)
        assert quant.device_status() != 0
        _close(got, s)
    # sequences outside the groups, and no groups at all
    s = _make(cuda, groups, 8, 2, 128, 32, kind, seed=5)
    s.update(shared=_int([140], cuda), group_start=_int([0, 2], cuda))
    _close(_attend(s), s)
    s.update(shared=_int([200], cuda), group_start=_int([3, 5], cuda))
    _close(_attend(s), s)
    s.update(shared=_int([], cuda), group_start=_int([0], cuda))
    _close(_attend(s), s)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_values_that_are_not_finite(cuda, kind):
    """An infinity of the prefix is the output of all its group, one behind it of
    its own sequence; both signs make NaN; a NaN key makes its rows NaN; others
    stay within their bound (not the same bits: the f32 kernel takes tiles with such
    values another way).  Garbage past the sequences does not count."""
    import torch
    s = _make(cuda, [(150, [(9, 1), (0, 2), (50, 1)]), (140, [(1, 1), (70, 1)])], 8, 2, 128, 32, kind, seed=6)
    used = torch.zeros(s["k"].shape[0], 32, dtype=torch.bool)
    for i, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        for p in range(n + c):
            used[int(s["table"][i, p // 32]), p % 32] = True
    want = _attend(s)
    ref, tol = _reference(s)

    def near(got, where):
        return bool(((got.double() - ref).abs() <= tol)[where].all())

    free = ~used.to(cuda)[:, None, :, None].expand(s["k"].shape)
    s["k"][free] = math.nan
    s["v"][free] = math.inf
    assert torch.equal(_attend(s), want)
    s["v"][int(s["table"][0, 2]), 0, 5, 7] = math.inf        # position 69 of the first group's prefix
    s["v"][int(s["table"][2, 6]), 1, 3, 9] = -math.inf       # position 195 of sequence 2 (one of the first group)
    got = _attend(s)
    spoiled = torch.zeros_like(got, dtype=torch.bool)
    spoiled[:4, :4, 7] = True
    assert (got[spoiled] == math.inf).all()
    spoiled[3, 4:, 9] = True
    assert (got[3, 4:, 9] == -math.inf).all()
    assert near(got, ~spoiled)
    s["v"][int(s["table"][2, 6]), 0, 3, 7] = -math.inf       # meets the prefix's
    got = _attend(s)
    assert torch.isnan(got[3, :4, 7]).all() and (got[:3, :4, 7] == math.inf).all()
    s["k"][int(s["table"][3, 1]), 1, 4, 0] = math.nan        # the second group's prefix
    got = _attend(s)
    assert torch.isnan(got[4:, 4:]).all() and near(got, (slice(4, None), slice(0, 4))) and not torch.isnan(got[:3]).any()


@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_captured_and_replayed(cuda, kind):
    import torch
    from hy_mt_rs_b200 import paged
    s = _make(cuda, [(300, [(9, 1), (0, 1), (50, 1)]), (129, [(1, 1), (70, 1)])], 16, 4, 128, 32, kind, seed=8)
    out = torch.empty_like(s["q"])
    ws = paged.attention_shared_workspace(16, 128, 5, cuda)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        _attend(s, out=out, workspace=ws)
        with torch.cuda.graph(graph, stream=stream):
            _attend(s, out=out, workspace=ws)
    torch.cuda.current_stream().wait_stream(stream)
    for shared, ctx in (([300, 129], s["ctx"]), ([128, 0], [301, 300, 349, 130, 198]), ([0, 64], [30, 300, 349, 64, 100])):
        s["q"].normal_()
        s["ctx"] = ctx
        s["pos"].copy_(_int(ctx, cuda))
        s["shared"].copy_(_int(shared, cuda))
        out.zero_()
        graph.replay()
        _close(out, s)
