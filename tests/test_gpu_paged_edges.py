"""Paged attention at its edges, each case with the kernel that it must reach:
infinities in cached values, scores of any size, keys that are NaN, values that
a row does not see in every kernel, bad page entries, graph capture."""
import math

import pytest

from test_gpu_paged import _attend, _int, _make

pytestmark = pytest.mark.gpu

# new tokens, context and page size that lead to each kernel, with 8 query and 2
# kv heads, max_len the longest sequence: (kernel, f16 cache, new, ctx, page, dim)
FEW = [("few_kernel", True, [1, 3], [700, 90], 32, 128), ("few_kernel", True, [4], [5000], 64, 64),
       ("few_kernel", False, [1, 3], [700, 90], 32, 128), ("few_kernel", False, [2], [3000], 16, 64)]
CHUNK = [("chunk_kernel", True, [40, 1], [200, 90], 32, 128), ("chunk_kernel", True, [150], [500], 48, 64),
         ("chunk_kernel", False, [40], [20], 32, 128)]
TC = [("chunk_tc_kernel", True, [200, 2], [500, 70], 32, 128), ("chunk_tc_kernel", True, [300], [1900], 128, 64),
      ("chunk_tc_kernel", True, [64] * 40, [400] * 40, 16, 64)]
TC32 = [("chunk_tc32_kernel", False, [200, 2], [500, 70], 32, 128), ("chunk_tc32_kernel", False, [130], [1900], 48, 64),
        ("chunk_tc32_kernel", False, [32] * 40, [400] * 40, 16, 64)]
OTHER = [("attend_kernel", True, [5, 1], [200, 90], 16, 80), ("attend_kernel", False, [3], [300], 7, 128 + 32)]
ALL = FEW + CHUNK + TC + TC32 + OTHER


def _ids(case):
    return f"{case[0]}-{'f16' if case[1] else 'f32'}-{case[2][0]}x{len(case[2])}at{case[3][0]}-p{case[4]}-d{case[5]}"


def _case(dev, case, **kw):
    _, kv16, new, ctx, page, dim = case
    return _make(dev, new, ctx, 8, 2, dim, page, kv16, seed=dim + sum(ctx), **kw)


def _run(case, s, reaches=True, **kw):
    """The call's output; `reaches`: the kernel that the case is for must be
    among those that ran."""
    import torch
    from torch.profiler import ProfilerActivity, profile
    length = max(n + c for n, c in zip(s["new"], s["ctx"]))
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        out = _attend(s, max_len=length, **kw)
        torch.cuda.synchronize()
    names = [e.name for e in p.events()]
    if reaches:
        assert any(case[0] + "<" in n for n in names), names
    return out


def _at(s, i, p):
    """Page and row of position p of sequence i."""
    return int(s["table"][s["slots"][i], p // s["page"]]), p % s["page"]


def _exact(s, drop=()):
    """The output in 64 bits, without the positions in `drop`, and the bound of
    test_gpu_paged._reference: products to 21 bits and sums in f32 put a score
    off by at most (2^-21 + dim 2^-24) sum|q k| / sqrt(dim), which counts twice
    in a weight; 2^-18 for the roundings of weights and sums.  Queries are kept
    to 2^-25 of their row's largest value at least: that times sum|k| on top."""
    import torch
    q = s["q"].double()
    heads, dim = q.shape[1:]
    group = heads // s["k"].shape[1]
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for i, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        a = s["starts"][i]
        held = s["table"][s["slots"][i], :-(-(n + c) // s["page"])].long()
        kept = torch.tensor([p for p in range(n + c) if p not in set(drop)], device=q.device)
        hide = kept[None] > torch.arange(c, n + c, device=q.device)[:, None]
        for h in range(heads):
            k = s["k"][held, h // group].double().reshape(-1, dim)[kept]
            v = s["v"][held, h // group].double().reshape(-1, dim)[kept]
            x = q[a:a + n, h] @ k.T / math.sqrt(dim)
            p = torch.softmax(x.masked_fill(hide, -math.inf), -1)
            rows = q[a:a + n, h].abs()
            off = (2.0 ** -21 + dim * 2.0 ** -24) * (rows @ k.abs().T) + 2.0 ** -25 * rows.amax(-1, keepdim=True) * k.abs().sum(-1)
            off = (off / math.sqrt(dim)).masked_fill(hide, 0).amax(-1, keepdim=True)
            out[a:a + n, h] = p @ v
            tol[a:a + n, h] = (p @ v.abs()) * (2 * off + 2.0 ** -18)
    return out, tol


def _within(got, ref, tol):
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), float((err / tol.clamp(min=1e-30)).max())


# ---------------------------------------------------------------- values
@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("case", TC32, ids=_ids)
def test_f32_tiles_left_out_of_the_products(cuda, case, bad):
    """A tile of an f32 cache with a value that is not finite is gone through
    position by position, in a time of its own for each warp: that value is its
    column's output, every other one is right, call after call."""
    s = _case(cuda, case)
    ref, tol = _exact(s)
    for i, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        if n > 4:
            for p in (0, c // 2):
                page, row = _at(s, i, p)
                s["v"][page, :, row, 3] = bad
    chunked = [r for n, a in zip(s["new"], s["starts"]) if n > 4 for r in range(a, a + n)]
    for _ in range(10):
        got = _run(case, s)
        col = got[chunked, :, 3]
        assert (col.isnan() if math.isnan(bad) else col == bad).all()
        got[chunked, :, 3] = ref[chunked, :, 3].float()
        _within(got, ref, tol)


@pytest.mark.parametrize("case", ALL, ids=_ids)
def test_infinities_in_cached_values(cuda, case):
    """Every weight is above zero, so an infinity in a value that a token sees
    is its output, two of different sign and a NaN are NaN; other columns and
    other kv heads are as without."""
    from hy_mt_rs_b200 import quant
    s = _case(cuda, case)
    ref, tol = _exact(s)
    put = [(0, 3, math.inf), (0, 5, -math.inf), (1, 6, math.inf), (9, 6, -math.inf), (11, 8, math.nan)]
    for i, c in enumerate(s["ctx"]):
        for p, d, x in put:
            page, row = _at(s, i, p)
            s["v"][page, 1, row, d] = x
    got = _run(case, s)
    rows = got[:, 4:]       # the query heads of kv head 1
    assert (rows[..., 3] == math.inf).all() and (rows[..., 5] == -math.inf).all()
    assert rows[..., 6].isnan().all() and rows[..., 8].isnan().all()
    for d in (3, 5, 6, 8):
        rows[..., d] = ref[:, 4:, d].float()
    _within(got, ref, tol)
    assert quant.device_status() == 0


@pytest.mark.parametrize("case", ALL, ids=_ids)
def test_nan_keys_outweigh_infinite_values(cuda, case):
    """NaN scores make a row NaN, also where its values hold an infinity and
    where whole blocks of positions are NaN."""
    for n in (1, 64, 130):
        s = _case(cuda, case)
        for i, c in enumerate(s["ctx"]):
            page, row = _at(s, i, 0)
            s["v"][page, :, row, 3] = math.inf
            for p in range(min(n, c)):
                page, row = _at(s, i, p)
                s["k"][page, :, row, 1] = math.nan
        assert _run(case, s).isnan().all()


LATER = [("few_kernel", True, [4], [600], 32, 128), ("few_kernel", False, [3], [1500], 32, 64),
         ("chunk_kernel", True, [100], [100], 32, 128), ("chunk_kernel", False, [50], [10], 16, 64),
         ("chunk_tc_kernel", True, [200], [500], 32, 128), ("chunk_tc_kernel", True, [200], [3000], 64, 64),
         ("chunk_tc_kernel", True, [600], [0], 128, 128), ("chunk_tc_kernel", True, [64, 3, 65, 64, 1] * 20, [400] * 100, 16, 64),
         ("chunk_tc32_kernel", False, [200], [500], 32, 128), ("chunk_tc32_kernel", False, [200], [3000], 64, 64),
         ("attend_kernel", True, [9], [60], 16, 40)]


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("case", LATER, ids=_ids)
def test_later_values_do_not_leak(cuda, case, bad):
    """A non-finite value of a new token is the output of the tokens from its
    position on, in its column, and reaches nothing else; what lies past every
    sequence holds anything."""
    s = _case(cuda, case, fill=bad)
    clean = dict(s, k=s["k"].nan_to_num(0, 0, 0), v=s["v"].nan_to_num(0, 0, 0))
    ref, tol = _exact(clean)
    want = ref.clone()
    for i, (n, c, a) in enumerate(zip(s["new"], s["ctx"], s["starts"])):
        at = (2 * n) // 3
        page, row = _at(s, i, c + at)
        s["v"][page, :, row, 7] = bad
        want[a + at:a + n, :, 7] = bad
    got = _run(case, s)
    col = got[..., 7].clone()
    hit = ~want[..., 7].isfinite()
    assert (col[hit].isnan() if math.isnan(bad) else col[hit] == bad).all()
    col[hit] = ref[..., 7][hit].float()
    got[..., 7] = col
    _within(got, ref, tol)


def test_taken_out_values_of_neighbouring_pieces(cuda):
    """Segments of two and of one row tile in turn, a non-finite value in every
    other one's new tokens: each row gets its own back, call after call."""
    case = ("chunk_tc_kernel", True, [64, 6, 64, 5] * 40, [90, 20, 300, 400] * 40, 16, 64)
    s = _case(cuda, case)
    ref, tol = _exact(s)
    want = ref.clone()
    for i, (n, c, a) in enumerate(zip(s["new"], s["ctx"], s["starts"])):
        if i % 4 in (0, 3):
            page, row = _at(s, i, c + n - 2)
            s["v"][page, :, row, i % 64] = math.inf
            want[a + n - 2:a + n, :, i % 64] = math.inf
    hit = ~want.isfinite()
    for _ in range(10):
        got = _run(case, s)
        assert (got[hit] == math.inf).all()
        got[hit] = ref[hit].float()
        _within(got, ref, tol)


# ---------------------------------------------------------------- scores
def _longer(case):
    """The case without its sequences of fewer than 140 cached positions."""
    kept = [(n, c) for n, c in zip(case[2], case[3]) if c >= 140]
    return (*case[:2], [n for n, _ in kept], [c for _, c in kept], *case[4:])


@pytest.mark.parametrize("low", [-20.0, -1e3, -65504.0])
@pytest.mark.parametrize("case", [c for c in ALL if max(c[3]) >= 200], ids=_ids)
def test_lowest_keys_then_ordinary_ones(cuda, case, low):
    """The first 130 positions score far below the others, in the manner of a
    mask of the type's lowest value (f32 caches: times 1e27 as well): weights
    of zero to 64 bits, and the others' are as if they were not there."""
    case = _longer(case)
    _, kv16, new, ctx, page, dim = case
    for up in (1.0,) if kv16 else (1.0, 1e27):
        s = _case(cuda, case)
        s["q"][..., 0] = 1000.0 if low == -20.0 else 20.0
        s["k"][..., 0] *= 0.01      # of the ordinary positions
        for i in range(len(ctx)):
            for p in range(130):
                pg, row = _at(s, i, p)
                s["k"][pg, :, row, 0] = low * up
        ref, tol = _exact(s, drop=range(130))
        _within(_run(case, s), ref, tol)


@pytest.mark.parametrize("size", [9.0e5, 2.5e7, 4.0e7, 9.0e7, 1.8e8, 3.0e9, -9.0e5, -2.5e7, -4.0e7, -1.8e8, -3.0e9])
@pytest.mark.parametrize("case", ALL, ids=_ids)
def test_equal_scores_of_any_size(cuda, case, size):
    """Equal scores, however large, are equal weights: the mean of the values
    seen, to 2^-18 of the mean magnitude (weights) and 2^-24 for each position
    (a sum in f32)."""
    import torch
    s = _case(cuda, case)
    s["q"].zero_()
    s["q"][..., 0] = size * math.sqrt(case[5]) / math.log2(math.e) / 1024
    s["k"].zero_()
    s["k"][..., 0] = 1024.0
    got = _run(case, s)
    for i, (n, c, a) in enumerate(zip(s["new"], s["ctx"], s["starts"])):
        held = s["table"][s["slots"][i], :-(-(n + c) // s["page"])].long()
        v = s["v"][held].double().transpose(1, 2).flatten(0, 1)[:n + c]     # [positions, kv heads, dim]
        count = torch.arange(1, n + c + 1, device=v.device)[:, None, None]
        mean, size_of = (x.cumsum(0) / count for x in (v, v.abs()))
        for h in range(8):
            err = (got[a:a + n, h].double() - mean[c:, h // 4]).abs()
            tol = (2.0 ** -18 + 2.0 ** -24 * count[c:, 0]) * size_of[c:, h // 4]
            assert (err <= tol).all(), float(err.max())


@pytest.mark.parametrize("case", [c for c in TC if c[3][0] >= 400] + [c for c in TC32 if c[3][0] >= 400], ids=_ids)
def test_scores_below_every_number_first(cuda, case):
    """The first 130 positions' scores overflow to -inf: weights of zero."""
    case = _longer(case)
    _, kv16, new, ctx, page, dim = case
    s = _case(cuda, case)
    s["k"][..., 0] = 0.0
    s["q"].zero_()
    s["q"][..., 0] = 1e36           # finite scores are all 0: the mean of the values
    for i in range(len(ctx)):
        for p in range(130):
            pg, row = _at(s, i, p)
            s["k"][pg, :, row, 0] = -65504.0 if kv16 else -math.inf
    ref, tol = _exact(dict(s, q=s["q"] * 0), drop=range(130))
    _within(_run(case, s), ref, tol)


# ------------------------------------------------------- bad arguments on the device
BAD = [("few_kernel", True, [1, 2, 1], [50, 300, 40], 16, 128), ("few_kernel", False, [1, 2, 1], [50, 300, 40], 16, 64),
       ("chunk_kernel", True, [40, 30, 40], [50, 100, 9], 16, 128), ("chunk_kernel", False, [9, 12, 9], [30, 40, 8], 16, 64),
       ("chunk_tc_kernel", True, [100, 90, 80], [500, 700, 9], 16, 128), ("chunk_tc_kernel", True, [100, 90, 80], [500, 700, 9], 128, 64),
       ("chunk_tc32_kernel", False, [100, 90, 80], [500, 700, 9], 16, 128), ("chunk_tc32_kernel", False, [70, 70, 70], [400, 300, 9], 48, 64),
       ("attend_kernel", True, [1, 4, 3], [50, 100, 9], 16, 48), ("attend_kernel", False, [1, 4, 3], [50, 100, 9], 16, 96)]


@pytest.mark.parametrize("infinite", [False, True])
@pytest.mark.parametrize("entry", [-1, -5, 1 << 30, None])
@pytest.mark.parametrize("case", BAD, ids=_ids)
def test_bad_page_entries_read_as_zeros(cuda, case, entry, infinite):
    """A table entry that names no page: its positions count as keys and values
    of zero (no other request's are read), beside an infinity in the same tile
    too; the other sequences are as they were, HYQ_DEV_BAD_ARGS is raised."""
    import torch
    from hy_mt_rs_b200 import quant
    s = _case(cuda, case)
    s["k"][0] = 3.0
    s["v"][0] = 1e4             # a page that must not be read
    taken = s["table"].clone()
    # no sequence holds page 0: swap it for a free one
    free = sorted(set(range(s["k"].shape[0])) - set(taken[taken >= 0].tolist()))
    if 0 not in free:
        s["table"][taken == 0] = free[-1]
    if infinite:
        page, row = _at(s, 1, 0)
        s["v"][page, :, row, 3] = math.inf
    good = _run(case, s)
    assert quant.device_status() == 0
    a, b = s["starts"][1], s["starts"][2]
    t = dict(s, table=s["table"].clone())
    t["table"][1, 1] = s["k"].shape[0] if entry is None else entry
    out = torch.zeros_like(good)
    _run(case, t, out=out)
    assert quant.device_status() == 8
    assert torch.equal(out[:a], good[:a]) and torch.equal(out[b:], good[b:])
    # zeros in their place, on a page of their own
    z = dict(s, table=s["table"].clone(), k=torch.cat([s["k"], torch.zeros_like(s["k"][:1])]),
             v=torch.cat([s["v"], torch.zeros_like(s["v"][:1])]))
    z["table"][1, 1] = s["k"].shape[0]
    z["v"].nan_to_num_(posinf=0.0)
    ref, tol = _exact(z)
    if infinite:
        assert (out[a:b, :, 3] == math.inf).all()
        out[a:b, :, 3] = ref[a:b, :, 3].float()
    _within(out[a:b], ref[a:b], tol[a:b])


@pytest.mark.parametrize("kv16", [True, False])
def test_more_tokens_than_max_new_are_reported(cuda, kv16):
    """max_new too small for a sequence raises HYQ_DEV_BAD_ARGS; the others are
    right."""
    import torch
    from hy_mt_rs_b200 import paged, quant
    s = _make(cuda, [1, 40, 2], [50, 20, 300], 8, 2, 128, 16, kv16)
    ref, tol = _exact(s)
    out = torch.zeros_like(s["q"])
    paged.attention(s["q"], s["k"], s["v"], s["table"], s["row_start"], s["pos"], 2, out=out)
    assert quant.device_status() == 8
    for rows in (slice(0, 1), slice(41, 43)):
        _within(out[rows], ref[rows], tol[rows])


# ---------------------------------------------------------------- graphs
GRAPH = [("chunk_tc_kernel", True, [200, 1, 3], [500, 900, 70], 32, 128), ("chunk_kernel", True, [40, 1], [100, 90], 32, 128),
         ("chunk_tc32_kernel", False, [130, 2, 1], [500, 90, 700], 32, 128), ("chunk_kernel", False, [30, 2], [10, 5], 32, 64)]


@pytest.mark.parametrize("overlap", [False, True])
@pytest.mark.parametrize("case", GRAPH, ids=_ids)
def test_chunk_calls_in_a_graph(cuda, case, overlap):
    """Two chunk calls captured with their programmatic edges, replayed while
    the positions change in place."""
    import torch
    from hy_mt_rs_b200 import paged, quant
    s = _case(cuda, case)
    ws = paged.attention_workspace(8, case[5], cuda)
    length = max(n + c for n, c in zip(s["new"], s["ctx"]))
    out, again = torch.empty_like(s["q"]), torch.empty_like(s["q"])
    _run(case, s, out=out, workspace=ws)
    quant.set_launch_overlap(overlap)
    try:
        g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=st):
            _attend(s, out=out, workspace=ws, max_len=length)
            _attend(dict(s, q=out), out=again, workspace=ws, max_len=length)
    finally:
        quant.set_launch_overlap(False)
    for less in (0, 1, 5):
        s["ctx"] = [max(c - less, 0) for c in case[3]]
        s["pos"].copy_(_int(s["ctx"], cuda))
        out.zero_()
        for _ in range(3):
            g.replay()
        torch.cuda.synchronize()
        ref, tol = _exact(s)
        _within(out, ref, tol)
        ref, tol = _exact(dict(s, q=out))
        _within(again, ref, tol)
    assert quant.device_status() == 0


@pytest.mark.parametrize("case", [FEW[1], FEW[3], TC[0], TC32[1]], ids=_ids)
def test_workspace_of_used_memory(cuda, case):
    """A workspace in memory that holds NaN and large numbers: only its first
    bytes are zero."""
    import torch
    from hy_mt_rs_b200 import paged
    s = _case(cuda, case)
    ref, tol = _exact(s)
    for x in (math.nan, 1e38):
        ws = paged.attention_workspace(8, case[5], cuda)
        ws[4096:] = torch.full((ws.numel() // 4,), x, device=cuda).view(torch.uint8)[:ws.numel() - 4096]
        _within(_run(case, s, workspace=ws), ref, tol)
        _within(_run(case, s, workspace=ws), ref, tol)
        assert int(ws[:4096].amax()) == 0


@pytest.mark.parametrize("case", [FEW[0], CHUNK[0], TC[0], TC32[0], OTHER[0]], ids=_ids)
def test_descending_row_starts_are_reported(cuda, case):
    """row_start that goes back gives rows to several sequences and others a
    negative number: HYQ_DEV_BAD_ARGS, and nothing past the rows is written."""
    import torch
    from hy_mt_rs_b200 import quant
    s = _case(cuda, case)
    n, seqs = s["new"][0], 40
    t = dict(s, row_start=_int([0, n] * seqs, cuda), pos=s["pos"][:1].repeat(2 * seqs - 1), slots=None,
             slot=torch.zeros(2 * seqs - 1, dtype=torch.int32, device=cuda))
    buf = torch.full((n + 8, 8, case[5]), 7.0, device=cuda)
    _run((case[0], *case[1:]), dict(t, q=s["q"][:n]), out=buf[:n])
    assert (buf[n:] == 7).all() and quant.device_status() == 8
