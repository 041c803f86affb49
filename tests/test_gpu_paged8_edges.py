"""Attention over 8-bit caches and of shared prefixes at their edges: a max_new that
is too small, tiles of far units, keys under uneven weights, workspaces of used memory,
overlapped launches."""
import math

import pytest

from test_gpu_paged import _int, _reference
from test_gpu_paged8 import KINDS, _attend, _make8
from test_gpu_shared import _attend as _attend_shared
from test_gpu_shared import _make as _make_shared

pytestmark = pytest.mark.gpu


def _bound(s):
    """test_gpu_paged8._close's reference and bound."""
    import torch
    ref, tol = _reference(s)
    heads = s["q"].shape[1]
    group = heads // s["k"].shape[1]
    for i, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        a = s["starts"][i]
        held = s["table"][s["slots"][i], :-(-(n + c) // s["page"])].long()
        for h in range(heads if n and s["kv"] else 0):
            k, v = (s[x][held, h // group].double().reshape(-1, s["q"].shape[2])[:n + c] for x in ("k", "v"))
            x = s["q"][a:a + n, h].double() @ k.T / math.sqrt(s["q"].shape[2])
            hide = torch.arange(n + c, device=x.device)[None] > torch.arange(c, n + c, device=x.device)[:, None]
            p = torch.softmax(x.masked_fill(hide, -math.inf), -1)
            tol[a:a + n, h] += 2.0 ** -18 * (p @ v.abs().amax(-1))[:, None]
    return ref, tol


def _right_or_left(got, s, ref, tol, fill, status):
    """Every sequence's rows within their bound; or left alone, and reported."""
    import torch
    for i, n in enumerate(s["new"]):
        rows = slice(s["starts"][i], s["starts"][i] + n)
        if torch.equal(got[rows], torch.full_like(got[rows], fill)) and n:
            assert status == 8, i
        else:
            err = (got[rows].double() - ref[rows]).abs()
            assert (err <= tol[rows]).all(), (i, float((err / tol[rows]).max()))


# ------------------------------------------------------------------- max_new
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,max_new,new", [(6, 2, 3, [5, 1]), (6, 2, 4, [5, 2]), (10, 2, 2, [3, 1, 2]), (8, 2, 1, [3, 1]),
                                                   (8, 2, 2, [4, 1]), (3, 3, 9, [16, 2]), (14, 2, 1, [2, 1]), (8, 2, 2, [40, 1])])
def test_more_tokens_than_max_new(cuda, heads, kvh, max_new, new, kind):
    """A sequence with more new tokens than max_new is taken whole, or left alone and
    reported; the others are right."""
    import torch
    from hy_mt_rs_b200 import paged, quant
    s = _make8(cuda, new, [50, 300, 20][:len(new)], heads, kvh, 128, 16, kind, seed=heads)
    out = torch.full_like(s["q"], 7.0)
    paged.attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos"], max_new, out=out, **s["kv"])
    _right_or_left(out, s, *_bound(s), 7.0, quant.device_status())


@pytest.mark.parametrize("kind", ["f32", "f16", *KINDS])
@pytest.mark.parametrize("heads,kvh,max_new,new", [(8, 2, 1, [1, 3, 1]), (8, 2, 2, [1, 4, 2]), (6, 2, 3, [5, 1, 2]), (8, 2, 1, [1, 1, 7])])
def test_more_tokens_than_max_new_behind_a_prefix(cuda, heads, kvh, max_new, new, kind):
    """Likewise of a group, next to a group without such a sequence; never outputs made
    of what the workspace held; reported in any case."""
    import torch
    from hy_mt_rs_b200 import paged, quant
    s = _make_shared(cuda, [(150, [(9 + i, n) for i, n in enumerate(new)]), (200, [(0, 1), (31, 1)])], heads, kvh, 128, 32, kind, seed=4)
    t = s["q"].shape[0]
    ws = paged.attention_shared_workspace(heads, 128, t, cuda)
    ws[4096:] = torch.full((ws.numel() // 4,), 1.0, device=cuda).view(torch.uint8)[:ws.numel() - 4096]
    out = torch.full_like(s["q"], 7.0)
    paged.attention_shared(s["q"], s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos"], s["group_start"], s["shared"],
                           max_new, out=out, workspace=ws, **s["kv"])
    status = quant.device_status()
    assert status == 8
    _right_or_left(out, s, *_bound(s), 7.0, status)
    assert (out[sum(new):] != 7.0).all()


# -------------------------------------------------------------- units of tiles
def _scaled(s, factor):
    """The values with V's scales times factor(positions) of every sequence."""
    import torch
    from test_gpu_paged8 import _values
    scale = s["kv"]["v_scale"]
    times = torch.ones_like(scale)
    for i, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        p = torch.arange(n + c, device=scale.device)
        times[s["table"][s["slots"][i]][(p // s["page"]).long()].long(), :, p % s["page"]] = factor(p).float()[:, None]
    scale *= times
    s["v"] = _values(s["v_pages"], scale)
    return s


def _where(condition, a, b):
    import torch
    return torch.where(condition, a, b)


UNITS = [(2.0 ** -70, 1.0), (1.0, 2.0 ** -70), (2.0 ** -30, 2.0 ** 70), (2.0 ** 50, 2.0 ** -50), (2.0 ** -20, 2.0 ** -12)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("first,then", UNITS)
@pytest.mark.parametrize("new,ctx", [([200, 1], [700, 300]), ([1, 3], [900, 400])])
def test_tiles_of_far_units(cuda, new, ctx, first, then, dim, kind):
    """Whole tiles of 128 positions whose scales of V are alike, far from those of the
    next tiles: their positions keep their weights, whatever their values' size."""
    import torch
    s = _make8(cuda, new, ctx, 16, 4, dim, 32, kind, seed=12, spread=0.1)
    _scaled(s, lambda p: _where(p // 128 % 3 == 0, first, then))
    _close_far(_attend(s), s)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("first,then", UNITS)
def test_tiles_of_far_units_in_a_prefix(cuda, first, then, kind):
    import torch
    s = _make_shared(cuda, [(640, [(9, 1), (0, 2), (50, 1)]), (200, [(1, 1), (70, 2)])], 8, 2, 128, 32, kind, seed=6)
    _scaled(s, lambda p: _where(p // 128 % 3 == 0, first, then))
    _close_far(_attend_shared(s), s)


def _close_far(got, s):
    """Within the element-wise bound alone: outputs are sums of very different sizes."""
    import torch
    from hy_mt_rs_b200 import quant
    ref, tol = _bound(s)
    assert torch.isfinite(got).all() and quant.device_status() == 0
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())


SIZES = [1.0, 2.0 ** -15, 2.0 ** -30, 2.0 ** 40]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("new,ctx", [([200, 260], [700, 600]), ([1, 3], [900, 400])])
def test_tiles_of_zeros_before_small_values(cuda, new, ctx, size, kind):
    """Sequences that begin with positions whose values are zeros, the second one behind
    one of large values: the values that follow keep their bits."""
    from test_gpu_paged8 import _values
    s = _make8(cuda, new, ctx, 16, 4, 128, 32, kind, seed=13, spread=0.1)
    large = s["table"][s["slots"][0]].long()
    large = large[large >= 0]
    keep = s["kv"]["v_scale"][large].clone()
    _scaled(s, lambda p: _where(p < 256, 0.0, size))
    _close_far(_attend(s), s)
    s["kv"]["v_scale"][large] = keep * 2.0 ** 60
    s["v"] = _values(s["v_pages"], s["kv"]["v_scale"])
    _close_far(_attend(s), s)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("new,ctx", [([200, 260], [700, 600]), ([1, 3], [900, 4000]), ([20], [150])])
def test_rows_of_zeros_among_others(cuda, new, ctx, size, kind):
    """Single positions without a value, and whole tiles of them, next to values: their
    weights count."""
    s = _make8(cuda, new, ctx, 8, 2, 128, 32, kind, seed=14, spread=0.1)
    _scaled(s, lambda p: _where((p % 3 == 1) | (p // 128 % 2 == 0) & (p > 60), 0.0, size))
    _close_far(_attend(s), s)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("first", [256, 0])
def test_prefixes_with_rows_of_zeros(cuda, first, size, kind):
    s = _make_shared(cuda, [(640, [(9, 1), (0, 2), (50, 1)]), (300, [(1, 1), (70, 2)])], 8, 2, 128, 32, kind, seed=7)
    _scaled(s, lambda p: _where((p < first) | (p % 3 == 1) & (first == 0), 0.0, size))
    _close_far(_attend_shared(s), s)


# ------------------------------------------------------------------- append
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("ratio", [1, 20, 200, 1000])
@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("dim,tokens", [(128, 40), (128, 8000), (64, 8000), (80, 40)])
def test_keys_next_to_borders_under_uneven_weights(cuda, dim, tokens, first, ratio, kind):
    """Heads with one value next to a border between two codes (the others lie on codes),
    whose weight is `ratio` times its partner's in the rotation: f32 moves it by a share
    of the pair.  All codes are those of 64 bits, where 2^-38 * ratio of a value does not
    decide (the kernel's 64-bit roundings: 2^-43 * ratio of 127, then 2^-40)."""
    import torch
    from test_gpu_paged8 import _append, _append_inputs, _exact_keys, _pages8, _quantise, _types
    s = _append_inputs(cuda, [tokens], [0], 2, 2, dim, 64, seed=dim + tokens, positions=tokens)
    g = torch.Generator(device=cuda).manual_seed(5)
    rand = lambda *n: torch.rand(*n, generator=g, device=cuda, dtype=torch.float64)  # noqa: E731
    whole = lambda lo, hi, *n: torch.randint(lo, hi, n, generator=g, device=cuda)  # noqa: E731
    half, largest = dim // 2, _types()[kind][1]
    heavy = torch.arange(half, device=cuda) % 2 == 0
    heavy = torch.cat([heavy, ~heavy])
    s["k_norm"] = (torch.where(heavy, float(ratio), 1.0) * (1 + 0.1 * rand(dim))).float()
    w, top = s["k_norm"].double(), 1 + rand(tokens, 2, 1)

    def code(n):
        return n.double() if kind == "i8" else n.to(torch.uint8).view(torch.float8_e4m3fn).double()

    n = whole(0, 127, tokens, 2, dim)
    z = code(n) * (2 * whole(0, 2, tokens, 2, dim) - 1)
    at = whole(0, half // 2, tokens, 2, 1) * 2 + whole(0, 2, tokens, 2, 1) * (half + 1)      # a heavy one
    n = whole(0, 126, tokens, 2, 1)
    z.scatter_(2, at, (code(n) + code(n + 1)) / 2)
    z.scatter_(2, (at + half) % dim, code(whole(112 if kind == "f8" else 64, 126, tokens, 2, 1)))
    on_top = (at + 2) % half
    z = z.scatter(2, on_top, torch.full_like(top, largest)) / largest * top
    c, sn = (s[t][:tokens, None].double() for t in ("cos", "sin"))
    a, b = (z if first else z / w).chunk(2, -1)
    x = torch.cat([a * c + b * sn, b * c - a * sn], -1)
    s["new_k"] = (x / w if first else x).float()
    k8, v8, scales = _pages8(cuda, s["k"], kind)
    k32, v32 = (torch.full_like(s[t], 777.0) for t in ("k", "v"))
    _append(s, k32, v32, True, first)
    _append(s, k8, v8, True, first, **scales)
    pages = s["table"][0, :-(-tokens // 64)].long()
    rows = lambda t: t[pages].transpose(1, 2).reshape(-1, 2, *t.shape[3:])[:tokens].cpu()  # noqa: E731
    exact = torch.stack([_exact_keys(s, t, t, True, first) for t in range(tokens)])
    got = rows(k8.view(torch.uint8))
    wants = [_quantise(rows(k32), kind, exact)]
    assert torch.equal(rows(scales["k_scale"]), wants[0][1])
    # what the kernel's 64-bit roundings may move over a border
    y = exact * largest / exact.abs().amax(-1, keepdim=True)
    either = [(v.round().clamp(-127, 127).to(torch.int8) if kind == "i8" else v.float().to(torch.float8_e4m3fn)).view(torch.uint8)
              for v in (y * (1 - 2.0 ** -38 * ratio), y * (1 + 2.0 ** -38 * ratio))]
    wrong = (got != wants[0][0].view(torch.uint8)) & ((got == either[0]) == (got == either[1]))
    assert not wrong.any(), int(wrong.sum())


def test_weights_of_zero(cuda):
    """A pair with one weight of zero, and one with two: its values are 0 or anything, and
    the codes those of 64 bits."""
    import torch
    from test_gpu_paged8 import _append, _append_inputs, _exact_keys, _pages8, _quantise
    for tokens in (40, 1000):
        s = _append_inputs(cuda, [tokens], [0], 2, 2, 128, 64, seed=tokens, positions=tokens)
        s["k_norm"][[3, 7, 71]] = 0.0
        k8, v8, scales = _pages8(cuda, s["k"], "i8")
        k32, v32 = (torch.full_like(s[t], 777.0) for t in ("k", "v"))
        _append(s, k32, v32, True, False)
        _append(s, k8, v8, True, False, **scales)
        pages = s["table"][0, :-(-tokens // 64)].long()
        rows = lambda t: t[pages].transpose(1, 2).reshape(-1, 2, *t.shape[3:])[:tokens].cpu()  # noqa: E731
        exact = torch.stack([_exact_keys(s, t, t, True, False) for t in range(tokens)])
        want, want_scale = _quantise(rows(k32), "i8", exact)
        assert torch.equal(rows(scales["k_scale"]), want_scale) and torch.equal(rows(k8), want)


# ----------------------------------------------------------------- in place
@pytest.mark.parametrize("kind", ["f32", "f16", *KINDS])
@pytest.mark.parametrize("dim", [128, 80])
@pytest.mark.parametrize("new,ctx", [([1, 3, 2], [900, 40, 5000]), ([200, 1, 70], [700, 300, 9]), ([40, 1], [20, 5])])
def test_in_place(cuda, new, ctx, dim, kind):
    """Outputs in the queries' place: the same bits."""
    import torch
    from test_gpu_paged import _make
    if kind in KINDS:
        s = _make8(cuda, new, ctx, 8, 2, dim, 32, kind, seed=21)
    else:
        s = _make(cuda, new, ctx, 8, 2, dim, 32, kind == "f16", seed=21)
        s.update(kv={}, k_pages=s["k"], v_pages=s["v"])
    want, wide = _attend(s), torch.full((sum(new), 11, dim), 3.0, device=cuda)
    wide[:, :8] = s["q"]
    s["q"] = wide[:, :8]
    _attend(s, out=s["q"])
    assert torch.equal(s["q"], want) and (wide[:, 8:] == 3).all()


@pytest.mark.parametrize("kind", ["f32", "f16", *KINDS])
@pytest.mark.parametrize("per", [2, 70])
def test_in_place_behind_a_prefix(cuda, per, kind):
    """A sequence's own positions are done long before its group's prefix: queries are
    read by that first."""
    import torch
    s = _make_shared(cuda, [(6000, [((i * 37) % 20, 1) for i in range(per)]), (200, [(0, 1), (31, 2)])], 16, 4, 128, 64, kind, seed=22)
    want, q = _attend_shared(s), s["q"].clone()
    for _ in range(5):
        s["q"] = q.clone()
        _attend_shared(s, out=s["q"])
        assert torch.equal(s["q"], want)


def test_in_place_wants_the_queries_stride(cuda):
    import torch
    from hy_mt_rs_b200._native import HyqError
    s = _make8(cuda, [1, 3], [90, 40], 8, 2, 128, 32, "i8", seed=21)
    buf = torch.zeros(4 * 11 * 128, device=cuda)
    s["q"] = buf.view(4, 11, 128)[:, :8]
    with pytest.raises(HyqError, match="in place with two strides"):
        _attend(s, out=buf[:4 * 8 * 128].view(4, 8, 128))
    s = _make8(cuda, [1], [90], 8, 2, 128, 32, "i8", seed=21)     # one row has none
    want, buf = _attend(s), torch.zeros(11 * 128, device=cuda)
    buf[:1024] = s["q"].flatten()
    s["q"] = buf.as_strided((1, 8, 128), (11 * 128, 128, 1))
    assert torch.equal(_attend(s, out=buf[:1024].view(1, 8, 128)), want)


# --------------------------------------------------------------------- scales
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("new,ctx", [([1, 3], [900, 400]), ([200, 1], [500, 70]), ([20], [60])])
def test_scales_of_either_sign(cuda, new, ctx, far, dim, kind):
    """A value is code * scale: scales that appending does not write, below zero, count like
    any; also in tiles that are left out of the products (`far`)."""
    import torch
    from test_gpu_paged8 import _values
    s = _make8(cuda, new, ctx, 8, 2, dim, 16, kind, seed=31)
    g = torch.Generator(device=cuda).manual_seed(6)
    for name in ("k", "v"):
        scale = s["kv"][name + "_scale"]
        scale *= 1 - 2 * torch.randint(0, 2, scale.shape, generator=g, device=cuda).float()
        if far and name == "v":
            scale *= torch.exp2(torch.randint(-20, 21, scale.shape, generator=g, device=cuda).float())
        s[name] = _values(s[name + "_pages"], scale)
    _close_far(_attend(s), s)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("far", [False, True])
def test_scales_of_a_prefix_of_either_sign(cuda, far, kind):
    """And 2^20 apart within a prefix's tiles, behind and in front of whole ones."""
    import torch
    s = _make_shared(cuda, [(900, [(9, 1), (0, 2), (150, 1)]), (300, [(1, 1), (270, 2)])], 8, 2, 128, 32, kind, seed=8)
    _scaled(s, lambda p: (1 - 2 * (p * 7 // 3 % 2)) * _where((p // 256 % 2 == 1) & far, torch.exp2(10.0 - (p * 37 % 21)), 1.0))
    _close_far(_attend_shared(s), s)


# --------------------------------------------------------------------- groups
@pytest.mark.parametrize("kind,dim", [("f32", 128), ("f16", 64), ("i8", 128), ("f8", 128), ("f16", 80), ("i8", 256)])
def test_bad_groups_of_small_prefixes_are_reported(cuda, kind, dim):
    """Also where the prefixes are not worth their own kernels, or not for them: the same
    outputs, and the device status; none for good groups."""
    import torch
    from hy_mt_rs_b200 import quant
    groups = [(140, [(9, 1), (0, 1), (50, 1)]), (200, [(1, 1), (70, 2)])]
    s = _make_shared(cuda, groups, 8, 2, dim, 32, kind, seed=4)
    good = [([140, 200], [0, 3, 5]), ([140], [0, 2]), ([200], [3, 5]), ([], [0]), ([140, 9999, 200], [0, 3, 3, 5]), ([99999, 1], [0, 1, 1]),
            ([0, 0], [0, 1, 5])]
    bad = [([141, 200], [0, 3, 5]), ([-1, 200], [0, 3, 5]), ([140, 200], [0, 3, 6]), ([140, 200], [0, 6, 5]), ([140, 200], [-1, 3, 5]),
           ([140, 2 ** 31 - 1], [0, 3, 5]), ([140, 202], [0, 3, 5])]
    want = None
    for shared, start in good + bad:
        s.update(shared=_int(shared, cuda), group_start=_int(start, cuda))
        got = _attend_shared(s, max_len=400, max_shared=300)
        want = got if want is None else want
        assert torch.equal(got, want)
        assert quant.device_status() == (0 if (shared, start) in good else 8), (shared, start)


def test_many_groups_of_small_prefixes(cuda):
    """More groups than a block has threads, one of them bad, wherever it is."""
    import torch
    from hy_mt_rs_b200 import quant
    n = 700
    s = _make_shared(cuda, [(3, [(i % 3, 1), (0, 1)]) for i in range(n)], 4, 2, 64, 16, "f16", seed=2)
    want = _attend_shared(s, max_len=10, max_shared=10)
    assert quant.device_status() == 0
    for i in (0, 299, n - 1):
        s["shared"][i] = 4      # its second sequence holds three
        assert torch.equal(_attend_shared(s, max_len=10, max_shared=10), want)
        assert quant.device_status() == 8
        s["shared"][i] = 3


# ------------------------------------------------- prefixes that are not finite
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("where", [0, 130, 640, 899])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_prefix_scales_that_are_not_finite(cuda, where, bad, kind):
    """A row of V of the prefix with such a scale makes its group NaN in that kv head (an
    infinite one infinities or NaN), one of K too, one behind the prefix its own sequence; the
    other head and the other group stay within their bound."""
    import torch
    s = _make_shared(cuda, [(900, [(9, 1), (0, 2), (150, 1)]), (300, [(1, 1), (270, 2)])], 8, 2, 128, 32, kind, seed=9)
    ref, tol = _bound(s)
    gone = (lambda x: bool(torch.isnan(x).all())) if math.isnan(bad) else (lambda x: not torch.isfinite(x).any())  # noqa: E731
    near = lambda got, rows, heads: bool(((got.double() - ref).abs() <= tol)[rows, heads].all())  # noqa: E731
    page, row = int(s["table"][0, where // 32]), where % 32
    pages = {page} if where < 896 else {int(s["table"][i, 28]) for i in range(3)}    # (the partial page: each one's own)
    for page in pages:
        s["kv"]["v_scale"][page, 1, row] = bad
    got = _attend_shared(s)
    assert gone(got[:4, 4:])
    assert near(got, slice(0, 4), slice(0, 4)) and near(got, slice(4, None), slice(0, 8))
    s["kv"]["k_scale"][int(s["table"][3, 2]), 0, 5] = math.nan     # position 69 of the other group's
    got = _attend_shared(s)
    assert torch.isnan(got[4:, :4]).all() and gone(got[:4, 4:])
    assert near(got, slice(0, 4), slice(0, 4)) and near(got, slice(4, None), slice(4, 8))
    for page in pages:
        s["kv"]["v_scale"][page, 1, row] = 0.01
    s["kv"]["v_scale"][int(s["table"][2, 1000 // 32]), 0, 1000 % 32] = bad     # sequence 2's own
    got = _attend_shared(s)
    assert gone(got[3, :4]) and near(got, slice(0, 3), slice(0, 4))


# -------------------------------------------------- workspaces, overlapped launches
def _calls(cuda, kind):
    """Calls of this file's operators that reach their kernels, and their workspaces."""
    import torch
    from hy_mt_rs_b200 import paged
    from test_gpu_paged import _make
    out = []
    for new, ctx in (([200, 1], [700, 300]), ([1, 3, 2], [900, 40, 5000]), ([40, 1], [20, 5])):
        if kind in KINDS:
            s = _make8(cuda, new, ctx, 8, 2, 128, 32, kind, seed=41)
        else:
            s = _make(cuda, new, ctx, 8, 2, 128, 32, kind == "f16", seed=41)
            s.update(kv={}, k_pages=s["k"], v_pages=s["v"])
        out.append((s, _attend, paged.attention_workspace(8, 128, cuda)))
    s = _make_shared(cuda, [(900, [(9, 1), (0, 2), (150, 1)]), (300, [(1, 1), (270, 2)])], 8, 2, 128, 32, kind, seed=42)
    out.append((s, _attend_shared, paged.attention_shared_workspace(8, 128, s["q"].shape[0], cuda)))
    return out


@pytest.mark.parametrize("kind", ["f32", "f16", *KINDS])
def test_workspaces_of_used_memory(cuda, kind):
    """Only a workspace's first bytes are zero: the same bits, call after call."""
    import torch
    for s, attend, ws in _calls(cuda, kind):
        want = attend(s)
        for x in (math.nan, 1e38, -1e-3):
            ws[4096:] = torch.full((ws.numel() // 4 + 1,), x, device=cuda).view(torch.uint8)[:ws.numel() - 4096]
            for _ in range(2):
                assert torch.equal(attend(s, workspace=ws), want)
            assert int(ws[:4096].amax()) == 0


@pytest.mark.parametrize("kind", ["f32", "f16", *KINDS])
@pytest.mark.parametrize("captured", [False, True])
def test_overlapped_launches(cuda, captured, kind):
    """Chains of appends, reads, attention and adjusted logits in which each takes what the
    one before wrote, with programmatic launches and without: the same bits."""
    import torch
    from hy_mt_rs_b200 import paged, quant, sampling
    from test_gpu_paged8 import _append_inputs
    g = torch.Generator(device=cuda).manual_seed(3)
    history = torch.randint(0, 9000, (8, 5000), generator=g, device=cuda, dtype=torch.int32)
    length = torch.full((8,), 5000, dtype=torch.int32, device=cuda)
    chains = []
    for s, attend, ws in _calls(cuda, kind):
        a = _append_inputs(cuda, s["new"], s["ctx"], 8, 2, 128, 32, seed=7, positions=6000)
        a["many"] = [torch.randn(600, h, 128, generator=g, device=cuda) for h in (8, 2, 2)]

        def chain(s=s, attend=attend, ws=ws, a=a):
            # (rows behind the last sequence take the staged append to them as well)
            q, k, v = a["many"]
            t = s["q"].shape[0]
            q[:t], k[:t], v[:t] = s["q"], a["new_k"], a["new_v"]
            pages = (s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos"])
            rotated = paged.rope_append(q, k, v, *pages, a["cos"], a["sin"], a["q_norm"], a["k_norm"], slot=s["slot"], **s["kv"])
            x = attend(dict(s, q=rotated[:t]), workspace=ws)
            back = paged.gather(*pages, t, slot=s["slot"], **s["kv"])
            y = attend(dict(s, q=x), workspace=ws)
            logits = torch.nn.functional.pad(y.reshape(t, -1)[:1].repeat(8, 9), (0, 0))
            z = sampling.adjust(logits, history, length, repetition=1.2, frequency=0.1)
            return [x, *back, y, z, *(p.view(torch.uint8) for p in pages[:2])]

        chains.append(chain)
    want = [[t.clone() for t in c()] for c in chains]       # (the appends write the same rows again)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        quant.set_launch_overlap(True)
        for c, w in zip(chains, want):
            if captured:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    got = c()
                for _ in range(3):
                    graph.replay()
            else:
                for _ in range(3):
                    got = c()
            torch.cuda.synchronize()
            for x, y in zip(got, w):
                assert torch.equal(x, y)
    finally:
        quant.set_launch_overlap(False)
    assert quant.device_status() == 0


@pytest.mark.parametrize("kind", ["f32", "f16", *KINDS])
@pytest.mark.parametrize("groups", [60, 200])
def test_many_short_prefixes(cuda, groups, kind):
    """CTAs that go through one prefix after another, each of a tile or two of which the last
    is masked: the pipelines run ahead from one into the next."""
    s = _make_shared(cuda, [(40 + 53 * i % 230, [(i % 9, 1), (0, 1 + i % 2)]) for i in range(groups)], 16, 4, 128, 32, kind, seed=groups)
    want = _attend_shared(s)
    _close_far(want, s)
    import torch
    for _ in range(20):
        assert torch.equal(_attend_shared(s), want)


def test_groups_of_a_batch_of_very_many_rows(cuda):
    """Rows behind the last sequence count as the call's, 2^25 of them here: threads of the
    grid that looks the groups over are numbered in 64 bits."""
    import torch
    from hy_mt_rs_b200 import paged, quant
    s = _make_shared(cuda, [(30, [(2, 1), (0, 2), (9, 1)])], 1, 1, 8, 16, "f16", seed=3)
    few = _attend_shared(s, max_len=50, max_shared=30)
    wide, out = (torch.zeros(2 ** 25 + 4, 1, 8, device=cuda) for _ in range(2))
    wide[:4] = s["q"]
    ws = paged.attention_shared_workspace(1, 8, wide.shape[0], cuda)
    for shared, status in ((30, 0), (31, 8)):
        s["shared"][0] = shared
        _attend_shared(dict(s, q=wide), max_len=50, max_shared=30, out=out, workspace=ws)
        assert torch.equal(out[:4], few) and not out[4:].any()
        assert quant.device_status() == status


@pytest.mark.parametrize("kind,dim", [("f16", 128), ("i8", 128), ("f32", 80)])
def test_more_tokens_than_max_new_behind_a_small_prefix(cuda, kind, dim):
    """Reported as behind a large one; the sequences are right, or left alone."""
    import torch
    from hy_mt_rs_b200 import paged, quant
    s = _make_shared(cuda, [(150, [(9, 1), (3, 2), (0, 1)]), (200, [(0, 1), (31, 1)])], 8, 2, dim, 32, kind, seed=4)
    out = torch.full_like(s["q"], 7.0)
    paged.attention_shared(s["q"], s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos"], s["group_start"], s["shared"],
                           1, max_len=400, max_shared=200, out=out, **s["kv"])
    status = quant.device_status()
    assert status == 8
    _right_or_left(out, s, *_bound(s), 7.0, status)
