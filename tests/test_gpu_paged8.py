"""GPU parity of the 8-bit paged cache: the codes and scales that appending
writes against those of an f32 cache's values (bit for bit), rows read back,
attention against a 64-bit softmax over the values that the codes stand for."""
import math

import pytest

from test_gpu_paged import _int, _make, _reference

pytestmark = pytest.mark.gpu

KINDS = ["i8", "f8"]
NAN_CODES = 0x7f, 0xff


def _types():
    import torch
    return {"i8": (torch.int8, 127.0), "f8": (torch.float8_e4m3fn, 448.0)}


def _values(codes, scale):
    """The values, f64 (the e4m3 codes without NaN: 0x7f and 0xff are +-480)."""
    import torch
    x = codes.double()
    if codes.dtype == torch.float8_e4m3fn:
        bits = codes.view(torch.uint8)
        x = torch.where(bits == 0x7f, 480.0, torch.where(bits == 0xff, -480.0, x))
    return x * scale.double()[..., None]


def _quantise(x, kind, exact=None):
    """Codes and scales of rows of f32 values, by the documented rule, on the CPU.
    exact: what they are before their roundings to f32, up to a factor of the row."""
    import torch
    dtype, largest = _types()[kind]
    x = x.cpu()
    top = x.abs().amax(-1)
    top = torch.where(top < 2.0 ** -90, 0.0, top)
    scale = top / largest
    y = x.double() if exact is None else exact.cpu()
    y = y * largest / y.abs().amax(-1, keepdim=True).clamp(min=1e-300)
    codes = y.round().clamp(-127, 127).to(dtype) if kind == "i8" else y.float().to(dtype)
    bad = ~torch.isfinite(x).all(-1)
    scale[bad] = math.nan
    codes.view(torch.uint8)[bad | (top == 0)] = 0    # (not -0)
    return codes, scale


def _make8(dev, new, ctx, heads, kvh, dim, page, kind, layout="hnd", spread=0.5, seed=0, **kw):
    """test_gpu_paged's inputs over codes: s["k"], s["v"] are the values (for the
    64-bit reference), codes and scales in s["kv"]."""
    import torch
    s = _make(dev, new, ctx, heads, kvh, dim, page, False, layout=layout, seed=seed, **kw)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    s["kv"] = {}
    for name in ("k", "v"):
        x = s[name]
        x = x * torch.exp(spread * torch.randn(x.shape[:3], generator=g, device=dev))[..., None]
        codes, scale = (t.to(dev) for t in _quantise(x, kind))
        if layout != "hnd":     # the layout of the values
            codes, scale = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (codes, scale))
        s[name + "_pages"], s["kv"][name + "_scale"] = codes, scale
        s[name] = _values(codes, scale)
    return s


def _attend(s, **kw):
    from hy_mt_rs_b200 import paged
    return paged.attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos"], max(s["new"] + [0]),
                           slot=s["slot"], **s["kv"], **kw)


def _close(got, s, rel=5e-6):
    """test_gpu_paged's bound, and one for values that are small where others of
    their row are not (a code of 0 is common): a block's weights times scales are
    f16 pairs in the unit of its largest one, so one is off by 2^-25 of that; over 32
    positions (chunks: a tile of 128) that is 2^-18 of the block's sum of weight
    times the largest value of each row at most."""
    import torch
    from hy_mt_rs_b200 import quant
    ref, tol = _reference(s)
    heads, dim = s["q"].shape[1:]
    group = heads // s["k"].shape[1]
    for i, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        a = s["starts"][i]
        held = s["table"][s["slots"][i], :-(-(n + c) // s["page"])].long()
        for h in range(heads if n else 0):
            k, v = (s[x][held, h // group].double().reshape(-1, dim)[:n + c] for x in ("k", "v"))
            x = s["q"][a:a + n, h].double() @ k.T / math.sqrt(dim)
            hide = torch.arange(n + c, device=x.device)[None] > torch.arange(c, n + c, device=x.device)[:, None]
            p = torch.softmax(x.masked_fill(hide, -math.inf), -1)
            tol[a:a + n, h] += 2.0 ** -18 * (p @ v.abs().amax(-1))[:, None]
    assert torch.isfinite(got).all()
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), float((err / tol.clamp(min=1e-30)).max())
    assert float(err.norm() / ref.norm()) <= rel
    assert quant.device_status() == 0


# ------------------------------------------------------------------- append
def _append_inputs(dev, new, ctx, heads, kvh, dim, page, seed=0, positions=600):
    import torch
    g = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *n: torch.randn(*n, generator=g, device=dev)  # noqa: E731
    t = sum(new)
    s = _make(dev, new, ctx, heads, kvh, dim, page, False, seed=seed)
    angle = torch.arange(positions, device=dev)[:, None] * 10000.0 ** (-torch.arange(dim // 2, device=dev) / (dim // 2))
    s.update(q=randn(t, heads, dim), new_k=randn(t, kvh, dim) * 3, new_v=randn(t, kvh, dim), cos=angle.cos(), sin=angle.sin(),
             q_norm=1 + 0.1 * randn(dim), k_norm=1 + 0.1 * randn(dim))
    return s


def _append(s, k_pages, v_pages, norms=True, first=False, **scales):
    from hy_mt_rs_b200 import paged
    w = (s["q_norm"], s["k_norm"]) if norms else (None, None)
    return paged.rope_append(s["q"], s["new_k"], s["new_v"], k_pages, v_pages, s["table"], s["row_start"], s["pos"], s["cos"],
                             s["sin"], *w, 1e-5, first, **scales)


def _exact_keys(s, t, p, norms, first):
    """Row t's keys at position p in 64 bits, up to each head's norm."""
    import torch
    x, w = s["new_k"][t].double(), s["k_norm"].double() if norms else 1.0
    a, b = (x * w if first else x).chunk(2, -1)
    c, n = s["cos"][p].double(), s["sin"][p].double()
    y = torch.cat([a * c - b * n, a * n + b * c], -1)
    return (y if first else y * w).cpu()


def _pages8(dev, like, kind, layout="hnd"):
    """Empty 8-bit pages of a shape: codes 3 and scales -1, to see what is written."""
    import torch
    out = []
    for _ in range(2):
        codes = torch.full(like.shape, 3, dtype=torch.uint8, device=dev)
        scale = torch.full(like.shape[:3], -1.0, device=dev)
        if layout != "hnd":
            codes, scale = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (codes, scale))
        out += [codes.view(_types()[kind][0]), scale]
    return out[0], out[2], dict(k_scale=out[1], v_scale=out[3])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("norms,first", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("heads,kvh,dim,page", [(16, 4, 128, 64), (8, 8, 64, 16), (6, 2, 80, 7), (3, 1, 6, 5), (4, 2, 256, 32)])
def test_append_matches_the_f32_cache(cuda, heads, kvh, dim, page, norms, first, layout, kind):
    """Queries bit for bit; scales those of the f32 cache's rows, codes those of the rows
    in 64 bits; nothing else written."""
    import torch
    from hy_mt_rs_b200 import quant
    s = _append_inputs(cuda, [1, 0, 37, 2], [0, 9, 63, 130], heads, kvh, dim, page, seed=dim)
    s["new_v"][3] = 0                    # a row of zeros
    s["new_v"][5, :, 1] = 1e30           # one large value
    s["new_k"][7] *= 1e-30
    k32, v32 = (torch.full_like(s[n], 777.0) for n in ("k", "v"))
    q32 = _append(s, k32, v32, norms, first)
    k8, v8, scales = _pages8(cuda, k32, kind, layout)
    q8 = _append(s, k8, v8, norms, first, **scales)
    assert torch.equal(q8, q32)
    exact = k32.double().cpu()
    for i, n in enumerate(s["new"]):
        for j in range(n):
            p, t = s["ctx"][i] + j, s["starts"][i] + j
            exact[int(s["table"][s["slots"][i], p // page]), :, p % page] = _exact_keys(s, t, p, norms, first)
    for x, y, codes, scale in ((k32, exact, k8, scales["k_scale"]), (v32, None, v8, scales["v_scale"])):
        want, want_scale = _quantise(x, kind, y)
        written = (x != 777.0).any(-1).cpu() | (x == 0).all(-1).cpu()
        assert torch.equal(scale.cpu()[written], want_scale[written])
        assert torch.equal(codes.view(torch.uint8).cpu()[written], want.view(torch.uint8)[written])
        assert (codes.view(torch.uint8).cpu()[~written] == 3).all() and (scale.cpu()[~written] == -1).all()
    assert int((scales["k_scale"] != -1).sum()) == sum(s["new"]) * kvh
    assert quant.device_status() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,tokens", [(128, 40), (128, 4000), (64, 4000), (80, 40)])
def test_append_next_to_borders_between_codes(cuda, dim, tokens, kind):
    """Values a few f32 steps from a border between two codes fall on their own side;
    keys too, which f32 arithmetic moves by more than that."""
    import torch
    s = _append_inputs(cuda, [tokens], [0], 2, 2, dim, 64, seed=dim + tokens, positions=tokens)
    g = torch.Generator(device=cuda).manual_seed(4)
    top = 1 + torch.rand(tokens, 2, 1, generator=g, device=cuda, dtype=torch.float64)
    if kind == "i8":
        border = torch.randint(-127, 127, (tokens, 2, dim), generator=g, device=cuda) + 0.5
    else:
        codes = torch.randint(0, 126, (tokens, 2, dim), generator=g, device=cuda).to(torch.uint8)
        up = [c.view(torch.float8_e4m3fn).double() for c in (codes, codes + 1)]
        border = (up[0] + up[1]) / 2 * (2 * torch.randint(0, 2, codes.shape, generator=g, device=cuda) - 1)
    x = (border * top / _types()[kind][1]).float()
    x = x.view(torch.int32).add(torch.randint(-2, 3, x.shape, generator=g, device=cuda, dtype=torch.int32)).view(torch.float32)
    x[..., 5] = top[..., 0].float()
    s["new_v"] = x
    # keys that the rotation takes next to borders
    c, n = (s[t][:, None].double() for t in ("cos", "sin"))
    a, b = (border * top / _types()[kind][1]).chunk(2, -1)
    s["new_k"] = torch.cat([a * c + b * n, b * c - a * n], -1).float()
    k8, v8, scales = _pages8(cuda, s["k"], kind)
    k32, v32 = (torch.full_like(s[t], 777.0) for t in ("k", "v"))
    _append(s, k32, v32, False)
    _append(s, k8, v8, False, **scales)
    pages = s["table"][0, :-(-tokens // 64)].long()
    rows = lambda t: t[pages].transpose(1, 2).reshape(-1, 2, *t.shape[3:])[:tokens].cpu()  # noqa: E731
    c, n, k = (t.cpu() for t in (c, n, s["new_k"].double()))
    a, b = k.chunk(2, -1)
    exact = torch.cat([a * c - b * n, a * n + b * c], -1)
    off = 0
    for x, y, codes, scale in ((rows(k32), exact, k8, "k_scale"), (rows(v32), None, v8, "v_scale")):
        want, want_scale = _quantise(x, kind, y)
        assert torch.equal(rows(scales[scale]), want_scale)
        assert torch.equal(rows(codes.view(torch.uint8)), want.view(torch.uint8))
        y = x * (_types()[kind][1] / x.abs().amax(-1))[..., None]   # f32 all the way takes the wrong side of some
        off += int(((y.round() if kind == "i8" else y.to(want.dtype).float()) != want.float()).sum())
    assert off > 0


@pytest.mark.parametrize("kind", [*KINDS, "f16", "f32"])
@pytest.mark.parametrize("heads,kvh,dim,first", [(16, 4, 128, False), (14, 2, 64, True), (3, 3, 64, False), (96, 16, 128, True), (104, 13, 128, False)])
def test_append_of_many_rows(cuda, heads, kvh, dim, first, kind):
    """Rows that come by bulk copies, rows that cannot (4 bytes off) and, the last
    ones, rows too long for it: the same, a call's few rows as its many; rows behind the
    last sequence, and behind the tables, are left; in place too."""
    import torch
    from hy_mt_rs_b200 import quant
    new, ctx = [300, 1, 0, 150], [17, 40, 3, 0]
    s = _append_inputs(cuda, new, ctx, heads, kvh, dim, 32, seed=heads)
    t = sum(new)
    pad = lambda x: torch.cat([x, torch.full_like(x[:5], math.nan)])  # noqa: E731
    s["q"], s["new_k"], s["new_v"] = (pad(s[n]) for n in ("q", "new_k", "new_v"))

    def run(off, lo=0, hi=len(new), out=None):
        c = dict(s)
        for n in ("q", "new_k", "new_v"):
            x = torch.empty(s[n].numel() + off, device=cuda)[off:].view(s[n].shape)
            c[n] = x.copy_(s[n])
        if kind in KINDS:
            k, v, scales = _pages8(cuda, s["k"], kind)
        else:
            k, v = (torch.full(s["k"].shape, 7.0, dtype=torch.float16 if kind == "f16" else torch.float32, device=cuda) for _ in range(2))
            scales = {}
        q = torch.full_like(c["q"], 7.0) if out is None else c["q"]
        if lo or hi < len(new):  # these sequences' rows alone
            a, b = s["starts"][lo], s["starts"][hi] if hi < len(new) else t
            c.update({n: c[n][a:b] for n in ("q", "new_k", "new_v")}, table=s["table"][s["slots"][lo:hi]].contiguous(),
                     row_start=s["row_start"][lo:hi + 1] - a, pos=s["pos"][lo:hi])
            q = q[a:b]
        _append(c, k, v, True, first, out=q, **scales)
        return [q, *(x.view(torch.uint8) for x in (k, v)), *scales.values()]

    many, off, inplace = run(0), run(1), run(0, out=True)
    assert (many[0][t:] == 7.0).all() and inplace[0][t:].isnan().all()
    assert torch.equal(inplace[0][:t], many[0][:t])
    for a, b in zip(many, off):
        assert torch.equal(a, b)
    few = run(0, 3, 4)
    assert torch.equal(few[0], many[0][s["starts"][3]:t])
    held = s["table"][s["slots"][3], :-(-150 // 32)].long()
    for a, b in zip(many[1:], few[1:]):
        assert torch.equal(a[held], b[held])
    assert quant.device_status() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_append_of_many_rows_captured_and_replayed(cuda, kind):
    """Beside another stream's call of its own, and with rows that are not finite."""
    import torch
    s, o = (_append_inputs(cuda, [500, 40], [3, 30], 16, 4, 128, 32, seed=i, positions=600) for i in (1, 2))
    out = [torch.zeros_like(s["q"]) for _ in range(3)]
    pages = [_pages8(cuda, s["k"], kind) for _ in range(3)]
    calls = [lambda i=i, c=c: _append(c, *pages[i][:2], out=out[i], **pages[i][2]) for i, c in enumerate((s, o, s))]
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        calls[0]()
    for turn in range(2):
        s["q"].normal_()
        s["new_v"].normal_()
        if turn:
            s["new_k"][7, 1, 3], s["new_v"][450, 0, 0] = math.inf, math.nan
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(other):
            calls[1]()
        torch.cuda.synchronize()
        calls[2]()
        both = [[out[i], *(t.view(torch.uint8) for t in pages[i][:2]), *pages[i][2].values()] for i in (0, 2)]
        for a, b in zip(*both):
            assert torch.equal(a.nan_to_num(-7.0), b.nan_to_num(-7.0)) if a.is_floating_point() else torch.equal(a, b)
        for name in ("k_scale", "v_scale"):
            assert int(pages[0][2][name].isnan().sum()) == turn


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [128, 64, 80])
def test_append_rows_that_are_not_finite(cuda, dim, kind):
    """Codes 0 and a NaN scale; other rows as they would be."""
    import torch
    s = _append_inputs(cuda, [4], [3], 4, 2, dim, 16, seed=1)
    clean = [t.clone() for t in (s["new_k"], s["new_v"])]
    results = []
    for bad in (False, True):
        if bad:
            s["new_k"][1, 0, 3], s["new_v"][2, 1, dim - 1], s["new_v"][0, 0, 0] = math.inf, math.nan, -math.inf
        k8, v8, scales = _pages8(cuda, s["k"], kind)
        _append(s, k8, v8, False, **scales)
        page = int(s["table"][0, 0])
        rows = [t[page].cpu() for t in (k8.view(torch.uint8), scales["k_scale"], v8.view(torch.uint8), scales["v_scale"])]
        results.append(rows)
    s["new_k"], s["new_v"] = clean
    want, got = results
    for codes, scale, spoiled in ((0, 1, [(0, 4)]), (2, 3, [(1, 5), (0, 3)])):
        for h, p in spoiled:
            assert math.isnan(float(got[scale][h, p])) and int(got[codes][h, p].sum()) == 0
            want[scale][h, p], want[codes][h, p] = 0, 0
            got[scale][h, p] = 0
        assert torch.equal(got[codes], want[codes]) and torch.equal(got[scale], want[scale])


# ------------------------------------------------------------------- gather
@pytest.mark.parametrize("kind", ["f32", "f16", "i8", "f8"])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 7), (80, 64), (17, 5)])
def test_gather(cuda, dim, page, layout, f16, kind):
    """The values of the pages, rounded once; rows of no sequence left alone; given
    outputs with a stride."""
    import torch
    from hy_mt_rs_b200 import paged, quant
    new, ctx, kvh = [3, 0, 40, 1], [0, 5, 31, 200], 3
    if kind in KINDS:
        s = _make8(cuda, new, ctx, 6, kvh, dim, page, kind, layout=layout, slots=True)
    else:
        s = _make(cuda, new, ctx, 6, kvh, dim, page, kind == "f16", layout=layout, slots=True)
        s.update(kv={}, k_pages=s["k"], v_pages=s["v"])
    dtype, tokens = torch.float16 if f16 else torch.float32, sum(new) + 2
    wide = torch.full((tokens, 2 * kvh + 1, dim), 9.0, dtype=dtype, device=cuda)
    k, v = paged.gather(s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos"], tokens, slot=s["slot"], dtype=dtype,
                        k_out=wide[:, :kvh], v_out=torch.full((tokens, kvh, dim), 9.0, dtype=dtype, device=cuda), **s["kv"])
    assert (wide[:, kvh:] == 9).all() and (k[-2:] == 9).all() and (v[-2:] == 9).all()
    row = 0
    for i, (n, c) in enumerate(zip(new, ctx)):
        for p in range(c, c + n):
            at = int(s["table"][s["slots"][i], p // page])
            for got, want in ((k, s["k"]), (v, s["v"])):
                want = want[at, :, p % page]
                # code * scale is one f32 product; then the output's rounding
                assert torch.equal(got[row], want.float().to(dtype))
            row += 1
    again = paged.gather(s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos"], sum(new), slot=s["slot"], dtype=dtype,
                         **s["kv"])
    assert torch.equal(again[0], k[:-2]) and torch.equal(again[1], v[:-2])
    assert quant.device_status() == 0


# ---------------------------------------------------------------- attention
SHAPES = [(16, 4, 128), (32, 8, 128), (16, 2, 128), (8, 8, 64), (12, 4, 64), (20, 5, 128), (6, 2, 80), (3, 1, 32), (16, 1, 128),
          (16, 1, 64), (4, 2, 256), (5, 5, 17)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,dim", SHAPES)
def test_attention_shapes(cuda, heads, kvh, dim, kind):
    """Ragged batch: empty, one-token and chunked sequences, contexts of zero,
    inside a page, at its end."""
    s = _make8(cuda, [1, 0, 5, 37, 1, 16], [0, 40, 63, 100, 127, 0], heads, kvh, dim, 16, kind, seed=dim + heads)
    _close(_attend(s), s)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [1, 7, 8, 16, 32, 48, 64, 100, 128, 256])
def test_attention_page_sizes(cuda, page, dim, kind):
    s = _make8(cuda, [1, 130, 3], [517, 71, 64], 8, 2, dim, page, kind, seed=page)
    _close(_attend(s), s)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("ctx", [0, 1, 15, 31, 32, 33, 127, 128, 129, 1000, 5000])
def test_attention_single_token(cuda, ctx, kind):
    s = _make8(cuda, [1], [ctx], 16, 4, 128, 64, kind, seed=ctx)
    _close(_attend(s), s)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,ctx", [([300], [0]), ([129], [1000]), ([31, 32, 33], [5, 96, 97]), ([64, 1, 257], [64, 900, 3]),
                                     ([2, 3, 4, 8], [700, 31, 64, 513]), ([1] * 70, list(range(0, 1400, 20)))])
def test_attention_chunks(cuda, new, ctx, dim, kind):
    s = _make8(cuda, new, ctx, 16, 4, dim, 32, kind, seed=sum(new))
    _close(_attend(s), s)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("new,ctx", [([1, 4, 1], [70, 600, 0]), ([90, 1], [333, 20])])
def test_attention_layouts_and_slots(cuda, new, ctx, layout, kind):
    s = _make8(cuda, new, ctx, 16, 4, 128, 32, kind, layout=layout, slots=True, seed=7)
    _close(_attend(s), s)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,ctx", [([1, 3], [900, 400]), ([200], [500])])
def test_scales_far_apart(cuda, new, ctx, kind):
    """Neighbouring positions of V whose scales differ by up to 2^60: every
    position that counts in an output keeps its bits.  (Outputs are then sums of
    very different sizes: only the element-wise bound holds.)"""
    import torch
    s = _make8(cuda, new, ctx, 16, 4, 128, 16, kind, seed=11)
    scale = s["kv"]["v_scale"]
    g = torch.Generator(device=cuda).manual_seed(3)
    scale *= torch.exp2(torch.randint(-30, 31, scale.shape, generator=g, device=cuda).float())
    s["v"] = _values(s["v_pages"], scale)
    _close(_attend(s), s)
    # weights far from each other as well, the large values behind the small weights
    s["q"] *= 4
    _close(_attend(s), s, rel=2e-5)
    scale.zero_()                       # a cache of zeros
    assert (_attend(s) == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 48), (80, 16)])
@pytest.mark.parametrize("new,ctx", [([1, 5], [300, 61]), ([90], [400])])
def test_positions_out_of_sight_do_not_count(cuda, new, ctx, dim, page, kind):
    """NaN scales and any codes past a token's position, or in pages of nobody:
    the same bits."""
    import torch
    s = _make8(cuda, new, ctx, 8, 2, dim, page, kind, seed=5)
    used = torch.zeros(s["k"].shape[0], page, dtype=torch.bool)
    for i, (n, c) in enumerate(zip(new, ctx)):
        for p in range(n + c):
            used[int(s["table"][i, p // page]), p % page] = True
    free = ~used.to(cuda)[:, None].expand(s["k"].shape[:3])
    want = _attend(s)
    for fill in NAN_CODES:
        for name in ("k", "v"):
            s[name + "_pages"].view(torch.uint8)[free] = fill
            s["kv"][name + "_scale"][free] = math.nan if fill == 0x7f else math.inf
        assert torch.equal(_attend(s), want)
    # the last new token's own row: only that token sees it
    last, n, c = s["starts"][-1] - 1, new[-1], ctx[-1]
    page_of, row = int(s["table"][len(new) - 1, (n + c - 1) // page]), (n + c - 1) % page
    if n > 1:
        s["kv"]["v_scale"][page_of, 0, row] = math.nan
        got = _attend(s)
        assert torch.isnan(got[last, :4]).all() and torch.isfinite(got[last, 4:]).all()
        # (a tile's unit may change with the scales it holds: the same values, other roundings)
        err, size = (got[:last] - want[:last]).abs(), want[:last].abs().amax()
        assert float((err / size).amax()) <= 2.0 ** -18
        s["kv"]["k_scale"][page_of, 1, row] = math.nan
        got = _attend(s)
        assert torch.isnan(got[last]).all() and torch.isfinite(got[:last]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_all_codes(cuda, kind):
    """Every code of the type, the two without a value among them, in K and V."""
    import torch
    s = _make8(cuda, [1, 40], [255, 215], 8, 2, 128, 32, kind, seed=2)
    for name in ("k", "v"):
        codes = torch.arange(256, dtype=torch.uint8, device=cuda)
        bits = s[name + "_pages"].view(torch.uint8)
        for j in range(8):
            bits[:, 0, 4 * j:4 * j + 4] = codes.view(-1, 128).repeat(2, 1)[:4].roll(j, 1)
        s["kv"][name + "_scale"].mul_(0.05)
        s[name] = _values(s[name + "_pages"], s["kv"][name + "_scale"])
    _close(_attend(s), s)


@pytest.mark.parametrize("kind", KINDS)
def test_captured_and_replayed(cuda, kind):
    """A captured append and attention, replayed with other inputs and lengths."""
    import torch
    from hy_mt_rs_b200 import paged
    s = _make8(cuda, [1, 6, 1], [30, 0, 700], 16, 4, 128, 32, kind, seed=9)
    a = _append_inputs(cuda, [1, 6, 1], [30, 0, 700], 16, 4, 128, 32, seed=9, positions=1000)
    a.update(table=s["table"], row_start=s["row_start"], pos=s["pos"])
    ws, out = paged.attention_workspace(16, 128, cuda), torch.empty_like(s["q"])

    def step():
        s["q"] = _append(a, s["k_pages"], s["v_pages"], **s["kv"])
        _attend(s, out=out, workspace=ws)

    step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        step()
        with torch.cuda.graph(graph, stream=stream):
            step()
    torch.cuda.current_stream().wait_stream(stream)
    for i in range(3):
        a["q"].normal_()
        a["new_k"].normal_()
        s["pos"].copy_(_int([29 - i, i, 690 + i], cuda))
        out.zero_()
        graph.replay()
        s["ctx"] = [29 - i, i, 690 + i]
        s["k"], s["v"] = (_values(s[n + "_pages"], s["kv"][n + "_scale"]) for n in ("k", "v"))
        _close(out, s)
