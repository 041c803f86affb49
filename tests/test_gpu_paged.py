"""GPU parity of the paged-cache operators: RoPE + norm + append against
hyq_rope_qk (bit for bit) and the formula, attention over pages against a
64-bit softmax, page handling against a host model of the tables."""
import ctypes as C
import math
import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _int(v, dev):
    import torch
    return torch.tensor(v, dtype=torch.int32).to(dev)


def _make(dev, new, ctx, heads, kvh, dim, page, kv16, layout="hnd", seed=0, extra=3, fill=None, slots=False):
    """Random pages, shuffled tables and queries.  fill: the value of every
    cache element outside the sequences' own positions."""
    import torch
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    counts = [-(-(a + b) // page) for a, b in zip(new, ctx)]
    pages = sum(counts) + extra
    held = list(range(pages))
    rng.shuffle(held)
    dtype = torch.float16 if kv16 else torch.float32
    shape = (pages, kvh, page, dim) if layout == "hnd" else (pages, page, kvh, dim)
    k, v = (torch.randn(*shape, generator=g, device=dev).to(dtype) for _ in range(2))
    if layout != "hnd":
        k, v = k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)
    n_slots = len(new) + (4 if slots else 0)
    slot = rng.sample(range(n_slots), len(new)) if slots else list(range(len(new)))
    table = torch.full((n_slots, max(counts + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    used = torch.zeros(pages, page, dtype=torch.bool)
    for i, c in enumerate(counts):
        mine = held[at:at + c]
        at += c
        table[slot[i], :c] = torch.tensor(mine, dtype=torch.int32)
        for p in range(new[i] + ctx[i]):
            used[mine[p // page], p % page] = True
    if fill is not None:
        mask = ~used.to(dev)[:, None, :, None].expand(k.shape)
        k[mask] = fill
        v[mask] = fill
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = torch.randn(max(starts[-1], 1), heads, dim, generator=g, device=dev)[:starts[-1]]
    q = q * (1 + torch.arange(heads, device=dev) % 3)[:, None]
    return dict(q=q, k=k, v=v, table=table.to(dev), row_start=_int(starts, dev), pos=_int(ctx, dev),
                slot=_int(slot, dev) if slots else None, new=new, ctx=ctx, starts=starts, page=page, slots=slot)


def _attend(s, out=None, workspace=None, max_len=None):
    from hy_mt_rs_b200 import paged
    return paged.attention(s["q"], s["k"], s["v"], s["table"], s["row_start"], s["pos"], max(s["new"] + [0]),
                           max_len, slot=s["slot"], out=out, workspace=workspace)


def _reference(s):
    """The output in 64 bits and an element-wise bound of its rounding error.

    Every product carries its operands to 21 bits at least and sums in f32, so
    a score is off by at most d = (2^-21 + dim 2^-24) sum|q k| / sqrt(dim); a
    weight by the factor e^(2 d) at most, and the output by that share of
    sum p |v|, plus the roundings of the weights and sums (2^-18 of it)."""
    import torch
    q = s["q"].double()
    heads, dim = q.shape[1:]
    group = heads // s["k"].shape[1]
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for i, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        a = s["starts"][i]
        if n == 0:
            continue
        held = s["table"][s["slots"][i], :-(-(n + c) // s["page"])].long()
        for h in range(heads):
            k = s["k"][held, h // group].double().reshape(-1, dim)[:n + c]
            v = s["v"][held, h // group].double().reshape(-1, dim)[:n + c]
            x = q[a:a + n, h] @ k.T / math.sqrt(dim)
            hide = torch.arange(n + c, device=x.device)[None] > torch.arange(c, n + c, device=x.device)[:, None]
            p = torch.softmax(x.masked_fill(hide, -math.inf), -1)
            out[a:a + n, h] = p @ v
            size = (q[a:a + n, h].abs() @ k.abs().T / math.sqrt(dim)).masked_fill(hide, 0).amax(-1, keepdim=True)
            tol[a:a + n, h] = (p @ v.abs()) * (2 * (2.0 ** -21 + dim * 2.0 ** -24) * size + 2.0 ** -18)
    return out, tol


def _close(got, s, rel=5e-6):
    """Element-wise within the bound; 2-norm within 5e-6 (operands at 21 bits,
    scores up to about 20 in magnitude)."""
    import torch
    from hy_mt_rs_b200 import quant
    ref, tol = _reference(s)
    assert torch.isfinite(got).all()
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), float((err / tol.clamp(min=1e-30)).max())
    assert float(err.norm() / ref.norm()) <= rel
    assert quant.device_status() == 0


SHAPES = [
    # heads, kv_heads, dim
    (16, 4, 128), (32, 8, 128), (16, 2, 128), (8, 8, 64), (12, 4, 64), (20, 5, 128), (6, 2, 80), (3, 1, 32),
    (16, 1, 128), (4, 2, 256), (5, 5, 17), (2, 1, 96),
]


@pytest.mark.parametrize("kv16", [True, False])
@pytest.mark.parametrize("heads,kvh,dim", SHAPES)
def test_attention_shapes(cuda, heads, kvh, dim, kv16):
    """Ragged batch: empty, one-token and chunked sequences, contexts of zero,
    inside a page, at its end."""
    s = _make(cuda, [1, 0, 5, 37, 1, 16], [0, 40, 63, 100, 127, 0], heads, kvh, dim, 16, kv16, seed=dim + heads)
    _close(_attend(s), s)


@pytest.mark.parametrize("kv16", [True, False])
@pytest.mark.parametrize("page", [1, 7, 8, 16, 32, 48, 64, 100, 128, 256])
def test_attention_page_sizes(cuda, page, kv16):
    s = _make(cuda, [1, 130, 3], [517, 71, 64], 8, 2, 128, page, kv16, seed=page)
    _close(_attend(s), s)


@pytest.mark.parametrize("kv16", [True, False])
@pytest.mark.parametrize("ctx", [0, 1, 15, 16, 63, 64, 127, 128, 129, 1000, 5000])
def test_attention_single_token(cuda, ctx, kv16):
    s = _make(cuda, [1], [ctx], 16, 4, 128, 64, kv16, seed=ctx)
    _close(_attend(s), s)


@pytest.mark.parametrize("kv16", [True, False])
@pytest.mark.parametrize("new,ctx", [([300], [0]), ([129], [1000]), ([31, 32, 33], [5, 96, 97]), ([64, 1, 257], [64, 900, 3]),
                                     ([2, 3, 4, 8], [700, 31, 64, 513])])
def test_attention_chunks(cuda, new, ctx, kv16):
    s = _make(cuda, new, ctx, 16, 4, 128, 32, kv16, seed=sum(new))
    _close(_attend(s), s)


@pytest.mark.parametrize("kv16", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_many_sequences(cuda, dim, kv16):
    rng = random.Random(dim)
    new = [rng.choice([1, 1, 1, 1, 2, 0, 40]) for _ in range(150)]
    ctx = [rng.randrange(0, 400) for _ in new]
    s = _make(cuda, new, ctx, 8, 2, dim, 16, kv16, seed=dim, slots=True)
    _close(_attend(s), s)


@pytest.mark.parametrize("kv16", [True, False])
def test_attention_layout_strides_slots(cuda, kv16):
    """[pages, page_size, kv_heads, dim] pages, query and output rows inside a
    wider tensor, table rows by slot, and an output row that no sequence has."""
    import torch
    from hy_mt_rs_b200 import paged
    s = _make(cuda, [1, 70, 2], [200, 30, 95], 8, 4, 128, 32, kv16, layout="nhd", slots=True, seed=5)
    wide = torch.randn(74, 8 * 128 + 64, device=cuda)
    q = wide.as_strided((74, 8, 128), (8 * 128 + 64, 128, 1))
    q[:73].copy_(s["q"])
    buf = torch.full((74, 8 * 128 + 32), 7.0, device=cuda)
    out = buf.as_strided((74, 8, 128), (8 * 128 + 32, 128, 1))
    paged.attention(q, s["k"], s["v"], s["table"], s["row_start"], s["pos"], 70, slot=s["slot"], out=out)
    _close(out[:73], s)
    assert (buf[73] == 7).all() and (buf[:, 8 * 128:] == 7).all()


@pytest.mark.parametrize("offset", [1, 2, 4])
def test_attention_unaligned(cuda, offset):
    """Pools and queries that start off a 16-byte boundary."""
    import torch
    s = _make(cuda, [1, 40], [130, 20], 8, 2, 128, 16, True, seed=offset)
    for n in ("k", "v"):
        flat = torch.empty(s[n].numel() + 8, dtype=torch.float16, device=cuda)
        t = flat[offset:offset + s[n].numel()].view(s[n].shape)
        t.copy_(s[n])
        s[n] = t
    flat = torch.empty(s["q"].numel() + 8, device=cuda)
    t = flat[1:1 + s["q"].numel()].view(s["q"].shape)
    s["q"] = t.copy_(s["q"])
    _close(_attend(s), s)


@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -65504.0])
@pytest.mark.parametrize("kv16", [True, False])
@pytest.mark.parametrize("dim", [128, 40])
def test_attention_ignores_what_is_not_seen(cuda, dim, kv16, fill):
    """Free pages and page tails hold anything."""
    s = _make(cuda, [1, 3, 150, 1], [100, 61, 77, 0], 8, 2, dim, 64, kv16, fill=fill, seed=3)
    got = _attend(s)
    clean = dict(s, k=s["k"].nan_to_num(0, 0, 0), v=s["v"].nan_to_num(0, 0, 0))
    _close(got, clean)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("kv16", [True, False])
@pytest.mark.parametrize("new,ctx,at", [(4, 60, 2), (200, 50, 133), (200, 0, 64)])
def test_attention_later_tokens_do_not_leak(cuda, new, ctx, at, kv16, bad):
    """A non-finite key and value inside the chunk reaches the tokens from its
    position on, and none before it."""
    import torch
    s = _make(cuda, [new], [ctx], 8, 2, 128, 32, kv16, seed=at)
    clean = dict(s, k=s["k"].clone(), v=s["v"].clone())
    p = ctx + at
    page = int(s["table"][0, p // 32])
    s["v"][page, :, p % 32, 5] = bad
    got = _attend(s)
    ref, tol = _reference(clean)
    assert ((got[:at].double() - ref[:at]).abs() <= tol[:at]).all()
    assert not torch.isfinite(got[at:, :, 5]).any()
    rest = [d for d in range(128) if d != 5]
    assert ((got[at:, :, rest].double() - ref[at:, :, rest]).abs() <= tol[at:, :, rest]).all()
    s["v"].copy_(clean["v"])
    s["k"][page, :, p % 32, 7] = float("nan")
    got = _attend(s)
    assert ((got[:at].double() - ref[:at]).abs() <= tol[:at]).all()
    assert got[at:].isnan().all()


@pytest.mark.parametrize("kv16", [True, False])
@pytest.mark.parametrize("scale", [1e-4, 30.0, 3000.0])
def test_attention_query_and_cache_magnitudes(cuda, scale, kv16):
    """Scores from all but equal to one-hot; values far from 1."""
    import torch
    s = _make(cuda, [1, 150, 3], [300, 20, 70], 8, 2, 128, 32, kv16, seed=1)
    s["q"] = s["q"] * scale
    s["v"] *= 100
    got = _attend(s)
    ref, tol = _reference(s)
    assert torch.isfinite(got).all()
    # scores past 1e3 lose their last bits in any f32 product: the bound alone
    assert ((got.double() - ref).abs() <= tol).all()


def test_attention_large_f32_values(cuda):
    """An f32 cache holds values no f16 does."""
    s = _make(cuda, [1, 140, 3], [300, 20, 70], 8, 2, 128, 32, False, seed=2)
    s["q"] = s["q"] * 1e-7
    s["k"] *= 1e7
    s["v"] *= 1e12
    _close(_attend(s), s)


def test_attention_repeats_bit_for_bit(cuda):
    """The same call twice, with one workspace, other calls between, and on
    another stream."""
    import torch
    from hy_mt_rs_b200 import paged
    for kv16 in (True, False):
        s = _make(cuda, [1] * 9 + [100, 4], [3000, 5, 64, 700, 20, 1500, 900, 10, 31, 50, 2000], 16, 4, 128, 64, kv16)
        other = _make(cuda, [1, 33], [4000, 100], 16, 4, 128, 64, kv16)
        ws = paged.attention_workspace(16, 128, cuda)
        first = _attend(s, workspace=ws).clone()
        _attend(other, workspace=ws)
        assert torch.equal(_attend(s, workspace=ws), first)
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            again = _attend(s, workspace=ws)
        stream.synchronize()
        assert torch.equal(again, first)


def test_attention_graph_replay(cuda):
    """Captured once, replayed while positions and tables change in place."""
    import torch
    from hy_mt_rs_b200 import paged
    a = _make(cuda, [1, 1, 1], [10, 300, 77], 16, 4, 128, 16, True, seed=1)
    ws = paged.attention_workspace(16, 128, cuda)
    out = torch.empty_like(a["q"])
    reach = a["table"].shape[1] * 16
    _attend(a, out=out, workspace=ws, max_len=reach)
    g = torch.cuda.CUDAGraph()
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        _attend(a, out=out, workspace=ws, max_len=reach)
    for ctx in ([10, 300, 77], [5, 17, 300], [0, 299, 1]):
        a["ctx"] = ctx
        a["table"][:, :] = a["table"][:, :].clamp(min=0)
        a["pos"].copy_(_int(ctx, cuda))
        g.replay()
        torch.cuda.synchronize()
        _close(out, a)


@pytest.mark.parametrize("dim", [128, 48])
def test_attention_bad_sequences_are_skipped(cuda, dim):
    """Positions past the table, a slot outside it, pages outside the pool:
    the sequence's rows stay as they were or are finite nonsense, the others
    are right and HYQ_DEV_BAD_ARGS is raised.  Every case is caught by the
    kernels' own checks."""
    import torch
    from hy_mt_rs_b200 import quant
    s = _make(cuda, [1, 2, 40], [50, 20, 10], 8, 2, dim, 16, True, slots=True)
    good = _attend(s)
    for change in ("pos", "slot", "page", "negative"):
        t = {k: (v.clone() if isinstance(v, torch.Tensor) else v) for k, v in s.items()}
        if change == "pos":
            t["pos"][1] = t["table"].shape[1] * 16
        elif change == "negative":
            t["pos"][1] = -1
        elif change == "slot":
            t["slot"][1] = 99
        else:
            t["table"][t["slots"][1], 0] = t["k"].shape[0]
        out = torch.zeros_like(good)
        _attend(t, out=out)
        assert quant.device_status() == 8      # HYQ_DEV_BAD_ARGS, cleared by the read
        assert torch.equal(out[:1], good[:1]) and torch.equal(out[3:], good[3:])
    assert quant.device_status() == 0


def test_offsets_past_32_bits(cuda):
    """A pool of more than 2^31 elements: append to and attend over its last
    pages."""
    import torch
    from hy_mt_rs_b200 import paged, quant
    pages, kvh, page, dim, heads = 66000, 4, 64, 128, 16
    k, v = (torch.empty(pages, kvh, page, dim, dtype=torch.float16, device=cuda) for _ in range(2))
    new, ctx = [1, 70, 3], [200, 3, 64]
    table = torch.zeros(3, 4, dtype=torch.int32)
    last = list(range(pages - 9, pages))
    for i in range(3):
        n = -(-(new[i] + ctx[i]) // page)
        table[i, :n] = torch.tensor([last.pop() for _ in range(n)], dtype=torch.int32)
    for p in range(pages - 9, pages):
        k[p].normal_()
        v[p].normal_()
    starts = [0, 1, 71, 74]
    s = dict(q=torch.randn(74, heads, dim, device=cuda), k=k, v=v, table=table.to(cuda), row_start=_int(starts, cuda),
             pos=_int(ctx, cuda), slot=None, new=new, ctx=ctx, starts=starts, page=page, slots=[0, 1, 2])
    cos, sin = torch.ones(256, 64, device=cuda), torch.zeros(256, 64, device=cuda)
    kn, vn = torch.randn(74, kvh, dim, device=cuda), torch.randn(74, kvh, dim, device=cuda)
    paged.rope_append(s["q"], kn, vn, k, v, s["table"], s["row_start"], s["pos"], cos, sin)
    p = int(s["table"][0, 200 // 64])
    assert torch.equal(k[p, :, 200 % 64], kn[0].half()) and torch.equal(v[p, :, 200 % 64], vn[0].half())
    got = _attend(s)
    sub = dict(s, k=k[pages - 9:], v=v[pages - 9:], table=(s["table"] - (pages - 9)).clamp(min=0))
    _close(got, sub)
    assert quant.device_status() == 0


# ------------------------------------------------------------------- append
def _p(t):
    return C.c_void_p(t.data_ptr())


@pytest.mark.parametrize("norm_first", [False, True])
@pytest.mark.parametrize("kv16", [True, False])
@pytest.mark.parametrize("heads,kvh,dim,page,layout", [(16, 4, 128, 64, "hnd"), (8, 8, 64, 16, "nhd"), (6, 2, 80, 7, "hnd"),
                                                       (4, 1, 256, 32, "hnd"), (3, 3, 34, 16, "nhd"), (2, 1, 32, 8, "hnd")])
def test_append_equals_rope_qk(cuda, heads, kvh, dim, page, layout, kv16, norm_first):
    """Bit for bit what hyq_rope_qk leaves in a contiguous cache; nothing else
    in the pages changes; k and v stay as they were."""
    import torch
    from hy_mt_rs_b200 import paged, quant
    from hy_mt_rs_b200._native import check, lib
    new, ctx = [1, 0, 30, 7], [page - 1, 4, 3 * page, 0]
    s = _make(cuda, new, ctx, heads, kvh, dim, page, kv16, layout, seed=dim, slots=True)
    t, positions = sum(new), 3 * page + 64
    g = torch.Generator(device=cuda).manual_seed(1)
    # q, k and v as columns of one product
    width = (heads + 2 * kvh) * dim
    qkv = torch.randn(t, width + 8, generator=g, device=cuda)
    part = lambda a, n: qkv.as_strided((t, n, dim), (width + 8, dim, 1), a * dim)  # noqa: E731
    q, k, v = part(0, heads), part(heads, kvh), part(heads + kvh, kvh)
    cos, sin = torch.rand(positions, dim // 2, generator=g, device=cuda), torch.rand(positions, dim // 2, generator=g, device=cuda)
    wq, wk = torch.randn(dim, generator=g, device=cuda), torch.randn(dim, generator=g, device=cuda)
    before = qkv.clone()
    k0, v0 = s["k"].clone(), s["v"].clone()
    out = paged.rope_append(q, k, v, s["k"], s["v"], s["table"], s["row_start"], s["pos"], cos, sin, wq, wk, 1e-5,
                            norm_first, slot=s["slot"])
    assert torch.equal(qkv, before)
    rope = lib.hyq_rope_qk_kv16 if kv16 else lib.hyq_rope_qk
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    for i, (n, c) in enumerate(zip(new, ctx)):
        if n == 0:
            continue
        a = s["starts"][i]
        qi, ki, vi = (x[a:a + n].contiguous() for x in (q, k, v))
        kc, vc = (torch.zeros(positions, kvh * dim, device=cuda, dtype=s["k"].dtype) for _ in range(2))
        check(rope(_p(qi), _p(ki), _p(vi), heads, kvh, dim, _p(cos), _p(sin), positions, _p(s["pos"][i:]), n, _p(wq), _p(wk),
                   1e-5, int(norm_first), _p(kc), _p(vc), st))
        assert torch.equal(out[a:a + n], qi)
        for j in range(n):
            p = c + j
            page_id = int(s["table"][s["slots"][i], p // page])
            assert torch.equal(s["k"][page_id, :, p % page].reshape(-1), kc[p])
            assert torch.equal(s["v"][page_id, :, p % page].reshape(-1), vc[p])
            k0[page_id, :, p % page] = s["k"][page_id, :, p % page]
            v0[page_id, :, p % page] = s["v"][page_id, :, p % page]
    assert torch.equal(k0, s["k"]) and torch.equal(v0, s["v"])
    assert quant.device_status() == 0


@pytest.mark.parametrize("norm_first", [False, True])
def test_append_formula_in_place_without_norms(cuda, norm_first):
    """Against the formula in 64 bits (one rounding per product and sum: 1e-6
    of a head's largest value), q rotated in place; without norms the rotation
    alone."""
    import torch
    from hy_mt_rs_b200 import paged
    s = _make(cuda, [5, 2], [9, 0], 8, 2, 128, 16, False, seed=4)
    g = torch.Generator(device=cuda).manual_seed(2)
    q, k, v = (torch.randn(7, n, 128, generator=g, device=cuda) for n in (8, 2, 2))
    angle = torch.rand(32, 64, generator=g, device=cuda) * 6
    cos, sin = angle.cos(), angle.sin()
    w = torch.rand(128, generator=g, device=cuda) + 0.5
    at = torch.tensor([9, 10, 11, 12, 13, 0, 1], device=cuda)

    def rope(x):
        c, n = cos[at].double()[:, None], sin[at].double()[:, None]
        return torch.cat([x[..., :64] * c - x[..., 64:] * n, x[..., :64] * n + x[..., 64:] * c], -1)

    def norm(x):
        return x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()

    both = (lambda x: rope(norm(x))) if norm_first else (lambda x: norm(rope(x)))
    for norms in (True, False):
        x = q.clone()
        f = both if norms else rope
        got = paged.rope_append(x, k, v, s["k"], s["v"], s["table"], s["row_start"], s["pos"], cos, sin,
                                w if norms else None, w if norms else None, 1e-5, norm_first, out=x)
        assert got.data_ptr() == x.data_ptr()
        ref = f(q.double())
        assert float((x.double() - ref).abs().max()) <= 1e-6 * float(ref.abs().max())
        kr = f(k.double())
        for r, p in enumerate(at.tolist()):
            page = int(s["table"][0 if r < 5 else 1, p // 16])
            assert float((s["k"][page, :, p % 16].double() - kr[r]).abs().max()) <= 1e-6 * float(kr.abs().max())


def test_append_bad_positions_are_skipped(cuda):
    import torch
    from hy_mt_rs_b200 import paged, quant
    s = _make(cuda, [2, 1], [3, 30], 4, 2, 64, 16, True)
    q, k, v = (torch.randn(3, n, 64, device=cuda) for n in (4, 2, 2))
    cos = torch.ones(16, 32, device=cuda)     # tables shorter than sequence 1
    k0 = s["k"].clone()
    out = torch.zeros_like(q)
    paged.rope_append(q, k, v, s["k"], s["v"], s["table"], s["row_start"], s["pos"], cos, cos, out=out)
    assert quant.device_status() == 8
    assert (out[2] == 0).all() and (out[:2] != 0).any()
    page = int(s["table"][1, 1])
    assert torch.equal(s["k"][page], k0[page])


# -------------------------------------------------------------------- pages
class _Model:
    """The tables on the host."""

    def __init__(self, slots, width, pages, page):
        self.table, self.length = [[] for _ in range(slots)], [0] * slots
        self.refs, self.page, self.width, self.pages = [0] * pages, page, width, pages

    def free_pages(self, n):
        return [p for p in range(self.pages) if self.refs[p] == 0][:n]

    def reserve(self, slot, extra):
        need = [-(-(self.length[s] + e) // self.page) - len(self.table[s]) for s, e in zip(slot, extra)]
        got = self.free_pages(sum(need))
        if len(got) < sum(need):
            return sum(need) - len(got)
        for s, e, n in zip(slot, extra, need):
            for _ in range(n):
                self.refs[got[0]] = 1
                self.table[s].append(got.pop(0))
            self.length[s] += e
        return 0

    def free(self, slot):
        for s in slot:
            for p in self.table[s]:
                self.refs[p] -= 1
            self.table[s], self.length[s] = [], 0

    def fork(self, src, dst):
        self.free(dst)
        part = [s for s in src if self.length[s] % self.page]
        got = self.free_pages(len(part))
        if len(got) < len(part):
            return len(part) - len(got), []
        copies = []
        for a, b in zip(src, dst):
            full = self.length[a] // self.page
            self.table[b], self.length[b] = self.table[a][:full], self.length[a]
            for p in self.table[b]:
                self.refs[p] += 1
            if self.length[a] % self.page:
                copies.append((self.table[a][full], got[0]))
                self.refs[got[0]] = 1
                self.table[b].append(got.pop(0))
        return 0, copies

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        high = [p for p in range(live, self.pages) if self.refs[p]]
        low = [p for p in range(live) if not self.refs[p]]
        to = dict(zip(high, low))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return list(to.items())

    def check(self, cache):
        assert cache.refs.tolist() == self.refs
        assert cache.length.tolist() == self.length
        assert cache.table.tolist() == [row + [-1] * (self.width - len(row)) for row in self.table]


@pytest.mark.parametrize("seed,slots,width,pages,page,layers,kv16", [
    (0, 5, 4, 12, 4, 2, True), (1, 12, 30, 150, 16, 1, False), (2, 40, 9, 200, 8, 3, True), (3, 3, 2, 5000, 16, 1, True),
    (4, 300, 12, 9000, 2, 1, False)])
def test_pages_random_operations(cuda, seed, slots, width, pages, page, layers, kv16):
    """A random history of reserve, free, fork and compact against a host
    model, the pool's contents included."""
    import torch
    from hy_mt_rs_b200 import quant
    from hy_mt_rs_b200.paged import PagedCache
    rng = random.Random(seed)
    cache = PagedCache(layers, 2, 8, pages, page, slots, width, cuda, torch.float16 if kv16 else torch.float32)
    g = torch.Generator(device=cuda).manual_seed(seed)
    cache.pool.copy_(torch.randn(cache.pool.shape, generator=g, device=cuda))
    pool = cache.pool.clone()
    host = _Model(slots, width, pages, page)
    for step in range(40):
        op = rng.choice(["reserve", "reserve", "reserve", "free", "fork", "compact"])
        n = rng.randint(1, min(slots, 40 if slots < 100 else slots))
        chosen = rng.sample(range(slots), n)
        if op == "reserve":
            extra = [rng.randint(0, min(2 * page + 3, width * page - host.length[s])) for s in chosen]
            before = [host.length[s] for s in chosen]
            pos = cache.reserve(_int(chosen, cuda), _int(extra, cuda))
            assert cache.shortage.item() == host.reserve(chosen, extra)
            assert pos.tolist() == before
        elif op == "free":
            cache.free(_int(chosen, cuda))
            host.free(chosen)
        elif op == "fork" and slots > 1:
            dst = chosen[:max(1, n // 2)]
            others = [s for s in range(slots) if s not in dst]
            src = [rng.choice(others) for _ in dst]
            cache.fork(_int(src, cuda), _int(dst, cuda))
            short, copies = host.fork(src, dst)
            assert cache.shortage.item() == short
            for a, b in copies:
                pool[:, :, b] = pool[:, :, a]
        else:
            cache.compact()
            for a, b in host.compact():
                pool[:, :, b] = pool[:, :, a]
        host.check(cache)
        assert torch.equal(cache.pool, pool)
    assert quant.device_status() == 0


def test_pages_refuse_bad_slots_on_the_device(cuda):
    """Slots out of range or repeated, growth past the table row, a fork onto
    a source: nothing changes and HYQ_DEV_BAD_ARGS is raised."""
    import torch
    from hy_mt_rs_b200 import quant
    from hy_mt_rs_b200.paged import PagedCache
    cache = PagedCache(1, 1, 8, 16, 4, 4, 3, cuda)
    cache.reserve(_int([0, 1], cuda), _int([5, 12], cuda))
    state = [t.clone() for t in (cache.table, cache.length, cache.refs)]
    calls = [lambda: cache.reserve(_int([4], cuda), _int([1], cuda)), lambda: cache.reserve(_int([-1], cuda), _int([1], cuda)),
             lambda: cache.reserve(_int([0, 0], cuda), _int([1, 1], cuda)), lambda: cache.reserve(_int([1], cuda), _int([1], cuda)),
             lambda: cache.reserve(_int([0], cuda), _int([-1], cuda)), lambda: cache.free(_int([2, 2], cuda)),
             lambda: cache.free(_int([7], cuda)), lambda: cache.fork(_int([0], cuda), _int([0], cuda)),
             lambda: cache.fork(_int([0, 1], cuda), _int([2, 1], cuda)), lambda: cache.fork(_int([9], cuda), _int([2], cuda))]
    for call in calls:
        call()
        assert quant.device_status() == 8
        for a, b in zip(state, (cache.table, cache.length, cache.refs)):
            assert torch.equal(a, b)


def test_pages_share_then_diverge(cuda):
    """Two forks of a prompt append different tokens: each sees its own, and
    attention over a shared prefix equals attention over a copy."""
    import torch
    from hy_mt_rs_b200 import paged
    from hy_mt_rs_b200.paged import PagedCache
    cache = PagedCache(1, 2, 128, 24, 16, 4, 8, cuda)
    kp, vp = cache.layer(0)
    cos, sin = torch.ones(128, 64, device=cuda), torch.zeros(128, 64, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(0)
    rand = lambda n, h: torch.randn(n, h, 128, generator=g, device=cuda)  # noqa: E731
    slot0 = _int([0], cuda)
    pos = cache.reserve(slot0, _int([37], cuda))
    paged.rope_append(rand(37, 8), rand(37, 2), rand(37, 2), kp, vp, cache.table, _int([0, 37], cuda), pos, cos, sin, slot=slot0)
    cache.fork(_int([0, 0], cuda), _int([2, 3], cuda))
    assert cache.refs.sum().item() == 2 * 3 + 3      # two shared pages, three partial ones
    slot = _int([0, 2, 3], cuda)
    pos = cache.reserve(slot, _int([1, 1, 1], cuda))
    k, v = rand(3, 2), rand(3, 2)
    starts = _int([0, 1, 2, 3], cuda)
    q = paged.rope_append(rand(3, 8), k, v, kp, vp, cache.table, starts, pos, cos, sin, slot=slot)
    out = paged.attention(q, kp, vp, cache.table, starts, pos, 1, slot=slot)
    s = dict(q=q, k=kp, v=vp, table=cache.table, new=[1, 1, 1], ctx=[37, 37, 37], starts=[0, 1, 2, 3], page=16,
             slots=[0, 2, 3])
    _close(out, s)
    tails = [cache.table[i, 2].item() for i in (0, 2, 3)]
    assert len(set(tails)) == 3
    for i, p in enumerate(tails):
        assert torch.equal(kp[p, :, 5], k[i].half())
        assert torch.equal(kp[p, :, :5], kp[tails[0], :, :5])


def test_python_refusals(cuda):
    """Shapes, types and layouts that the calls do not take."""
    import torch
    from hy_mt_rs_b200 import paged, quant, sampling
    from hy_mt_rs_b200._native import HyqError
    s = _make(cuda, [1, 3], [20, 5], 8, 2, 64, 16, True)
    args = lambda **kw: {**dict(q=s["q"], k_pages=s["k"], v_pages=s["v"], table=s["table"], row_start=s["row_start"],  # noqa: E731
                                pos=s["pos"], max_new=3), **kw}
    bad = [dict(q=s["q"].half()), dict(q=s["q"][:, :, :32]), dict(q=s["q"].transpose(0, 1)), dict(q=s["q"][:, :7]),
           dict(k_pages=s["k"].float()), dict(v_pages=s["v"][:, :1]), dict(k_pages=s["k"].bfloat16(), v_pages=s["v"].bfloat16()),
           dict(k_pages=s["k"].transpose(2, 3), v_pages=s["v"].transpose(2, 3)), dict(table=s["table"].long()),
           dict(table=s["table"][0]), dict(row_start=s["row_start"][:2]), dict(pos=s["pos"].long()), dict(max_new=-1),
           dict(max_len=10 ** 6), dict(max_len=1), dict(slot=s["pos"][:1]), dict(out=s["q"][:2]),
           dict(workspace=torch.zeros(8, dtype=torch.uint8, device=cuda))]
    for kw in bad:
        with pytest.raises(HyqError):
            paged.attention(**args(**kw))
    cos = torch.zeros(64, 32, device=cuda)
    k = torch.zeros(4, 2, 64, device=cuda)
    for kw in (dict(k=k[:3]), dict(v=k[:, :1]), dict(cos=cos[:, :16]), dict(sin=cos[:10]), dict(q_norm=cos[0]),
               dict(k_norm=cos[:2].reshape(64).half()), dict(out=torch.zeros(4, 8, 64, device=cuda).half())):
        a = {**dict(q=s["q"], k=k, v=k, k_pages=s["k"], v_pages=s["v"], table=s["table"], row_start=s["row_start"],
                    pos=s["pos"], cos=cos, sin=cos), **kw}
        with pytest.raises(HyqError):
            paged.rope_append(**a)
    x, u = torch.zeros(3, 100, device=cuda), torch.zeros(3, device=cuda)
    for a in ((x.half(), u), (x.t(), u), (x, u[:2]), (x, u, u[:1]), (x, u, None, u), (x, u, None, None, u.double()),
              (x, None)):
        with pytest.raises(HyqError):
            sampling.sample(*a)
    with pytest.raises(HyqError):
        sampling.sample(x, u, token=u)
    # nothing to do is not an error
    empty = paged.attention(s["q"][:0], s["k"], s["v"], s["table"], s["row_start"][:1], s["pos"][:0], 0)
    assert empty.shape == (0, 8, 64)
    token, prob = sampling.sample(x[:0], u[:0])
    assert token.numel() == 0 and prob.numel() == 0
    assert quant.device_status() == 0


@pytest.mark.parametrize("kv16", [True, False])
def test_attention_launch_overlap(cuda, kv16):
    """The chain of a call's kernels and the next call's, launched early."""
    import torch
    from hy_mt_rs_b200 import paged, quant
    s = _make(cuda, [1, 150, 3, 700], [300, 20, 70, 500], 16, 4, 128, 32, kv16, seed=5)
    ws = paged.attention_workspace(16, 128, cuda)
    want = _attend(s, workspace=ws).clone()
    q = s["q"].clone()
    out, again = torch.empty_like(want), torch.empty_like(want)
    quant.set_launch_overlap(True)
    try:
        for _ in range(10):
            s["q"].copy_(q * 2)
            _attend(s, out=out, workspace=ws)
            s["q"].copy_(q)
            _attend(s, out=out, workspace=ws)
            _attend(s, out=again, workspace=ws)
            assert torch.equal(out, want) and torch.equal(again, want)
    finally:
        quant.set_launch_overlap(False)
    assert quant.device_status() == 0


@pytest.mark.parametrize("dim", [128, 64])
@pytest.mark.parametrize("keys,values", [(0, 6), (10, 0), (10, 20), (0, 40)])
def test_attention_positions_of_different_sizes(cuda, dim, keys, values):
    """An f32 cache whose positions differ by powers of two: keys and values
    are split after a scale for each position or tile, which must lose nothing
    (the bound is relative to each row's own sum of p |v|)."""
    import torch
    s = _make(cuda, [200, 3, 40], [150, 100, 300], 8, 2, dim, 32, False, seed=keys + values)
    g = torch.Generator(device=cuda).manual_seed(1)
    size = s["k"].shape[0], 1, s["k"].shape[2], 1
    up = torch.randint(-keys, keys + 1, size, generator=g, device=cuda).float()
    s["k"] *= torch.exp2(up - keys)         # scores stay of ordinary size
    s["v"] *= torch.exp2(torch.randint(-values, values + 1, size, generator=g, device=cuda).float())
    got = _attend(s)
    ref, tol = _reference(s)
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("kv16,huge", [(True, 65504.0), (False, 1e30)])
def test_attention_huge_later_token(cuda, kv16, huge):
    """A finite, huge key and value of a later token leaves the tokens before it
    as they were."""
    s = _make(cuda, [200], [50], 8, 2, 128, 32, kv16, seed=9)
    clean = dict(s, k=s["k"].clone(), v=s["v"].clone())
    p = 50 + 133
    page = int(s["table"][0, p // 32])
    s["k"][page, :, p % 32] = -huge
    s["v"][page, :, p % 32] = huge
    got = _attend(s)
    ref, tol = _reference(clean)
    assert ((got[:133].double() - ref[:133]).abs() <= tol[:133]).all()
    assert got.isfinite().all()


@pytest.mark.parametrize("kv16", [True, False])
@pytest.mark.parametrize("new,ctx,at", [(3, 1500, 1), (4, 700, 3), (2, 3000, 0)])
def test_attention_few_later_tokens_do_not_leak(cuda, new, ctx, at, kv16):
    """The same where a sequence's positions are split over many CTAs: an
    infinity in a new token's values reaches it and the later ones only."""
    s = _make(cuda, [1, new, 2], [900, ctx, 40], 8, 2, 128, 32, kv16, seed=at)
    clean = dict(s, k=s["k"].clone(), v=s["v"].clone())
    p = ctx + at
    s["v"][int(s["table"][1, p // 32]), :, p % 32, 77] = float("inf")
    got = _attend(s)
    ref, tol = _reference(clean)
    rows = list(range(1 + at, 1 + new))           # of sequence 1, from that token on
    ok = (got.double() - ref).abs() <= tol
    ok[rows, :, 77] = ~got[rows, :, 77].isfinite()
    assert ok.all()
