"""Serving operators over an 8-bit paged cache and shared prefixes, and over
logits before sampling, measured on real calls.

  append   RMSNorm of the query and key heads, the position rotation, the
           quantising write of the keys and values into the cache's pages, and
           reading the new rows back as values
  attend   attention of each sequence's new tokens over its 8-bit pages, causal,
           grouped-query
  shared   attention of groups of sequences that have a prefix in common (forked
           answers, a system prompt), the prefix taken once per group, over any
           cache type
  adjust   repetition, presence and frequency penalties from token histories,
           biases and grammar masks on logits

`own` false runs the plain form of each (elementary torch operations), true the
calls of hy_mt_rs_b200.paged and hy_mt_rs_b200.sampling.  A row of an 8-bit cache
(one position of one kv head, of K or of V) is head_dim codes, int8 or e4m3, and
one f32 scale: the row's largest magnitude over 127 or 448.
"""
import math
import random

import torch

own = False

EPS = 1e-5
ROPE_BASE = 10000.0
DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "i8": torch.int8, "f8": torch.float8_e4m3fn}
LARGEST = {"i8": 127.0, "f8": 448.0}     # code of a row's largest magnitude


# --------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of 64 requests of the 1.8B architecture: latency
        dict(name="append_step", op="append", seqs=64, new_lo=1, new_hi=1, ctx_lo=40, ctx_hi=500, heads=16,
             kv_heads=4, dim=128, page=64, kv="i8", norm_first=False),
        # prompt chunks of four requests of the 7B layer, ragged, small pages, norm before rotation
        dict(name="append_chunks", op="append", seqs=4, new_lo=1801, new_hi=2303, ctx_lo=0, ctx_hi=1000, heads=32,
             kv_heads=8, dim=128, page=16, kv="f8", norm_first=True),
        # a single request decoding at a short context: latency
        dict(name="attend_one", op="attend", seqs=1, new_lo=1, new_hi=1, ctx_lo=511, ctx_hi=511, heads=16,
             kv_heads=4, dim=128, page=16, kv="i8"),
        # 64 requests decoding together, contexts from a sentence to a long document
        dict(name="attend_batch64", op="attend", seqs=64, new_lo=1, new_hi=1, ctx_lo=90, ctx_hi=4000, heads=16,
             kv_heads=4, dim=128, page=64, kv="i8"),
        # four requests decoding at very long contexts, the 7B layer: what an 8-bit cache makes room for
        dict(name="attend_long", op="attend", seqs=4, new_lo=1, new_hi=1, ctx_lo=60001, ctx_hi=100003, heads=32,
             kv_heads=8, dim=128, page=64, kv="f8"),
        # a large prompt chunk over a long context already in the cache, the 7B layer
        dict(name="attend_chunk", op="attend", seqs=1, new_lo=2048, new_hi=2048, ctx_lo=8192, ctx_hi=8192, heads=32,
             kv_heads=8, dim=128, page=128, kv="i8"),
        # a mixed step: most requests decode one token, a few feed a ragged prompt chunk
        dict(name="attend_mixed", op="attend", seqs=32, new_lo=1, new_hi=499, ctx_lo=0, ctx_hi=3001, heads=16,
             kv_heads=4, dim=128, page=32, kv="f8", chunk_every=8),
        # sixteen answers to one prompt, forked from it, f16 cache
        dict(name="shared_answers", op="shared", groups=1, per=16, prefix_lo=2001, prefix_hi=2001, own_lo=1, own_hi=200,
             new=1, heads=16, kv_heads=4, dim=128, page=64, kv="f16"),
        # 64 requests behind one long system prompt, 8-bit cache
        dict(name="shared_system", op="shared", groups=1, per=64, prefix_lo=8000, prefix_hi=8000, own_lo=30, own_hi=600,
             new=1, heads=16, kv_heads=4, dim=128, page=64, kv="i8"),
        # four documents, eight questions to each, the 7B layer
        dict(name="shared_documents", op="shared", groups=4, per=8, prefix_lo=12003, prefix_hi=20001, own_lo=20, own_hi=900,
             new=1, heads=32, kv_heads=8, dim=128, page=32, kv="f16"),
        # one request's logits at the framework's vocabulary, a translation's history
        dict(name="adjust_one", op="adjust", rows=1, vocab=120832, past_lo=700, past_hi=700, biases=0, masks=0),
        # a full batch, histories up to a long chat's, some rows with biases, some under a grammar
        dict(name="adjust_batch", op="adjust", rows=256, vocab=120832, past_lo=10, past_hi=4000, biases=40, masks=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "shared", "shared", "adjust"])
    heads, kv_heads = rng.choice([(16, 4), (32, 8), (8, 8), (12, 4), (16, 2), (20, 5)])
    dim, page, kv = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128]), rng.choice(["i8", "f8"])
    head = dict(heads=heads, kv_heads=kv_heads, dim=dim, page=page, kv=kv)
    if op == "append":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, max(1, 8192 // seqs))
        return dict(op=op, seqs=seqs, new_lo=rng.randint(1, hi), new_hi=hi, ctx_lo=rng.randint(0, 99),
                    ctx_hi=_log(rng, 100, 3000), norm_first=rng.random() < 0.5, **head)
    if op == "attend":
        # padded scores of the plain form and cached values, at most the largest listed cases'
        seqs = _log(rng, 1, 64)
        new = rng.choice([1, 1, rng.randint(2, 5), _log(rng, 6, min(2048, math.sqrt(5e8 / (heads * seqs))))])
        room = min(6e8 / (heads * new), 4e8 / (kv_heads * dim)) / seqs - new
        top = int(max(64, min(100000 if new == 1 else 10000, room)))
        hi = _log(rng, 32, top)
        case = dict(op=op, seqs=seqs, new_lo=rng.randint(1, new), new_hi=new, ctx_lo=rng.randint(0, hi), ctx_hi=hi, **head)
        if new > 8 and rng.random() < 0.5:
            case["chunk_every"] = rng.randint(2, 6)
        return case
    if op == "shared":
        groups = _log(rng, 1, 8)
        per = _log(rng, 2, 64 // groups)
        prefix = _log(rng, 30, int(min(24000, 2e8 / (groups * kv_heads * dim), 3e8 / (groups * per * heads))))
        last = _log(rng, 2, 1000)
        return dict(op=op, groups=groups, per=per, prefix_lo=rng.randint(prefix // 2, prefix), prefix_hi=prefix,
                    own_lo=rng.randint(1, last), own_hi=last, new=rng.choice([1, 1, min(2, 16 * kv_heads // heads)]),
                    **{**head, "kv": rng.choice(["f32", "f16", "i8", "f8"])})
    past = _log(rng, 2, 8000)
    return dict(op=op, rows=_log(rng, 1, 256), vocab=_log(rng, 1000, 160000), past_lo=rng.randint(0, past), past_hi=past,
                biases=rng.choice([0, 1, 37, 300]), masks=rng.choice([0, 1, 16]))


def _spread(lo, hi, n, step=7919):
    """n whole numbers of [lo, hi], spread over it in no order, the same for every seed."""
    return [lo + ((hi - lo) * ((i * step) % n) // (n - 1) if n > 1 else (hi - lo)) for i in range(n)]


def _lengths(case):
    """New tokens and positions already cached of every sequence."""
    if case["op"] == "shared":
        n = case["groups"] * case["per"]
        own_ = _spread(case["own_lo"], case["own_hi"], n, 104729)
        return [case["new"]] * n, [p + own_[i * case["per"] + j] for i, p in enumerate(_prefixes(case)) for j in range(case["per"])]
    n = case["seqs"]
    new = _spread(case["new_lo"], case["new_hi"], n)
    if "chunk_every" in case:
        new = [v if i % case["chunk_every"] == 0 else 1 for i, v in enumerate(new)]
    return new, _spread(case["ctx_lo"], case["ctx_hi"], n, 104729)


def _prefixes(case):
    return _spread(case["prefix_lo"], case["prefix_hi"], case["groups"])


def _row_bytes(case):
    """Bytes of one position of one kv head, K and V."""
    return 2 * {"f32": 4 * case["dim"], "f16": 2 * case["dim"]}.get(case["kv"], case["dim"] + 4)


def work(case):
    op = case["op"]
    if op == "adjust":
        n = case["rows"] * case["vocab"]
        past = sum(_spread(case["past_lo"], case["past_hi"], case["rows"]))
        return {"bytes": 8 * n + 4 * past + case["masks"] * case["vocab"] / 8 + 8 * case["biases"] * case["rows"], "flops": 4 * n}
    new, ctx = _lengths(case)
    t, row, kv_heads = sum(new), case["dim"] * case["heads"], case["kv_heads"]
    kv_row = 2 * kv_heads * case["dim"]
    if op == "append":
        # q in and out, k and v in, codes and scales out and in again, their values (f16) out
        return {"bytes": t * (8 * row + 4 * kv_row + 2 * kv_heads * _row_bytes(case) + 2 * kv_row), "flops": t * 9 * (row + kv_row)}
    seen = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, ctx))
    held = sum(n + c for n, c in zip(new, ctx))
    if op == "shared":
        held -= (case["per"] - 1) * sum(_prefixes(case))
    return {"bytes": 8 * t * row + _row_bytes(case) * kv_heads * held, "flops": 4 * row * seen}


# ------------------------------------------------------------------- prepare
def _int(values):
    return torch.tensor(values, dtype=torch.int32).to(DEVICE)


def _quantise(x, kv):
    """Codes and scales of rows of values."""
    top = x.abs().amax(-1)
    scale = top / LARGEST[kv]
    y = x / torch.where(scale > 0, scale, 1.0)[..., None]
    codes = y.round().clamp(-127, 127).to(torch.int8) if kv == "i8" else y.float().clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, scale.float()


def _values(codes, scale):
    """Values of rows of any cache type, in 32 bits."""
    return codes.float() if scale is None else codes.float() * scale[..., None]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = random.Random(seed)
    randn = lambda *n: torch.randn(*n, generator=g, device=DEVICE)  # noqa: E731
    s = {"case": case, "op": case["op"]}
    return _prepare_adjust(s, g, rng, randn) if case["op"] == "adjust" else _prepare_paged(s, rng, randn)


def _prepare_adjust(s, g, rng, randn):
    case, floats = s["case"], lambda v: torch.tensor(v, dtype=torch.float32).to(DEVICE)
    rows, vocab = case["rows"], case["vocab"]
    logits = randn(rows, vocab) * 2.5
    peaks = torch.randint(0, vocab, (rows, 24), generator=g, device=DEVICE)
    logits.scatter_add_(1, peaks, 6 + 2 * randn(rows, 24))
    past = _spread(case["past_lo"], case["past_hi"], rows)
    # text repeats itself: tokens fall off as the cube of a uniform number; some are the likely next ones
    width = max(1, case["past_hi"])
    history = (torch.rand(rows, width, generator=g, device=DEVICE) ** 3 * vocab).int().clamp(max=vocab - 1)
    k = min(24, width)
    history[:, :k] = torch.where(torch.rand(rows, k, generator=g, device=DEVICE) < 0.5, peaks[:, :k].int(), history[:, :k])
    pick = lambda *v: floats([rng.choice(v) for _ in range(rows)])  # noqa: E731
    s.update(logits=logits, history=history, length=_int(past), prompt=_int([n // 2 for n in past]),
             repetition=pick(1.05, 1.0, 1.2, 0.9), presence=pick(0.0, 0.5, 1.5), frequency=pick(0.0, 0.1, 0.7),
             slot=_int(rng.sample(range(rows), rows)), bias=None, mask=None, mask_row=None)
    if case["biases"]:
        counts = [rng.choice([0, case["biases"], case["biases"] // 2 + 1]) for _ in range(rows)]
        start = [sum(counts[:i]) for i in range(rows + 1)]
        total = max(1, start[-1])
        s["bias"] = (_int(start), torch.randint(0, vocab, (total,), generator=g, device=DEVICE, dtype=torch.int32), 5 * randn(total))
    if case["masks"]:
        words = -(-vocab // 32)
        # a grammar allows a few tokens, or most of them
        dense = torch.rand(case["masks"], words * 32, generator=g, device=DEVICE)
        allowed = (dense < torch.tensor([[0.002, 0.7][i % 2] for i in range(case["masks"])], device=DEVICE)[:, None]).long()
        packed = (allowed.view(case["masks"], words, 32) << torch.arange(32, device=DEVICE)).sum(-1)
        s["mask"] = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).int()
        s["mask_row"] = _int([rng.choice([-1, rng.randrange(case["masks"])]) for _ in range(rows)])
    return s


def _prepare_paged(s, rng, randn):
    case, op = s["case"], s["op"]
    kvh, dim, page, kv = case["kv_heads"], case["dim"], case["page"], case["kv"]
    new, ctx = _lengths(case)
    n, t = len(new), sum(new)
    counts = [-(-(a + b) // page) for a, b in zip(new, ctx)]
    prefix = _prefixes(case) if op == "shared" else []
    shared = [p // page for p in prefix for _ in range(case["per"])] if prefix else [0] * n   # full pages of the prefix
    pages = sum(counts) - sum(shared) + sum(p // page for p in prefix) + 3
    held = list(range(pages))
    rng.shuffle(held)
    table, at, base = torch.zeros(n, max(counts), dtype=torch.int32), 0, []
    for i, c in enumerate(counts):
        if prefix and i % case["per"] == 0:
            base = held[at:at + shared[i]]
            at += shared[i]
        mine = base + held[at:at + c - shared[i]]
        at += c - shared[i]
        table[i, :c] = torch.tensor(mine, dtype=torch.int32)
    s["k_scale"] = s["v_scale"] = None
    for name in ("k", "v"):
        x = randn(pages, kvh, page, dim)
        if kv in LARGEST:
            # heads and positions differ in size
            x *= torch.exp(0.5 * randn(pages, kvh, page, 1))
            s[name + "_pages"], s[name + "_scale"] = _quantise(x, kv)
        else:
            s[name + "_pages"] = x.to(TYPES[kv])
        del x
    for i, p in enumerate(prefix):   # the prefix's partial page: each sequence's own copy
        if p % page:
            mine = table[i * case["per"]:(i + 1) * case["per"], p // page].long().to(DEVICE)
            for name in ("k_pages", "v_pages", "k_scale", "v_scale"):
                if s[name] is not None:
                    x = s[name].view(torch.uint8) if s[name].dtype == torch.float8_e4m3fn else s[name]
                    x[mine, :, :p % page] = x[mine[:1], :, :p % page]
    starts = [0]
    for v in new:
        starts.append(starts[-1] + v)
    s.update(table=table.to(DEVICE), row_start=_int(starts), pos=_int(ctx), tokens=t, max_new=max(new),
             max_len=max(a + b for a, b in zip(new, ctx)))
    if op == "shared":
        s.update(group_start=_int([i * case["per"] for i in range(case["groups"] + 1)]), shared=_int(prefix),
                 max_shared=max(prefix), max_own=max(a + b for a, b in zip(_spread(case["own_lo"], case["own_hi"], n, 104729), new)))
    if op in ("attend", "shared"):
        # normalised heads; half of them twice as sharp
        s["q"] = randn(t, case["heads"], dim) * (1 + torch.arange(case["heads"], device=DEVICE) % 2)[:, None]
        if own:
            from hy_mt_rs_b200 import paged
            s["workspace"] = (paged.attention_workspace(case["heads"], dim, DEVICE) if op == "attend"
                              else paged.attention_shared_workspace(case["heads"], dim, t, DEVICE))
        return s
    half = dim // 2
    freq = ROPE_BASE ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
    angle = torch.arange(s["max_len"], device=DEVICE, dtype=torch.float64)[:, None] * freq
    s.update(q=randn(t, case["heads"], dim) * 1.7, k=randn(t, kvh, dim) * 1.7, v=randn(t, kvh, dim),
             cos=angle.cos().float(), sin=angle.sin().float(), q_norm=1 + 0.02 * randn(dim), k_norm=1 + 0.02 * randn(dim))
    return s


# ----------------------------------------------------------------------- run
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from hy_mt_rs_b200 import paged, sampling

    op = s["op"]
    if op == "append":
        q = paged.rope_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos"],
                              s["cos"], s["sin"], s["q_norm"], s["k_norm"], EPS, s["case"]["norm_first"],
                              k_scale=s["k_scale"], v_scale=s["v_scale"])
        k, v = paged.gather(s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos"], s["tokens"],
                            dtype=torch.float16, k_scale=s["k_scale"], v_scale=s["v_scale"])
        return {"q": q, "k": k, "v": v}
    if op == "attend":
        return paged.attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos"], s["max_new"],
                               s["max_len"], workspace=s["workspace"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if op == "shared":
        return paged.attention_shared(s["q"], s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos"],
                                      s["group_start"], s["shared"], s["max_new"], s["max_len"], s["max_shared"],
                                      workspace=s["workspace"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return sampling.adjust(s["logits"], s["history"], s["length"], s["prompt"], slot=s["slot"], repetition=s["repetition"],
                           presence=s["presence"], frequency=s["frequency"], bias=s["bias"], mask=s["mask"],
                           mask_row=s["mask_row"])


def _run_plain(s):
    return {"append": _plain_append, "attend": _plain_attend, "shared": _plain_shared, "adjust": _plain_adjust}[s["op"]](s)


def _rows(s, t):
    """The sequence of every row and its position in it."""
    row = torch.arange(t, device=DEVICE)
    seq = torch.searchsorted(s["row_start"][1:].long(), row, right=True)
    return seq, row - s["row_start"].long()[seq]


def _plain_append(s):
    page, kv = s["case"]["page"], s["case"]["kv"]
    seq, off = _rows(s, s["q"].shape[0])
    at = s["pos"].long()[seq] + off

    # 64 bits: a value next to a border between two codes falls on its own side
    def norm(x, w):
        return x * (1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * w.double()

    def rope(x):
        c, n, h = s["cos"][at][:, None].double(), s["sin"][at][:, None].double(), x.shape[-1] // 2
        a, b = x[..., :h], x[..., h:]
        return torch.cat([a * c - b * n, a * n + b * c], -1)

    both = (lambda x, w: rope(norm(x.double(), w))) if s["case"]["norm_first"] else (lambda x, w: norm(rope(x.double()), w))
    where, off, back = s["table"][seq, at // page].long(), at % page, []
    for x, pages, scales in ((both(s["k"], s["k_norm"]), s["k_pages"], s["k_scale"]), (s["v"].double(), s["v_pages"], s["v_scale"])):
        codes, scale = _quantise(x, kv)
        pages.view(torch.uint8)[where, :, off] = codes.view(torch.uint8)
        scales[where, :, off] = scale
        codes = pages.view(torch.uint8)[where, :, off].view(pages.dtype)
        back.append(_values(codes, scales[where, :, off]).half())
    return {"q": both(s["q"], s["q_norm"]).float(), "k": back[0], "v": back[1]}


def _gathered(s, name, table, count):
    """The first `count` positions of each table row: [rows, kv_heads, count, dim] in 32 bits."""
    case = s["case"]
    held = table[:, :-(-count // case["page"])].long()
    codes, scale = s[name + "_pages"], s[name + "_scale"]
    x = codes.view(torch.uint8)[held].view(codes.dtype) if codes.element_size() == 1 else codes[held]
    x = _values(x, None if scale is None else scale[held])
    return x.permute(0, 2, 1, 3, 4).reshape(table.shape[0], case["kv_heads"], -1, case["dim"])[:, :, :count]


def _plain_attend(s):
    case = s["case"]
    t, heads, dim = s["q"].shape
    n, kvh, group = case["seqs"], case["kv_heads"], heads // case["kv_heads"]
    seq, off = _rows(s, t)
    q = torch.zeros(n, s["max_new"], heads, dim, device=DEVICE)
    q[seq, off] = s["q"] * (1 / math.sqrt(dim))
    q = q.view(n, -1, kvh, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kvh, -1, dim)
    score = (q @ _gathered(s, "k", s["table"], s["max_len"]).transpose(2, 3)).view(n, kvh, group, s["max_new"], -1)
    last = s["pos"].long()[:, None] + torch.arange(s["max_new"], device=DEVICE)
    hidden = torch.arange(s["max_len"], device=DEVICE) > last[:, :, None]
    score.masked_fill_(hidden[:, None, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.view(n, kvh, group * s["max_new"], -1) @ _gathered(s, "v", s["table"], s["max_len"])).view(n, kvh, group, s["max_new"], dim)
    return (out / total).permute(0, 3, 1, 2, 4).reshape(n, s["max_new"], heads, dim)[seq, off]


def _plain_shared(s):
    case = s["case"]
    groups, per, new, kvh, dim, page = (case[k] for k in ("groups", "per", "new", "kv_heads", "dim", "page"))
    n, group = groups * per, case["heads"] // case["kv_heads"]
    shared = s["shared"].long()
    q = (s["q"] * (1 / math.sqrt(dim))).view(n, new, kvh, group, dim).permute(0, 2, 1, 3, 4)    # [seqs, kv_heads, new, group, dim]
    by_group = q.reshape(groups, per, kvh, new * group, dim).transpose(1, 2).reshape(groups, kvh, -1, dim)
    first = s["table"][::per]
    before = by_group @ _gathered(s, "k", first, s["max_shared"]).transpose(2, 3)
    before.masked_fill_((torch.arange(s["max_shared"], device=DEVICE) >= shared[:, None])[:, None, None], -math.inf)
    before = before.view(groups, kvh, per, new * group, -1).transpose(1, 2).reshape(n, kvh, new * group, -1)
    # each sequence's own positions, behind the prefix
    at = shared.repeat_interleave(per)[:, None] + torch.arange(s["max_own"], device=DEVICE)
    held = s["table"].long().gather(1, (at // page).clamp(max=s["table"].shape[1] - 1))

    def behind(name):   # [seqs, kv_heads, positions, dim]
        codes, scale = s[name + "_pages"], s[name + "_scale"]
        x = codes.view(torch.uint8)[held, :, at % page].view(codes.dtype) if codes.element_size() == 1 else codes[held, :, at % page]
        return _values(x, None if scale is None else scale[held, :, at % page]).transpose(1, 2)

    after = (q.reshape(n, kvh, -1, dim) @ behind("k").transpose(2, 3)).view(n, kvh, new, group, -1)
    last = s["pos"].long()[:, None] + torch.arange(new, device=DEVICE)
    after.masked_fill_((at[:, None] > last[:, :, None])[:, None, :, None], -math.inf)
    score = torch.cat([before, after.view(n, kvh, new * group, -1)], -1)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    w = score[..., :s["max_shared"]].view(groups, per, kvh, new * group, -1).transpose(1, 2).reshape(groups, kvh, per * new * group, -1)
    out = (w @ _gathered(s, "v", first, s["max_shared"])).view(groups, kvh, per, new * group, dim).transpose(1, 2).reshape(n, kvh, -1, dim)
    out = (out + score[..., s["max_shared"]:] @ behind("v")) / total
    return out.view(n, kvh, new, group, dim).permute(0, 2, 1, 3, 4).reshape(n * new, case["heads"], dim)


def _plain_adjust(s):
    x = s["logits"]
    rows, n = x.shape
    slot = s["slot"].long()
    past = s["history"][slot].long()
    index = torch.arange(past.shape[1], device=DEVICE)
    valid = index < s["length"][slot][:, None]
    made = valid & (index >= s["prompt"][slot][:, None])
    zero = torch.zeros(rows, n, dtype=torch.int32, device=DEVICE)
    seen = zero.scatter_add(1, past, valid.int()) > 0
    count = zero.scatter_add_(1, past, made.int())
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = torch.where(count > 0, x - (s["frequency"][:, None] * count.float() + s["presence"][:, None]), x)
    if s["bias"] is not None:   # of several entries for one token the last counts
        start, token, value = s["bias"]
        entry = torch.arange(token.numel(), device=DEVICE)
        row = torch.searchsorted(start[1:].long(), entry, right=True).clamp(max=rows - 1)
        last = torch.full((rows * n,), -1, dtype=torch.int64, device=DEVICE)
        last.scatter_reduce_(0, row * n + token.long(), torch.where(entry < start[-1], entry, -1), "amax")
        last = last.view(rows, n)
        x = torch.where(last >= 0, x + value[last.clamp(min=0)], x)
    if s["mask"] is not None:
        token = torch.arange(n, device=DEVICE)
        bits = (s["mask"][:, token // 32] >> (token % 32)) & 1
        m = s["mask_row"].long()
        x = torch.where((m[:, None] < 0) | (bits[m.clamp(min=0)] > 0), x, -math.inf)
    return x


# --------------------------------------------------------------------- exact
def exact(case, seed):
    """What run() returns, from the definitions, one sequence, head or row at
    a time in 64 bits."""
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "shared": _exact_attend, "adjust": _exact_adjust}[case["op"]](s)


def _exact_attend(s):
    case, starts, ctx = s["case"], s["row_start"].tolist(), s["pos"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    group = case["heads"] // case["kv_heads"]
    for i, c in enumerate(ctx):
        a, b = starts[i], starts[i + 1]
        length = c + b - a
        held = s["table"][i, :-(-length // case["page"])].long()
        # (a shared prefix's pages are in every sequence's own table row too)
        seen = torch.arange(length, device=DEVICE)[None] <= torch.arange(c, length, device=DEVICE)[:, None]
        for h in range(case["kv_heads"]):
            def rows(name):
                codes = s[name + "_pages"][:, h]
                x = (codes.view(torch.uint8)[held].view(codes.dtype) if codes.element_size() == 1 else codes[held]).double()
                if s[name + "_scale"] is not None:
                    x = x * s[name + "_scale"][held, h].double()[..., None]
                return x.reshape(-1, case["dim"])[:length]
            k, v = rows("k"), rows("v")
            for j in range(h * group, (h + 1) * group):
                x = s["q"][a:b, j].double() @ k.T / case["dim"] ** 0.5
                out[a:b, j] = torch.softmax(x.masked_fill(~seen, -math.inf), -1) @ v
    return out


def _exact_append(s):
    case, starts, h = s["case"], s["row_start"].tolist(), s["case"]["dim"] // 2
    out, back = torch.empty_like(s["q"], dtype=torch.float64), torch.empty_like(s["k"], dtype=torch.float64)
    for i, c in enumerate(s["pos"].tolist()):
        mine = slice(starts[i], starts[i + 1])
        at = torch.arange(c, c + starts[i + 1] - starts[i], device=DEVICE)
        turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
        for x, w, to in ((s["q"], s["q_norm"], out), (s["k"], s["k_norm"], back)):
            x = x[mine].double()
            size = (x.square().mean(-1, keepdim=True) + EPS).sqrt()   # a rotation keeps it
            if case["norm_first"]:
                x = x * w.double()
            z = torch.complex(x[..., :h], x[..., h:]) * turn
            x = torch.cat([z.real, z.imag], -1)
            to[mine] = x / size if case["norm_first"] else x * w.double() / size

    def held(x):   # the value that a row's codes stand for
        step = x.abs().amax(-1, keepdim=True) / LARGEST[case["kv"]]
        y = x / step
        if case["kv"] == "i8":
            return y.round() * step
        unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)   # e4m3: 3 bits behind the first, 2^-9 at least
        return (y / unit).round() * unit * step

    return {"q": out, "k": held(back), "v": held(s["v"].double())}


def _exact_adjust(s):
    case, x = s["case"], s["logits"].double().cpu()
    history, slot, length, prompt = (s[k].cpu().tolist() if k != "history" else s[k].cpu() for k in ("history", "slot", "length", "prompt"))
    rep, presence, frequency = (s[k].double().cpu().tolist() for k in ("repetition", "presence", "frequency"))
    bias = [v.cpu() for v in s["bias"]] if s["bias"] is not None else None
    mask_row = s["mask_row"].tolist() if s["mask"] is not None else None
    if s["mask"] is not None:
        words = s["mask"].cpu().long() & 0xffffffff
        allowed = ((words[:, :, None] >> torch.arange(32)) & 1).bool().view(words.shape[0], -1)[:, :case["vocab"]]
    for r in range(case["rows"]):
        past, y = history[slot[r]][:length[slot[r]]].long(), x[r]
        seen = torch.unique(past)
        y[seen] = torch.where(y[seen] > 0, y[seen] / rep[r], y[seen] * rep[r])
        token, count = torch.unique(past[prompt[slot[r]]:], return_counts=True)
        y[token] -= frequency[r] * count.double() + presence[r]
        if bias is not None:
            a, b = bias[0][r:r + 2].tolist()
            last = dict(zip(bias[1][a:b].tolist(), bias[2][a:b].double().tolist()))
            for token, value in last.items():
                y[token] += value
        if mask_row is not None and mask_row[r] >= 0:
            y[~allowed[mask_row[r]]] = -math.inf
    return x.to(DEVICE)
