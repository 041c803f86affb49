"""Serving operators over a paged KV cache, measured on real calls.

Four operators that one step of a serving loop runs next to the quantized
products of this framework:

  append   RMSNorm of every query and key head, the position rotation and the
           write of the rotated keys and the values into the cache's pages
  attend   attention of each sequence's new tokens (one, a few or a prompt
           chunk) over its pages, causal, grouped-query
  sample   temperature, top-k, top-p and min-p sampling from given uniform
           numbers
  pages    fork sequences (full pages shared, the partial page copied), and
           compact the live pages to the front of the pool

`own` false runs the plain form of each (elementary torch operations), true
the calls of hy_mt_rs_b200.paged and hy_mt_rs_b200.sampling.  Caches are
[pages, kv_heads, page_size, head_dim] per layer, f32 or f16; all other values
are f32 and all indexes int32, as in the rest of the framework.
"""
import math
import random

import torch

own = False

EPS = 1e-5
ROPE_BASE = 10000.0
GRID = 24            # uniform numbers and top-p are read on a grid of 2^-24
WEIGHT_BITS = 40     # a token's weight is floor(2^40 exp((logit - max) / temperature))
DEVICE = "cuda"


# --------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of 64 requests of the 1.8B architecture, f16 cache
        dict(name="append_step", op="append", seqs=64, new_lo=1, new_hi=1, ctx_lo=40, ctx_hi=500, heads=16,
             kv_heads=4, dim=128, page=64, kv="f16", norm_first=False),
        # prompt chunks of four requests of the 7B layer, ragged, f32 cache, small pages, norm before rotation
        dict(name="append_chunks", op="append", seqs=4, new_lo=1801, new_hi=2303, ctx_lo=0, ctx_hi=1000, heads=32,
             kv_heads=8, dim=128, page=16, kv="f32", norm_first=True),
        # a single request decoding at a short context, the framework's default f32 cache: latency
        dict(name="attend_one", op="attend", seqs=1, new_lo=1, new_hi=1, ctx_lo=511, ctx_hi=511, heads=16,
             kv_heads=4, dim=128, page=16, kv="f32"),
        # 64 requests decoding together, contexts from a sentence to a long document
        dict(name="attend_batch64", op="attend", seqs=64, new_lo=1, new_hi=1, ctx_lo=90, ctx_hi=4000, heads=16,
             kv_heads=4, dim=128, page=64, kv="f16"),
        # four requests decoding at very long contexts, the 7B layer
        dict(name="attend_long", op="attend", seqs=4, new_lo=1, new_hi=1, ctx_lo=60001, ctx_hi=100003, heads=32,
             kv_heads=8, dim=128, page=64, kv="f16"),
        # the largest prompt chunk over a long context already in the cache, the 7B layer
        dict(name="attend_chunk", op="attend", seqs=1, new_lo=4096, new_hi=4096, ctx_lo=12288, ctx_hi=12288, heads=32,
             kv_heads=8, dim=128, page=128, kv="f16"),
        # a mixed step: most requests decode one token, a few feed a ragged prompt chunk
        dict(name="attend_mixed", op="attend", seqs=32, new_lo=1, new_hi=499, ctx_lo=0, ctx_hi=3001, heads=16,
             kv_heads=4, dim=128, page=32, kv="f16", chunk_every=8),
        # prompt chunks over the default f32 cache
        dict(name="attend_chunk_f32", op="attend", seqs=3, new_lo=201, new_hi=256, ctx_lo=0, ctx_hi=2050, heads=16,
             kv_heads=4, dim=128, page=16, kv="f32"),
        # one request's next token at the framework's vocabulary
        dict(name="sample_one", op="sample", rows=1, vocab=120832, mixed=False, ties=False),
        # a full batch with parameters of its own for each request, some logits tied
        dict(name="sample_batch", op="sample", rows=256, vocab=120832, mixed=True, ties=True),
        # eight parallel answers to one prompt: share its pages, copy the partial one in every layer
        dict(name="pages_fork", op="fork", layers=32, parents=1, children=8, len_lo=1000, len_hi=1000, kv_heads=4,
             dim=128, page=64, kv="f16", pages=64),
        # a fragmented pool: a quarter of the pages lie high and move down, in every layer
        dict(name="pages_compact", op="compact", layers=16, seqs=24, live=250, movers=125, kv_heads=4, dim=128, page=64,
             kv="f16", pages=512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "sample", "pages"])
    heads, kv_heads = rng.choice([(16, 4), (32, 8), (8, 8), (12, 4), (16, 2), (20, 5)])
    dim, page, kv = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128]), rng.choice(["f32", "f16", "f16"])
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
        room = min(2e9 / (heads * new), 3e8 / (kv_heads * dim)) / seqs - new
        top = int(max(64, min(100000 if new == 1 else 16000, room)))
        hi = _log(rng, 32, top)
        case = dict(op=op, seqs=seqs, new_lo=rng.randint(1, new), new_hi=new, ctx_lo=rng.randint(0, hi), ctx_hi=hi, **head)
        if new > 8 and rng.random() < 0.5:
            case["chunk_every"] = rng.randint(2, 6)
        return case
    if op == "sample":
        return dict(op=op, rows=_log(rng, 1, 256), vocab=_log(rng, 1000, 160000), mixed=rng.random() < 0.7,
                    ties=rng.random() < 0.5)
    layers = rng.randint(2, 16)
    # pages of a pool of at most 1.2 GB
    most = int(1.2e9 / (2 * layers * kv_heads * page * dim * (2 if kv == "f16" else 4)))
    if rng.random() < 0.5:
        parents, children = rng.randint(1, 4), rng.randint(1, 4)
        longest = _log(rng, page, max(page, min(2000, page * (most // parents - 12))))
        pages = parents * (longest // page + 2) + 2 * parents * children + rng.randint(1, 99)
        return dict(op="fork", layers=layers, parents=parents, children=children, len_lo=rng.randint(1, longest),
                    len_hi=longest, kv_heads=kv_heads, dim=dim, page=page, kv=kv, pages=pages)
    pages = _log(rng, 30, max(40, min(1000, most)))
    live = rng.randint(pages // 4, pages // 2)
    return dict(op="compact", layers=layers, seqs=rng.randint(1, 40), live=live, movers=rng.randint(1, live // 2),
                kv_heads=kv_heads, dim=dim, page=page, kv=kv, pages=pages)


def _spread(lo, hi, n, step=7919):
    """n whole numbers of [lo, hi], spread over it in no order, the same for every seed."""
    return [lo + ((hi - lo) * ((i * step) % n) // (n - 1) if n > 1 else (hi - lo)) for i in range(n)]


def _lengths(case):
    """New tokens and positions already cached of every sequence."""
    n = case["seqs"]
    new = _spread(case["new_lo"], case["new_hi"], n)
    if "chunk_every" in case:
        new = [v if i % case["chunk_every"] == 0 else 1 for i, v in enumerate(new)]
    return new, _spread(case["ctx_lo"], case["ctx_hi"], n, 104729)


def _kv_bytes(case):
    return 2 if case["kv"] == "f16" else 4


def work(case):
    op = case["op"]
    if op in ("append", "attend"):
        new, ctx = _lengths(case)
        t, row = sum(new), case["dim"] * case["heads"]
        kv_row = 2 * case["kv_heads"] * case["dim"]
    if op == "append":
        # q in and out, k and v in, the cache rows out
        return {"bytes": t * (8 * row + 4 * kv_row + _kv_bytes(case) * kv_row), "flops": t * 7 * (row + kv_row // 2)}
    if op == "attend":
        seen = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, ctx))
        return {"bytes": 8 * t * row + _kv_bytes(case) * kv_row * sum(n + c for n, c in zip(new, ctx)),
                "flops": 4 * row * seen}
    if op == "sample":
        return {"bytes": 4 * case["rows"] * case["vocab"], "flops": 4 * case["rows"] * case["vocab"]}
    page = 2 * case["layers"] * case["kv_heads"] * case["page"] * case["dim"] * _kv_bytes(case)
    if op == "fork":   # one page for every child of a sequence that ends inside a page
        lens = _spread(case["len_lo"], case["len_hi"], case["parents"])
        moved = case["children"] * sum(n % case["page"] > 0 for n in lens)
    else:
        moved = case["movers"]
    return {"bytes": 2 * moved * page + 4 * case["pages"], "flops": 0}


# ------------------------------------------------------------------- prepare
def _int(values):
    return torch.tensor(values, dtype=torch.int32).to(DEVICE)


def _kv_dtype(case):
    return torch.float16 if case["kv"] == "f16" else torch.float32


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = random.Random(seed)
    randn = lambda *n: torch.randn(*n, generator=g, device=DEVICE)  # noqa: E731
    op = case["op"]
    s = {"case": case, "op": op}
    if op == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = randn(rows, vocab) * 2.5
        peaks = torch.randint(0, vocab, (rows, 24), generator=g, device=DEVICE)
        logits.scatter_add_(1, peaks, 6 + 2 * randn(rows, 24))
        if case["ties"]:   # values of a bf16 product: many equal logits
            logits[::2] = logits[::2].bfloat16().float()
        pick = lambda *v: [rng.choice(v) for _ in range(rows)] if case["mixed"] else [v[1]] * rows  # noqa: E731
        floats = lambda v: torch.tensor(v, dtype=torch.float32).to(DEVICE)  # noqa: E731
        s.update(logits=logits, temperature=floats(pick(1.0, 0.7, 0.0, 1.3)), top_k=_int(pick(0, 40, 20, 1000)),
                 top_p=floats(pick(1.0, 0.9, 0.6, 0.95)), min_p=floats(pick(0.0, 0.02, 0.1)),
                 u=torch.rand(rows, generator=g, device=DEVICE))
        return s
    kvh, dim, page, dtype = case["kv_heads"], case["dim"], case["page"], _kv_dtype(case)
    if op in ("fork", "compact"):
        pool = randn(case["layers"], 2, case["pages"], kvh, page, dim).to(dtype)
        if op == "fork":
            lens = _spread(case["len_lo"], case["len_hi"], case["parents"])
            held = list(range(case["pages"]))
            rng.shuffle(held)
            slots = case["parents"] * (1 + case["children"])
        else:
            # `live` pages in use, `movers` of them above the first `live`
            held = rng.sample(range(case["live"]), case["live"] - case["movers"])
            held += rng.sample(range(case["live"], case["pages"]), case["movers"])
            rng.shuffle(held)
            slots = min(case["seqs"], case["live"])
            cut = sorted(rng.sample(range(1, case["live"]), slots - 1))
            counts = [b - a for a, b in zip([0] + cut, cut + [case["live"]])]
            lens = [page * n - rng.randrange(page) for n in counts]
        width = case["live"] if op == "compact" else -(-case["len_hi"] // page) + 1
        table = torch.full((slots, width), -1, dtype=torch.int32)
        refs, length, at = torch.zeros(case["pages"], dtype=torch.int32), torch.zeros(slots, dtype=torch.int32), 0
        for i, n in enumerate(lens):
            slot = i * (1 + case["children"]) if op == "fork" else i
            mine = held[at:at + -(-n // page)]
            at += len(mine)
            table[slot, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
            refs[mine] = 1
            length[slot] = n
        s.update(pool=pool, table=table.to(DEVICE), length=length.to(DEVICE), refs=refs.to(DEVICE))
        if op == "fork":
            step = 1 + case["children"]
            s["src"] = _int([step * i for i in range(case["parents"]) for _ in range(case["children"])])
            s["dst"] = _int([step * i + 1 + j for i in range(case["parents"]) for j in range(case["children"])])
        else:
            s["before"] = (s["table"].clone(), s["refs"].clone())
        if own:
            from hy_mt_rs_b200 import paged
            s["cache"] = paged.PagedCache.over(s["pool"], s["table"], s["length"], s["refs"])
        return s
    new, ctx = _lengths(case)
    n, t = case["seqs"], sum(new)
    counts = [-(-(a + b) // page) for a, b in zip(new, ctx)]
    pages = sum(counts) + 3
    held = list(range(pages))
    rng.shuffle(held)
    table, at = torch.zeros(n, max(counts), dtype=torch.int32), 0
    for i, c in enumerate(counts):
        table[i, :c] = torch.tensor(held[at:at + c], dtype=torch.int32)
        at += c
    k_pages, v_pages = (randn(pages, kvh, page, dim).to(dtype) for _ in range(2))
    starts = [0]
    for v in new:
        starts.append(starts[-1] + v)
    s.update(k_pages=k_pages, v_pages=v_pages, table=table.to(DEVICE), row_start=_int(starts), pos=_int(ctx),
             max_new=max(new), max_len=max(a + b for a, b in zip(new, ctx)))
    if op == "attend":
        # normalised heads; half of them twice as sharp
        s["q"] = randn(t, case["heads"], dim) * (1 + torch.arange(case["heads"], device=DEVICE) % 2)[:, None]
        if own:
            from hy_mt_rs_b200 import paged
            s["workspace"] = paged.attention_workspace(case["heads"], dim, DEVICE)
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
                              s["cos"], s["sin"], s["q_norm"], s["k_norm"], EPS, s["case"]["norm_first"])
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if op == "attend":
        return paged.attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["row_start"], s["pos"], s["max_new"],
                               s["max_len"], workspace=s["workspace"])
    if op == "sample":
        token, prob = sampling.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        return {"token": token, "prob": prob}
    if op == "fork":
        s["cache"].fork(s["src"], s["dst"])
    else:
        s["table"].copy_(s["before"][0])
        s["refs"].copy_(s["before"][1])
        s["cache"].compact()
    return {"table": s["table"], "length": s["length"], "refs": s["refs"], "pool": s["pool"]}


def _run_plain(s):
    if s["op"] == "fork":
        return _plain_fork(s)
    if s["op"] == "compact":
        s["table"].copy_(s["before"][0])
        s["refs"].copy_(s["before"][1])
        return _plain_compact(s)
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[s["op"]](s)


def _rows(s, t):
    """The sequence of every row and its position in it."""
    row = torch.arange(t, device=DEVICE)
    seq = torch.searchsorted(s["row_start"][1:].long(), row, right=True)
    return seq, row - s["row_start"].long()[seq]


def _plain_append(s):
    page = s["case"]["page"]
    seq, off = _rows(s, s["q"].shape[0])
    at = s["pos"].long()[seq] + off

    def norm(x, w):
        return x * (1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * w

    def rope(x):
        c, n, h = s["cos"][at][:, None], s["sin"][at][:, None], x.shape[-1] // 2
        a, b = x[..., :h], x[..., h:]
        return torch.cat([a * c - b * n, a * n + b * c], -1)

    both = (lambda x, w: rope(norm(x, w))) if s["case"]["norm_first"] else (lambda x, w: norm(rope(x), w))
    where = s["table"][seq, at // page].long()
    s["k_pages"][where, :, at % page] = both(s["k"], s["k_norm"]).to(s["k_pages"].dtype)
    s["v_pages"][where, :, at % page] = s["v"].to(s["v_pages"].dtype)
    return {"q": both(s["q"], s["q_norm"]), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attend(s):
    case = s["case"]
    t, heads, dim = s["q"].shape
    n, kvh, group = case["seqs"], case["kv_heads"], heads // case["kv_heads"]
    seq, off = _rows(s, t)
    held = s["table"][:, :-(-s["max_len"] // case["page"])].long()

    def gather(x):   # [seqs, kv_heads, positions, dim]
        return x[held].float().permute(0, 2, 1, 3, 4).reshape(n, kvh, -1, dim)[:, :, :s["max_len"]]

    q = torch.zeros(n, s["max_new"], heads, dim, device=DEVICE)
    q[seq, off] = s["q"] * (1 / math.sqrt(dim))
    q = q.view(n, -1, kvh, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kvh, -1, dim)
    score = (q @ gather(s["k_pages"]).transpose(2, 3)).view(n, kvh, group, s["max_new"], -1)
    last = s["pos"].long()[:, None] + torch.arange(s["max_new"], device=DEVICE)
    hidden = torch.arange(s["max_len"], device=DEVICE) > last[:, :, None]
    score.masked_fill_(hidden[:, None, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.view(n, kvh, group * s["max_new"], -1) @ gather(s["v_pages"])).view(n, kvh, group, s["max_new"], dim) / total
    return out.permute(0, 3, 1, 2, 4).reshape(n, s["max_new"], heads, dim)[seq, off]


def _plain_sample(s):
    x = torch.where(torch.isnan(s["logits"]), -math.inf, s["logits"])
    rows, n = x.shape
    one = 1 << GRID
    greedy = s["temperature"] <= 0
    inverse = 1 / torch.where(greedy, 1.0, s["temperature"])
    sorted_x, order = torch.sort(x, dim=1, descending=True, stable=True)
    e = torch.exp((sorted_x - sorted_x[:, :1]) * inverse[:, None])
    w = (e * float(1 << WEIGHT_BITS)).to(torch.int64)
    rank = torch.arange(n, device=DEVICE)
    k = torch.where(greedy, 1, torch.where(s["top_k"] > 0, s["top_k"], n)).long()
    w = torch.where(rank < k[:, None], w, 0)
    before = w.cumsum(1) - w
    total = w.sum(1)
    # ceil(total * p / 2^24) in whole numbers
    p = (s["top_p"].clamp(0, 1) * one).ceil().long()
    limit = (total >> GRID) * p + (((total & (one - 1)) * p + one - 1) >> GRID)
    keep = (before < limit.clamp(min=1)[:, None]) & (e >= s["min_p"][:, None])
    w = torch.where(keep, w, 0)
    total = w.sum(1)
    w = torch.zeros_like(w).scatter_(1, order, w)
    u = (s["u"].clamp(0, 1) * one).long().clamp(max=one - 1)
    aim = (total >> GRID) * u + (((total & (one - 1)) * u) >> GRID)
    token = (w.cumsum(1) <= aim[:, None]).sum(1)
    prob = w.gather(1, token[:, None])[:, 0].float() / total.float()
    return {"token": token.int(), "prob": prob}


def _plain_fork(s):
    page, width = s["case"]["page"], s["table"].shape[1]
    src, dst, refs, column = s["src"].long(), s["dst"].long(), s["refs"], torch.arange(width, device=DEVICE)

    def count(slots, last):   # +-1 for every page that these slots hold in columns < last
        held = (column < last[:, None])
        return torch.zeros_like(refs).index_add_(0, s["table"][slots].clamp(min=0).long().view(-1), held.int().view(-1))

    refs -= count(dst, (s["length"][dst] + page - 1) // page)
    full, part = s["length"][src] // page, s["length"][src] % page > 0
    refs += count(src, full)
    free = torch.argsort((refs > 0).int(), stable=True)     # free pages first, lowest first
    got = free[(part.cumsum(0) - 1).clamp(min=0)]
    tail = s["table"][src].gather(1, full.clamp(max=width - 1).long()[:, None])[:, 0]
    row = torch.where(column < full[:, None], s["table"][src], -1)
    s["table"][dst] = torch.where((column == full[:, None]) & part[:, None], got.int()[:, None], row)
    s["length"][dst] = s["length"][src]
    refs.index_add_(0, got, part.int())
    s["pool"][:, :, torch.where(part, got, tail.clamp(min=0))] = s["pool"][:, :, tail.clamp(min=0).long()]
    return {"table": s["table"], "length": s["length"], "refs": refs, "pool": s["pool"]}


def _plain_compact(s):
    refs, pages = s["refs"], s["refs"].numel()
    live = (refs > 0).sum()
    index = torch.arange(pages, device=DEVICE)
    mover, hole = (refs > 0) & (index >= live), (refs == 0) & (index < live)
    # the j-th page that moves goes to the j-th hole
    movers, holes = torch.argsort((~mover).int(), stable=True), torch.argsort((~hole).int(), stable=True)
    to = torch.where(index < mover.sum(), holes, movers)
    new = torch.empty_like(index).scatter_(0, movers, to)
    new = torch.where(mover, new, index)
    moved = s["case"]["movers"]
    s["pool"][:, :, holes[:moved]] = s["pool"][:, :, movers[:moved]]
    s["table"].copy_(torch.where(s["table"] >= 0, new[s["table"].clamp(min=0).long()], s["table"].long()))
    refs.copy_(torch.where(index < live, torch.where(hole, 1, refs), 0))
    return {"table": s["table"], "length": s["length"], "refs": refs, "pool": s["pool"]}


# --------------------------------------------------------------------- exact
def exact(case, seed):
    """What run() returns, from the definitions, one sequence, head or row at
    a time in 64 bits."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "attend":
        return _exact_attend(s)
    if op == "append":
        return _exact_append(s)
    if op == "sample":
        return _exact_sample(s)
    return _exact_pages(s)


def _exact_attend(s):
    case, starts, ctx = s["case"], s["row_start"].tolist(), s["pos"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    group = case["heads"] // case["kv_heads"]
    for i, c in enumerate(ctx):
        a, b = starts[i], starts[i + 1]
        held = s["table"][i, :-(-(c + b - a) // case["page"])].long()
        for h in range(case["heads"]):
            k = s["k_pages"][held, h // group].double().reshape(-1, case["dim"])[:c + b - a]
            v = s["v_pages"][held, h // group].double().reshape(-1, case["dim"])[:c + b - a]
            x = s["q"][a:b, h].double() @ k.T / case["dim"] ** 0.5
            seen = torch.arange(c + b - a, device=DEVICE)[None] <= torch.arange(c, c + b - a, device=DEVICE)[:, None]
            out[a:b, h] = torch.softmax(x.masked_fill(~seen, -math.inf), -1) @ v
    return out


def _exact_append(s):
    case, starts, ctx, h = s["case"], s["row_start"].tolist(), s["pos"].tolist(), s["case"]["dim"] // 2
    k_pages, v_pages, out = s["k_pages"].double(), s["v_pages"].double(), torch.empty_like(s["q"], dtype=torch.float64)
    for i, c in enumerate(ctx):
        at = torch.arange(c, c + starts[i + 1] - starts[i], device=DEVICE)
        turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
        got = []
        for x, w in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
            x = x[starts[i]:starts[i + 1]].double()
            size = (x.square().mean(-1, keepdim=True) + EPS).sqrt()   # a rotation keeps it
            if case["norm_first"]:
                x = x * w.double()
            z = torch.complex(x[..., :h], x[..., h:]) * turn
            x = torch.cat([z.real, z.imag], -1)
            got.append(x / size if case["norm_first"] else x * w.double() / size)
        out[starts[i]:starts[i + 1]] = got[0]
        where = s["table"][i].long()[at // case["page"]]
        k_pages[where, :, at % case["page"]] = got[1]
        v_pages[where, :, at % case["page"]] = s["v"][starts[i]:starts[i + 1]].double()
    return {"q": out, "k_pages": k_pages, "v_pages": v_pages}


def _exact_sample(s):
    prob = torch.empty(s["case"]["rows"], dtype=torch.float64)
    for r in range(s["case"]["rows"]):
        x = s["logits"][r].double()
        temperature, k = float(s["temperature"][r]), int(s["top_k"][r])
        if temperature <= 0:
            prob[r] = 1.0
            continue
        p = torch.exp((x - x.max()) / temperature)
        order = torch.argsort(x, descending=True, stable=True)
        kept = order[:k] if k > 0 else order
        mass = p[kept].cumsum(0)
        kept = kept[(mass - p[kept] < float(s["top_p"][r]) * mass[-1]) & (p[kept] >= float(s["min_p"][r]))]
        chosen = torch.zeros_like(p)
        chosen[kept] = p[kept]
        token = int((chosen.cumsum(0) <= float(s["u"][r]) * chosen.sum()).sum())
        prob[r] = chosen[token] / chosen.sum()
    return {"token": None, "prob": prob}


def _exact_pages(s):
    case, page = s["case"], s["case"]["page"]
    table, refs, length = s["table"].tolist(), s["refs"].tolist(), s["length"].tolist()
    copies = []
    if case["op"] == "fork":
        pairs = list(zip(s["src"].tolist(), s["dst"].tolist()))
        for a, b in pairs:
            table[b], length[b] = [-1] * len(table[b]), length[a]
            for j in range(length[a] // page):
                table[b][j] = table[a][j]
                refs[table[a][j]] += 1
        for a, b in pairs:
            if length[a] % page:
                j, got = length[a] // page, refs.index(0)
                refs[got], table[b][j] = 1, got
                copies.append((table[a][j], got))
    else:
        live = sum(r > 0 for r in refs)
        holes = [i for i in range(live) if refs[i] == 0]
        copies = list(zip([i for i in range(live, len(refs)) if refs[i] > 0], holes))
        for a, b in copies:
            refs[b], refs[a] = refs[a], 0
        moved = dict(copies)
        table = [[moved.get(v, v) for v in row] for row in table]
    pool = s["pool"]
    for a, b in copies:
        pool[:, :, b] = pool[:, :, a]
    return {"table": _int(table), "length": _int(length), "refs": _int(refs), "pool": pool}
