"""Serving many requests over one paged cache: prompt chunks and decoding
tokens mixed in a step, sampled tokens, answers that share their prompt's
pages.

The reference serves one Session per request (README.md:139-141), each with a
contiguous cache (model.rs:116-120) and a Sampler on the host (generation.rs).
Here a step runs the batched forward (model.rs:549-646) over the new rows of
all requests at once: hyq_embed and the batched products as DenseBatch runs
them, hyq_paged_rope_append and hyq_paged_attention over the requests' pages
(hy_mt_rs_b200.paged), and hyq_sample for the next tokens
(hy_mt_rs_b200.sampling).
"""
import torch

from . import paged, quant, sampling
from ._native import HyqError, check, lib
from .model import _Acts, _add_norm, _gate_up_normed, _matmul_normed, _p, _qkv_normed
from .quant import _need_cuda

__all__ = ["PagedBatch"]


class PagedBatch:
    """Requests in the slots of a PagedCache, over a DenseModel's weights
    (either architecture; the cache type and the products' precision are the
    model's).

    slots: requests at a time, at most 1024.  They share `pages` pages of page_size
    positions (by default enough for every slot to reach cfg.positions).
    chunk: prompt tokens that generate() feeds in a step, next to the tokens of
    the requests that decode already."""

    def __init__(self, model, slots, pages=None, page_size=64, chunk=256):
        cfg, dev = model.cfg, model.device
        if not 1 <= slots <= 1024:
            raise ValueError("1 to 1024 slots")
        if chunk < 1 or page_size < 1:
            raise ValueError("at least one position of a page and one prompt token of a step")
        self.m, self.slots, self.chunk = model, slots, chunk
        width = -(-cfg.positions // page_size)
        self.cache = paged.PagedCache(len(model.layers), cfg.kv_heads, cfg.head_dim, pages or slots * width, page_size,
                                      slots, width, dev, dtype=model.kv_dtype)
        half = cfg.head_dim // 2
        self.cos, self.sin = model.cos.view(cfg.positions, half), model.sin.view(cfg.positions, half)
        self.workspace = paged.attention_workspace(cfg.heads, cfg.head_dim, dev)
        self.acts = _Acts(cfg, slots + chunk, dev)
        self._known([0] * slots)

    def _state(self):
        length = self.cache.length
        return self.cache.changes, 0 if length.is_inference() else length._version

    def _known(self, held):
        """The slots' lengths after the calls so far: exact, or past the cache's
        where pages were short."""
        self._held, self._held_at = held, self._state()

    def _fork(self, src, dst):
        self.cache.fork(*self._ints(src, dst))
        held = list(self._held)
        for a, b in zip(src, dst):
            held[b] = self._held[a]
        self._known(held)

    def _lengths_after(self, slots, lengths):
        """The requests' lengths after `lengths` more tokens; ValueError if one
        would pass the model's positions.  The cache's own lengths are read (the
        host waits) only where they changed by other hands, or to refuse."""
        after = [self._held[s] + n for s, n in zip(slots, lengths)]
        if self._held_at != self._state() or max(after) > self.m.cfg.positions:
            self._known(self.cache.length.tolist())
            after = [self._held[s] + n for s, n in zip(slots, lengths)]
            if max(after) > self.m.cfg.positions:
                raise ValueError(f"a request would pass the model's {self.m.cfg.positions} positions")
        return after

    def _ints(self, *lists):
        """Device int32 arrays of some host lists, by one copy."""
        host = torch.tensor([x for values in lists for x in values], dtype=torch.int32).pin_memory()
        return host.to(self.m.device, non_blocking=True).split([len(values) for values in lists])

    def step(self, slots, lengths, ids):
        """Forward lengths[i] new tokens of the request in slot slots[i] (host
        lists; ids: the tokens of all, one request after another, device
        int32), append them to the cache, and return the logits of each
        request's last token, [len(slots), vocab].  cache.shortage tells
        afterwards whether the pages sufficed.  A slot given twice or out of
        range, or a request that would pass the model's positions, is refused
        (ValueError) before anything changes."""
        m, cfg, dev = self.m, self.m.cfg, self.m.device
        _need_cuda(ids, "ids", torch.int32)
        if ids.device != self.cache.pool.device:
            raise HyqError(-1, "ids: on another device")
        rows, n = sum(lengths), len(slots)
        if n == 0 or len(lengths) != n or min(lengths) < 1 or ids.numel() != rows:
            raise ValueError("at least one new token per request, and one id per new token")
        if len(set(slots)) != n or min(slots) < 0 or max(slots) >= self.slots:
            raise ValueError(f"slots of a step are distinct, from 0 to {self.slots - 1}")
        after = self._lengths_after(slots, lengths)
        if rows > self.acts.M:
            self.acts = _Acts(cfg, rows, dev)
        a = self.acts
        ends = torch.tensor(lengths).cumsum(0).tolist()
        slot, extra, row_start = self._ints(slots, lengths, [0] + ends)
        pos = self.cache.reserve(slot, extra)
        held = list(self._held)
        for s, length in zip(slots, after):
            held[s] = length
        self._known(held)
        q, k, v, attended = (t[:rows].view(rows, -1, cfg.head_dim) for t in (a.q, a.k, a.v, a.attended))
        logits = torch.empty(n, cfg.vocab, device=dev)
        st, fused = m._stream(), m.precision == quant.GEMM_F32
        with quant.gemm_precision(m.precision):
            check(lib.hyq_embed(m.embed.handle, _p(ids), rows, _p(a.hidden), st))
            delta = None
            for i, W in enumerate(m.layers):
                k_pages, v_pages = self.cache.layer(i)
                _qkv_normed(fused, W, _p(a.hidden), delta, _p(W["input_norm"]), cfg.eps, rows, _p(a.normalized),
                            (_p(a.q), _p(a.k), _p(a.v)), st)
                paged.rope_append(q, k, v, k_pages, v_pages, self.cache.table, row_start, pos, self.cos, self.sin,
                                  W["q_norm"], W["k_norm"], cfg.eps, bool(m.norm_first), slot=slot, out=q)
                paged.attention(q, k_pages, v_pages, self.cache.table, row_start, pos, max(lengths),
                                max(after), slot=slot, out=attended, workspace=self.workspace)
                check(lib.hyq_matmul(W["o"].handle, _p(a.attended), rows, _p(a.projected), st))
                if "moe" in W:
                    _add_norm(_p(a.hidden), _p(a.projected), _p(W["ffn_norm"]), cfg.hidden, rows, cfg.eps,
                              _p(a.normalized), st)
                    W["moe"].forward(a.normalized[:rows], rows, out=a.ff)
                else:
                    _gate_up_normed(fused, W, _p(a.hidden), _p(a.projected), _p(W["ffn_norm"]), cfg.eps, rows,
                                    _p(a.normalized), _p(a.gate), st)
                    check(lib.hyq_matmul(W["down"].handle, _p(a.gate), rows, _p(a.ff), st))
                delta = _p(a.ff)
            # the output norm and the lm_head of each request's last row only
            last = (row_start[1:] - 1).long()
            hidden, ff = a.hidden.index_select(0, last), a.ff.index_select(0, last)
            normalized = torch.empty_like(hidden)
            _matmul_normed(fused, m.output, _p(hidden), _p(ff), _p(m.output_norm), cfg.eps, n, _p(normalized), _p(logits),
                           st)
        return logits

    def generate(self, prompts, n_new, answers=1, temperature=0.0, top_k=None, top_p=None, min_p=None, seed=0):
        """n_new tokens of each of `answers` answers to each prompt (lists of
        ids): [prompt][answer][token].  A prompt's answers share its full pages
        (PagedCache.fork).  The sampling parameters hold for all requests
        (temperature 0: greedy); `seed` seeds the uniform numbers.  The tokens
        stay on the device until the end."""
        dev, used = self.m.device, len(prompts) * answers
        if not prompts or min(len(p) for p in prompts) < 1 or answers < 1 or n_new < 1:
            raise ValueError("at least one prompt token, answer and new token")
        if used > self.slots:
            raise ValueError(f"{used} answers need as many slots, there are {self.slots}")
        if max(len(p) for p in prompts) + n_new > self.m.cfg.positions:
            raise ValueError("prompt + generated tokens exceed the rotary tables")
        random = torch.Generator(device=dev).manual_seed(seed)
        prompt_ids = self._ints(*prompts)
        fed = [0] * len(prompts)
        latest = torch.zeros(self.slots, dtype=torch.int32, device=dev)     # each slot's last token
        out = torch.zeros(self.slots, n_new, dtype=torch.int32, device=dev)
        made = {}                                                           # decoding slot: its tokens so far
        short = torch.zeros(1, dtype=torch.int32, device=dev)
        self.cache.free(self._ints(range(self.slots))[0])
        self._known([0] * self.slots)
        while True:
            # a token of every decoding request, then prompt tokens
            slots = [s for s, count in made.items() if count < n_new]
            lengths, parts, room, complete = [1] * len(slots), [], self.chunk, []
            sources = list(zip(range(len(slots)), slots))                   # (logits row, slot) of the tokens to come
            if slots:
                parts.append(latest.index_select(0, self._ints(slots)[0]))
            for i, ids in enumerate(prompt_ids):
                count = min(room, ids.numel() - fed[i])
                if count > 0:
                    parts.append(ids[fed[i]:fed[i] + count])
                    fed[i] += count
                    room -= count
                    if fed[i] == ids.numel():
                        complete.append(i)
                        sources += [(len(slots), i * answers + j) for j in range(answers)]
                    slots.append(i * answers)
                    lengths.append(count)
            if not slots:
                break
            logits = self.step(slots, lengths, torch.cat(parts))
            torch.maximum(short, self.cache.shortage, out=short)
            if complete and answers > 1:
                self._fork([i * answers for i in complete for _ in range(1, answers)],
                           [i * answers + j for i in complete for j in range(1, answers)])
                torch.maximum(short, self.cache.shortage, out=short)
            if not sources:
                continue
            row, slot, column = self._ints([r for r, _ in sources], [s for _, s in sources],
                                           [made.get(s, 0) for _, s in sources])
            token, _ = sampling.sample(logits.index_select(0, row), torch.rand(len(sources), generator=random, device=dev),
                                       temperature, top_k, top_p, min_p)
            latest[slot.long()] = token
            out[slot.long(), column.long()] = token
            for _, s in sources:
                made[s] = made.get(s, 0) + 1
        if int(short.item()):
            raise RuntimeError(f"the cache lacked {int(short.item())} pages")
        result = out[:used].cpu().tolist()
        return [result[i:i + answers] for i in range(0, used, answers)]
