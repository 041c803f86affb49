"""PagedBatch over 8-bit caches, with prefixes shared by forked requests, and with
penalties, biases and masks on its logits."""
import numpy as np
import pytest

from test_gpu_serving import _close, _model

pytestmark = pytest.mark.gpu


def _put(x, cuda):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=cuda)


def _one_layer(cuda, positions=512):
    import torch
    from hy_mt_rs_b200 import quant
    from hy_mt_rs_b200.model import DenseConfig, DenseModel, random_weights
    cfg = DenseConfig(layers=1, vocab=4096, ffn=1024, positions=positions)
    weights = random_weights(cfg, cuda, seed=12)
    torch.cuda.synchronize()
    return DenseModel(cfg, weights, cuda, gemm_precision=quant.GEMM_F32)


@pytest.mark.parametrize("dtype", ["int8", "float8_e4m3fn"])
def test_chunks_match_single_tokens(cuda, dtype):
    """One layer, whose keys and values come from the embeddings alone: the products
    of a chunk and of single tokens differ by 1e-6 of a row at most (f32 accuracy), so
    a code differs for about one value in 10^3 (int8: steps of 2^-7 of the largest),
    by one step: with 2^-7 / sqrt(10^3) = 2.5e-4 of a row's norm for int8 and four times
    that for e4m3's steps of 2^-4, attention of 100 rows stays below 1e-3.  Forks,
    compaction, the pages' scales among what they move."""
    import torch
    from hy_mt_rs_b200 import quant
    from hy_mt_rs_b200.serving import PagedBatch
    model = _one_layer(cuda)
    rng = np.random.default_rng(6)
    prompts = [rng.integers(0, model.cfg.vocab, n).tolist() for n in (75, 100)]
    batch, single = (PagedBatch(model, 5, page_size=16, kv_dtype=getattr(torch, dtype)) for _ in range(2))
    batch.step([4], [40], _put(rng.integers(0, model.cfg.vocab, 40), cuda))       # leaves a hole
    got = batch.step([0, 2], [74, 99], _put(prompts[0][:-1] + prompts[1][:-1], cuda))
    batch.cache.free(_put([4], cuda))
    batch.cache.fork(_put([2], cuda), _put([1], cuda))
    batch.cache.compact()
    got = batch.step([0, 2, 1], [1, 1, 1], _put([prompts[0][-1], prompts[1][-1], prompts[1][-1]], cuda))
    assert torch.equal(got[1], got[2])
    for i, slot in enumerate((0, 1)):
        for t in prompts[i]:
            want = single.step([slot], [1], _put([t], cuda))
        assert _close(got[i].cpu().numpy(), want[0].cpu().numpy(), 1e-3)
    # and near the f32 cache's: a key or value is off by half a step at most, 2^-8 of
    # its row's largest magnitude (int8) or 2^-4 of itself (e4m3); rows of 128 normal
    # values have a largest of about 2.6 and a step's rms is 1 / sqrt(12), so scores and
    # outputs move by 0.6 % and 3 % of a row at most
    full = PagedBatch(model, 5, page_size=16)
    full.step([0, 2], [74, 99], _put(prompts[0][:-1] + prompts[1][:-1], cuda))
    want = full.step([0, 2], [1, 1], _put([prompts[0][-1], prompts[1][-1]], cuda))
    off = float((got[:2] - want).norm() / want.norm())
    assert off <= (0.02 if dtype == "int8" else 0.1), off
    assert quant.device_status() == 0


@pytest.mark.parametrize("dtype", [None, "int8"])
def test_forked_requests_share_their_prefix(cuda, dtype, monkeypatch):
    """Steps of forked requests go through attention_shared, with the groups that the
    forks made; its kernels (whatever the sizes) give attention's logits."""
    import torch
    from hy_mt_rs_b200 import paged, quant
    from hy_mt_rs_b200.serving import PagedBatch
    model = _one_layer(cuda)
    rng = np.random.default_rng(7)
    prompts = [rng.integers(0, model.cfg.vocab, n).tolist() for n in (130, 40)]
    calls = []
    shared = paged.attention_shared

    def watched(*args, **kw):
        calls.append((args[6].tolist(), args[7].tolist()))
        return shared(*args, **kw)

    def logits(bound=None):
        batch = PagedBatch(model, 6, page_size=16, kv_dtype=getattr(torch, dtype) if dtype else None)
        batch.step([0, 3], [130, 40], _put(prompts[0] + prompts[1], cuda))
        batch._fork([0, 0, 3], [1, 2, 4])
        out = []
        for i in range(3):
            out.append(batch.step([0, 1, 2, 5, 3, 4] if i else [0, 1, 2, 3, 4], [1] * (6 if i else 5),
                                  _put([5 + i, 6, 7, 9, 8, 9] if i else [5, 6, 7, 8, 9], cuda)))
        batch.cache.free(_put([1], cuda))       # by other hands: what was known of prefixes is dropped
        out.append(batch.step([0, 2], [1, 1], _put([1, 2], cuda)))
        return batch, out

    monkeypatch.setattr(paged, "attention_shared", watched)
    _, got = logits()
    assert calls[0] == ([0, 3, 5], [130, 40]) and calls[1] == ([0, 3, 4, 6], [130, 0, 40])
    assert len(calls) == 3
    # without groups
    monkeypatch.setattr(PagedBatch, "_groups", lambda *a: None)
    _, want = logits()
    for a, b in zip(got, want):
        assert torch.equal(a, b)                # small prefixes are not worth their kernels: the same bits
    monkeypatch.undo()

    # as if they were: a cache whose table reaches far, and no bound
    def forced(*args, **kw):
        args = list(args)
        args[3] = torch.nn.functional.pad(args[3], (0, 20000), value=-1)
        return shared(*args[:9], None, None, **kw)

    monkeypatch.setattr(paged, "attention_shared", forced)
    _, got = logits()
    for a, b in zip(got, want):
        assert _close(a.cpu().numpy(), b.cpu().numpy(), 1e-4)
    assert not all(torch.equal(a, b) for a, b in zip(got, want))
    assert quant.device_status() == 0


def test_generate_with_adjusted_logits(cuda):
    """Greedy answers under penalties, biases and a mask are those of a loop over
    step() that applies the rule on the host."""
    import torch
    from hy_mt_rs_b200.serving import PagedBatch
    from test_gpu_adjust import _expected
    model = _model(cuda, "dense", True)
    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, model.cfg.vocab, n).tolist() for n in (20, 33)]
    vocab, n_new = model.cfg.vocab, 6
    words = np.stack([rng.integers(-2 ** 31, 2 ** 31, vocab // 32), np.full(vocab // 32, -1)]).astype(np.int32)
    bias = {5: 3.0, 17: -100.0, vocab - 1: 2.5}
    for kw in (dict(repetition=1.3), dict(presence=0.7, frequency=0.2), dict(bias=bias), dict(mask=words),
               dict(repetition=1.2, frequency=0.1, bias=bias, mask=words)):
        batch = PagedBatch(model, 4, page_size=32)
        given = {**kw, **({"mask": torch.from_numpy(words).to(cuda)} if "mask" in kw else {})}
        got = batch.generate(prompts, n_new, answers=2, **given)
        alone = PagedBatch(model, 1, page_size=32)
        for i, prompt in enumerate(prompts):
            assert got[i][0] == got[i][1]
            made = []
            for step in range(n_new):
                if step == 0:
                    alone.cache.free(_put([0], cuda))
                    x = alone.step([0], [len(prompt)], _put(prompt, cuda))
                else:
                    x = alone.step([0], [1], _put(made[-1:], cuda))
                past = prompt + made
                c = dict(history=[past], length=[len(past)], prompt=[len(prompt)], slot=[0])
                c.update({k: [kw[k]] for k in ("repetition", "presence", "frequency") if k in kw})
                if "bias" in kw:
                    c["bias"] = ([0, len(bias)], list(bias), list(bias.values()))
                if "mask" in kw:
                    c.update(mask=words, mask_row=[i])
                y = _expected(x.cpu().numpy(), c)[0]
                best = int(y.argmax())
                if got[i][0][step] != best:    # only where the two are as close as other batches' roundings
                    assert abs(y[got[i][0][step]] - y[best]) <= 2e-3 * np.linalg.norm(y[np.isfinite(y)])
                    break
                made.append(best)


def test_generate_wants_a_mask_for_all_or_for_each_prompt(cuda):
    import torch
    from hy_mt_rs_b200.serving import PagedBatch
    model = _model(cuda, "dense", True)
    batch = PagedBatch(model, 3, page_size=32)
    words = torch.full((2, (model.cfg.vocab + 31) // 32), -1, dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError, match="2 masks for 3 prompts"):
        batch.generate([[1], [2], [3]], 2, mask=words)
    assert batch.generate([[1], [2]], 2, mask=words) == batch.generate([[1], [2]], 2)
