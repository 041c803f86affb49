"""PagedBatch.step: arguments that must not reach the cache, and the lengths it
keeps for the attention calls."""
import numpy as np
import pytest

from test_gpu_serving import _alone, _close, _model

pytestmark = pytest.mark.gpu


def _put(x, cuda):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=cuda)


@pytest.mark.parametrize("kv16", [True, False])
def test_step_refuses_what_would_spoil_others(cuda, kv16):
    """A request at the end of the positions, a slot given twice, out of range:
    ValueError before any launch; the other requests' pages stay bit for bit
    and their next logits are what they would have been."""
    import torch
    from hy_mt_rs_b200 import quant
    from hy_mt_rs_b200.serving import PagedBatch

    model = _model(cuda, "dense", kv16)
    end = model.cfg.positions
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, model.cfg.vocab, n).tolist() for n in (30, 21, end)]
    batches = [PagedBatch(model, 4, page_size=16) for _ in range(2)]
    for b in batches:
        b.step([0, 1, 2], [30, 21, end], _put(sum(prompts, []), cuda))
    batch, other = batches
    pool = batch.cache.pool.clone()
    state = [t.clone() for t in (batch.cache.table, batch.cache.length, batch.cache.refs)]
    for slots, lengths in (([0, 1, 2], [1, 1, 1]), ([0, 1, 0], [1, 1, 1]), ([0, 4], [1, 1]), ([0, -1], [1, 1]),
                           ([0, 3], [1, end + 1]), ([1, 0], [end - 20, 1])):
        with pytest.raises(ValueError):
            batch.step(slots, lengths, _put([1] * sum(lengths), cuda))
        assert torch.equal(batch.cache.pool, pool)
        for a, b in zip(state, (batch.cache.table, batch.cache.length, batch.cache.refs)):
            assert torch.equal(a, b)
    ids = _put([11, 12], cuda)
    assert torch.equal(batch.step([0, 1], [1, 1], ids), other.step([0, 1], [1, 1], ids))
    assert quant.device_status() == 0


def test_lengths_follow_the_cache(cuda):
    """Slots freed or forked through the cache itself, and steps that found no
    pages, neither refuse a request that fits nor let one through that does
    not."""
    from hy_mt_rs_b200 import quant
    from hy_mt_rs_b200.serving import PagedBatch

    model = _model(cuda, "dense", True)
    end = model.cfg.positions
    batch = PagedBatch(model, 3, page_size=16, pages=end // 16 + 2)
    batch.step([0], [end], _put([1] * end, cuda))
    with pytest.raises(ValueError):
        batch.step([0], [1], _put([1], cuda))
    batch.cache.free(_put([0], cuda))
    batch.step([0], [end - 1], _put([1] * (end - 1), cuda))
    batch.cache.fork(_put([0], cuda), _put([1], cuda))
    batch.step([1], [1], _put([1], cuda))
    with pytest.raises(ValueError):
        batch.step([1], [1], _put([1], cuda))
    batch.step([2], [end], _put([1] * end, cuda))       # no pages are left for that many
    assert batch.cache.shortage.item() > 0
    quant.device_status()
    batch.step([2], [10], _put([1] * 10, cuda))         # but for these
    assert batch.cache.shortage.item() == 0 and batch.cache.length.tolist() == [end - 1, end, 10]
    assert quant.device_status() == 0


@pytest.mark.parametrize("kv16", [True, False])
def test_attention_gets_the_longest_length(cuda, kv16, monkeypatch):
    """The bound that the choice of attention kernels goes by."""
    from hy_mt_rs_b200 import paged
    from hy_mt_rs_b200.serving import PagedBatch

    model = _model(cuda, "dense", kv16)
    batch = PagedBatch(model, 3, page_size=16)
    seen, call = [], paged.attention

    def record(*a, **kw):
        seen.append((a[6], a[7] if len(a) > 7 else kw.get("max_len")))
        return call(*a, **kw)

    monkeypatch.setattr(paged, "attention", record)
    batch.step([0, 2], [20, 9], _put([1] * 29, cuda))
    batch.step([0, 1], [1, 7], _put([1] * 8, cuda))
    batch.step([2], [1], _put([1], cuda))
    n = len(model.layers)
    assert seen == [(20, 20)] * n + [(7, 21)] * n + [(1, 10)] * n


def test_arguments_are_checked(cuda):
    import torch
    from hy_mt_rs_b200._native import HyqError
    from hy_mt_rs_b200.serving import PagedBatch

    model = _model(cuda, "dense", True)
    for kw in (dict(chunk=0), dict(chunk=-4), dict(page_size=0)):
        with pytest.raises(ValueError):
            PagedBatch(model, 2, **{"page_size": 16, **kw})
    batch = PagedBatch(model, 2, page_size=16)
    for ids in (torch.zeros(2, dtype=torch.int64, device=cuda), torch.zeros(2, dtype=torch.int32),
                torch.zeros(4, dtype=torch.int32, device=cuda)[::2]):
        with pytest.raises(HyqError):
            batch.step([0], [2], ids)
    assert batch.cache.length.tolist() == [0, 0]


@pytest.mark.parametrize("kv16", [True, False])
def test_long_contexts_match_single_requests(cuda, kv16):
    """Prompts past the lengths of the one-launch chunk kernel, in chunks, beside
    short ones (tolerances of test_gpu_serving)."""
    import torch
    from hy_mt_rs_b200 import quant
    from hy_mt_rs_b200.model import DenseConfig, DenseModel, random_weights
    from hy_mt_rs_b200.serving import PagedBatch

    cfg = DenseConfig(layers=3, vocab=8192, ffn=2048, positions=1024)
    weights = random_weights(cfg, cuda, seed=12)
    torch.cuda.synchronize()
    model = DenseModel(cfg, weights, cuda, kv16=kv16, gemm_precision=quant.GEMM_F32)
    tol = 1e-3 if kv16 else 1e-4
    rng = np.random.default_rng(6)
    prompts = [rng.integers(0, cfg.vocab, n).tolist() for n in (700, 20, 450)]
    ids, logits = _alone(model, prompts, 3)
    batch = PagedBatch(model, 3, page_size=32)
    batch.step([0], [300], _put(prompts[0][:300], cuda))
    batch.step([0, 2], [399, 449], _put(prompts[0][300:699] + prompts[2][:449], cuda))
    got = batch.step([1, 0, 2], [20, 1, 1], _put(prompts[1] + prompts[0][699:] + prompts[2][449:], cuda)).cpu().numpy()
    for g, r in zip(got, (1, 0, 2)):
        assert _close(g, logits[r][0], tol), r
    got = batch.step([0, 1, 2], [1] * 3, _put([i[0] for i in ids], cuda)).cpu().numpy()
    for r, g in enumerate(got):
        assert _close(g, logits[r][1], tol), r
    assert quant.device_status() == 0


def test_under_inference_mode(cuda):
    """A batch made and stepped where tensors have no version counter."""
    import torch
    from hy_mt_rs_b200.serving import PagedBatch

    model = _model(cuda, "dense", True)
    with torch.inference_mode():
        batch = PagedBatch(model, 2, page_size=16)
        batch.step([0], [5], _put([1] * 5, cuda))
        batch.step([0, 1], [1, 3], _put([1] * 4, cuda))
        assert len(batch.generate([[1, 2, 3]], 4, answers=2)[0][1]) == 4
    other = PagedBatch(model, 2, page_size=16)
    other.step([0], [5], _put([1] * 5, cuda))
    assert batch.generate([[5, 6]], 3) == other.generate([[5, 6]], 3)
