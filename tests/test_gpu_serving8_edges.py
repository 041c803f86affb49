"""What PagedBatch takes for shared among forked requests, after calls that lacked
pages and lengths that changed by other hands."""
import numpy as np
import pytest

from test_gpu_serving8 import _one_layer, _put

pytestmark = pytest.mark.gpu


def _watch(monkeypatch):
    from hy_mt_rs_b200 import paged
    calls, shared = [], paged.attention_shared

    def watched(*args, **kw):
        calls.append((args[6].tolist(), args[7].tolist()))
        return shared(*args, **kw)

    monkeypatch.setattr(paged, "attention_shared", watched)
    return calls


def test_nothing_is_shared_after_pages_were_short(cuda, monkeypatch):
    """A generate() that lacked pages may have forked requests whose prompts never came
    in: what they hold afterwards has no common prefix."""
    import torch
    from hy_mt_rs_b200 import quant
    from hy_mt_rs_b200.serving import PagedBatch
    model = _one_layer(cuda)
    ids = np.random.default_rng(3).integers(0, model.cfg.vocab, 100).tolist()
    calls, logits = _watch(monkeypatch), []
    for grouped in (True, False):
        batch = PagedBatch(model, 4, pages=4, page_size=16)
        with pytest.raises(RuntimeError, match="lacked"):
            batch.generate([ids], 3, answers=2)          # 7 pages
        quant.device_status()                            # (the skipped rows' report)
        assert max(batch.cache.length.tolist()) < 100    # (some tokens that were made without it)
        if not grouped:
            monkeypatch.setattr(PagedBatch, "_groups", lambda *a: None)
        calls.clear()
        logits.append([batch.step([0, 1], [1, 1], _put([5 + i, 400 + i], cuda)) for i in range(12)])
        assert not calls
        assert quant.device_status() == 0
    for a, b in zip(*logits):
        assert torch.equal(a, b)


@pytest.mark.parametrize("inference", [False, True])
def test_a_request_taken_back_into_its_prefix(cuda, inference, monkeypatch):
    """Lengths written in place, also of a batch made under inference mode: the forks'
    prefix is no longer taken for shared."""
    import torch
    from hy_mt_rs_b200 import quant
    from hy_mt_rs_b200.serving import PagedBatch
    model = _one_layer(cuda)
    rng = np.random.default_rng(4)
    ids = rng.integers(0, model.cfg.vocab, 80).tolist()
    calls = _watch(monkeypatch)
    with torch.inference_mode(inference):
        batch = PagedBatch(model, 3, page_size=16)
        batch.step([0], [80], _put(ids, cuda))
        batch._fork([0], [1])
        batch.step([0, 1], [1, 1], _put([5, 6], cuda))
        assert calls == [([0, 2], [80])]
        # request 1 goes back to 64 positions (whole pages, which it still shares) on pages
        # of its own from there
        batch.cache.length[1] = 64
        got = [batch.step([0, 1], [1, 20], _put([7] + ids[:20], cuda)), batch.step([0, 1], [1, 1], _put([8, 9], cuda))]
        assert len(calls) == 1
    alone = PagedBatch(model, 2, page_size=16)
    alone.step([0, 1], [80, 64], _put(ids + ids[:64], cuda))
    alone.step([0], [1], _put([5], cuda))
    want = [alone.step([0, 1], [1, 20], _put([7] + ids[:20], cuda)), alone.step([0, 1], [1, 1], _put([8, 9], cuda))]
    # (prompts in other batches: f32 products in another order, 1e-6 of a row, three layers' worth)
    for a, b in zip(got, want):
        assert float((a - b).norm() / b.norm()) <= 1e-4
    assert quant.device_status() == 0
