"""Requests over one paged cache (hy_mt_rs_b200.serving.PagedBatch): chunked
prompts mixed with decoding rows, forks and compaction must give each request
the logits and tokens it gets alone (DenseModel.generate).

Tolerances, on the relative 2-norm of a logits row.  f32 cache, split-operand
products: both sides compute every product and the attention to about 1e-6
and differ in the order of their sums; 3 layers with ~6 roundings each in
series, amplified by the norms and the softmax by less than 4, stay below
1e-4.  f16 cache: keys and values that differ by 1e-6 round to different
halves (2^-11 apart) for 1 element in ~2^11 * 1e-6 = 1/500, an error of
2^-11 / sqrt(500) = 2.2e-5 a layer on top; 1e-3 bounds it with the same
factors."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _model(cuda, arch, kv16):
    import torch
    from hy_mt_rs_b200 import quant
    from hy_mt_rs_b200.model import DenseConfig, DenseModel, random_weights

    if arch == "dense":
        cfg = DenseConfig(layers=3, vocab=8192, ffn=2048, positions=128)
    else:
        cfg = DenseConfig(arch="hyv3", layers=2, vocab=8192, ffn=2048, positions=128, linear_dtype=2, expert_ffn=512,
                          shared_ffn=512, experts=16, experts_used=4)
    weights = random_weights(cfg, cuda, seed=11)
    torch.cuda.synchronize()
    return DenseModel(cfg, weights, cuda, kv16=kv16, gemm_precision=quant.GEMM_F32)


def _alone(model, prompts, n_new):
    import torch
    from hy_mt_rs_b200 import quant

    stream = torch.cuda.Stream(model.device)
    ids, logits = [], []
    try:
        for p in prompts:
            lg = torch.zeros(n_new, model.cfg.vocab, device=model.device)
            ids.append(model.generate(p, n_new, stream, logits_out=lg, batched_prefill=True))
            logits.append(lg.cpu().numpy())
    finally:
        quant.set_launch_overlap(False)
    return ids, logits


def _close(got, want, tol):
    return np.linalg.norm(got - want) <= tol * np.linalg.norm(want)


@pytest.mark.parametrize("arch,kv16", [("dense", False), ("dense", True), ("hyv3", True)])
def test_steps_match_single_requests(cuda, arch, kv16):
    """Teacher-forced: each step's logits against the request's own decode,
    with a fork and a compaction on the way."""
    import torch
    from hy_mt_rs_b200 import quant
    from hy_mt_rs_b200.serving import PagedBatch

    model = _model(cuda, arch, kv16)
    tol = 1e-3 if kv16 else 1e-4
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, model.cfg.vocab, n).tolist() for n in (37, 1, 70)]
    n_new = 5
    ids, logits = _alone(model, prompts, n_new)
    batch = PagedBatch(model, 6, page_size=16)
    put = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731

    def check(got, wanted):
        got = got.cpu().numpy()
        for g, (r, i) in zip(got, wanted):
            assert _close(g, logits[r][i], tol), (r, i)

    # a request that is gone before the others end leaves holes in the pool
    batch.step([5], [50], put(rng.integers(0, model.cfg.vocab, 50)))
    batch.step([2, 0], [40, 37], put(prompts[2][:40] + prompts[0]))
    # the last 30 tokens of a prompt beside a decoding token and a prompt of one
    got = batch.step([0, 2, 3], [1, 30, 1], put(ids[0][:1] + prompts[2][40:] + prompts[1]))
    check(got, [(0, 1), (2, 0), (1, 0)])
    batch.cache.free(put([5]))
    batch.cache.fork(put([2]), put([4]))
    batch.cache.compact()
    for i in range(1, n_new - 1):
        got = batch.step([4, 3, 0, 2], [1] * 4, put([ids[2][i - 1], ids[1][i - 1], ids[0][i], ids[2][i - 1]]))
        check(got, [(2, i), (1, i), (0, i + 1), (2, i)])
    assert int(batch.cache.shortage.item()) == 0
    assert quant.device_status() == 0


def test_generate(cuda):
    """Greedy answers are the requests' own; answers of one prompt and of
    equal seeds agree as they must; the filters reach the sampler."""
    from hy_mt_rs_b200 import quant
    from hy_mt_rs_b200.serving import PagedBatch

    model = _model(cuda, "dense", True)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, model.cfg.vocab, n).tolist() for n in (20, 90, 3)]
    n_new = 6
    ids, logits = _alone(model, prompts, n_new)
    batch = PagedBatch(model, 9, page_size=32, chunk=48)    # the second prompt takes several steps
    greedy = batch.generate(prompts, n_new, answers=3)
    for r in range(len(prompts)):
        assert greedy[r][0] == greedy[r][1] == greedy[r][2]
        for i, (a, b) in enumerate(zip(greedy[r][0], ids[r])):
            if a != b:   # only where the two best logits are as close as the tolerance
                top = np.sort(logits[r][i])[-2:]
                assert top[1] - top[0] <= 2e-3 * np.linalg.norm(logits[r][i])
                break
    assert batch.generate(prompts, n_new, temperature=1.0, top_k=1) == [[g[0]] for g in greedy]
    drawn = batch.generate(prompts, n_new, answers=3, temperature=1.5, top_k=50, top_p=0.95, min_p=0.01, seed=7)
    assert drawn == batch.generate(prompts, n_new, answers=3, temperature=1.5, top_k=50, top_p=0.95, min_p=0.01, seed=7)
    assert any(len({tuple(a) for a in answers}) > 1 for answers in drawn)
    assert all(0 <= t < model.cfg.vocab for answers in drawn for a in answers for t in a)
    assert quant.device_status() == 0


def test_out_of_pages(cuda):
    import torch
    from hy_mt_rs_b200 import quant
    from hy_mt_rs_b200.serving import PagedBatch

    model = _model(cuda, "dense", True)
    batch = PagedBatch(model, 2, pages=3, page_size=16)
    with pytest.raises(RuntimeError, match="pages"):
        batch.generate([list(range(40)), list(range(20))], 4)
    quant.device_status()    # the rows without a page are reported there too: read and clear
    assert len(batch.generate([list(range(40))], 4)[0][0]) == 4
    assert quant.device_status() == 0
    with pytest.raises(ValueError):
        batch.generate([[1], [2], [3]], 1)
    with pytest.raises(ValueError):
        batch.step([0], [2], torch.zeros(1, dtype=torch.int32, device=cuda))
