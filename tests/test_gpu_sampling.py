"""GPU parity of hyq_sample: every token against the rule in whole numbers
(include/hyq.h), and the distribution against the probabilities."""
import math
import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _rule(x, temperature, k, p, min_p, u, e_of):
    """One row by the rule, in Python integers: (token, kept weight, total).
    e_of: the f32 exponentials of (x - max) * (1 / temperature)."""
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float32)
    top = x.max()
    if top == -np.inf:
        return 0, 0, 1
    if not temperature > 0:
        return int(np.argmax(x)), 1, 1
    e = e_of(x, top, temperature)
    order = np.argsort(-x.astype(np.float64), kind="stable")
    if 0 < k < len(x):
        order = order[:k]
    w = [int(np.float64(e[i]) * 2.0 ** 40) for i in order]
    if p < 1:
        share = math.ceil(max(float(np.float32(p)), 0.0) * 2 ** 24)
        limit = max(1, (sum(w) * share + 2 ** 24 - 1) >> 24)
        run, keep = 0, 0
        for v in w:
            if run >= limit:
                break
            run += v
            keep += 1
        order, w = order[:keep], w[:keep]
    floor = np.float32(min(min_p, 1.0))
    kept = {int(i): v for i, v in zip(order, w) if e[i] >= floor}
    total = sum(kept.values())
    aim = total * min(int(float(np.float32(u)) * 2 ** 24), 2 ** 24 - 1) >> 24
    run = 0
    for i in sorted(kept):
        run += kept[i]
        if run > aim:
            return i, kept[i], total
    raise AssertionError


def _exps(cuda):
    """f32 exponentials of the device (the weights are defined on them)."""
    import torch

    def e_of(x, top, temperature):
        if np.isinf(top):
            return (x == top).astype(np.float32)
        t = torch.from_numpy(x).to(cuda)
        inv = torch.ones((), device=cuda) / torch.tensor(temperature, dtype=torch.float32, device=cuda)
        return torch.exp((t - t.max()) * inv).cpu().numpy()
    return e_of


def _check(cuda, x, temperature, k, p, min_p, u):
    import torch
    from hy_mt_rs_b200 import quant, sampling
    f = lambda v: torch.tensor(v, dtype=torch.float32).to(cuda)  # noqa: E731
    token, prob = sampling.sample(x, f(u), f(temperature), torch.tensor(k, dtype=torch.int32).to(cuda), f(p), f(min_p))
    token, prob, rows = token.tolist(), prob.tolist(), x.cpu().numpy()
    e_of = _exps(cuda)
    for r in range(len(u)):
        want, w, total = _rule(rows[r], np.float32(temperature[r]), k[r], np.float32(p[r]), np.float32(min_p[r]), u[r], e_of)
        assert token[r] == want, (r, token[r], want, temperature[r], k[r], p[r], min_p[r], u[r])
        # two f32 conversions and one division
        assert abs(prob[r] - w / total) <= 4 * 2.0 ** -24 * w / total
    assert quant.device_status() == 0


def _params(rows, rng, n):
    ks = [0, 1, 2, 5, 40, n - 1 if n > 1 else 0, n, n + 7, -3, max(1, n // 3)]
    return ([rng.choice([0.0, 0.2, 0.7, 1.0, 1.7, -1.0]) for _ in range(rows)], [rng.choice(ks) for _ in range(rows)],
            [rng.choice([0.0, 0.1, 0.5, 0.9, 0.999, 1.0, 1.5]) for _ in range(rows)],
            [rng.choice([0.0, 0.0, 0.05, 0.5, 1.0, 2.0, -1.0]) for _ in range(rows)],
            [rng.choice([0.0, rng.random(), rng.random(), rng.random(), 1 - 2.0 ** -24, 1.0]) for _ in range(rows)])


@pytest.mark.parametrize("n", [1, 2, 3, 31, 32, 33, 255, 1000, 1025, 4097, 31999, 120832, 151937])
def test_rows_by_the_rule(cuda, n):
    import torch
    rows, rng = 24, random.Random(n)
    g = torch.Generator(device=cuda).manual_seed(n)
    x = torch.randn(rows, n, generator=g, device=cuda) * 3
    x[:4] = x[:4].bfloat16().float()                         # ties
    x[4:8] = (x[4:8] * 2).round() / 2                        # many ties
    x[8] = 1.25                                              # all equal
    x[9] = torch.where(torch.rand(n, generator=g, device=cuda) < 0.9, -math.inf, x[9])   # masked
    x[10] = torch.where(torch.rand(n, generator=g, device=cuda) < 0.5, math.nan, x[10])
    x[11] = -3e38                                            # the lowest values there are
    x[12] = torch.finfo(torch.float32).min
    x[12, n // 2] = 0
    x[13] *= 100                                             # weights down to nothing
    x[14] = 0.0
    x[14, ::2] = -0.0                                        # zeros of both signs tie
    _check(cuda, x, *_params(rows, rng, n))


@pytest.mark.parametrize("rows", [1, 2, 37, 150, 400])
def test_batches(cuda, rows):
    import torch
    rng = random.Random(rows)
    g = torch.Generator(device=cuda).manual_seed(rows)
    x = torch.randn(rows, 5003, generator=g, device=cuda) * 2.5
    _check(cuda, x, *_params(rows, rng, 5003))


@pytest.mark.parametrize("n", [400000, 1000003])
def test_long_rows(cuda, n):
    import torch
    rng = random.Random(n)
    x = torch.randn(4, n, generator=torch.Generator(device=cuda).manual_seed(n), device=cuda) * 2.5
    _check(cuda, x, *_params(4, rng, n))


def test_special_rows(cuda):
    """No logit above -inf: token 0 with probability 0.  +inf logits share
    everything; greedy takes the first of equal maxima."""
    import torch
    from hy_mt_rs_b200 import sampling
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf, -inf, -inf, -inf], [nan, nan, nan, nan], [nan, -inf, nan, -inf], [0., inf, 1., inf],
                      [0., inf, 1., inf], [2., 5., 5., nan], [-inf, nan, -1e30, -inf]], device=cuda)
    u = torch.tensor([0.3, 0.3, 0.9, 0.49, 0.51, 0.9, 0.99], device=cuda)
    temperature = torch.tensor([1., 1., 0., 1., 1., 0., 1.], device=cuda)
    for kw in (dict(), dict(top_k=3), dict(top_p=0.999), dict(min_p=0.5), dict(top_k=2, top_p=0.9, min_p=0.1)):
        token, prob = sampling.sample(x, u, temperature, **kw)
        assert token.tolist() == [0, 0, 0, 1, 3, 1, 2]
        assert prob.tolist() == [0, 0, 0, 0.5, 0.5, 1, 1]


def test_strided_rows_and_given_outputs(cuda):
    import torch
    from hy_mt_rs_b200 import sampling
    g = torch.Generator(device=cuda).manual_seed(0)
    for start, n in ((0, 1001), (1, 999), (3, 1000)):
        wide = torch.randn(9, 1037, generator=g, device=cuda) * 3
        x = wide[:, start:start + n]
        u = torch.rand(9, generator=g, device=cuda)
        token, prob = torch.empty(9, dtype=torch.int32, device=cuda), torch.empty(9, device=cuda)
        sampling.sample(x, u, 0.8, 50, 0.9, token=token, prob=prob)
        t2, p2 = sampling.sample(x.contiguous(), u, 0.8, 50, 0.9)
        assert torch.equal(token, t2) and torch.equal(prob, p2)


def test_distribution(cuda):
    """65,536 draws of one row on a grid of u: each token comes up as often as
    its share says, within the grid's step and the weights' rounding."""
    import torch
    from hy_mt_rs_b200 import sampling
    x = torch.randn(300, generator=torch.Generator().manual_seed(0)) * 2
    draws = 65536
    u = (torch.arange(draws, dtype=torch.float32) + 0.5) / draws
    token, prob = sampling.sample(x.to(cuda).expand(draws, 300).contiguous(), u.to(cuda), 0.9, top_k=100)
    e = torch.exp((x.double() - x.max()) / 0.9)
    e[torch.argsort(x, descending=True)[100:]] = 0
    share = e / e.sum()
    count = torch.bincount(token.cpu().long(), minlength=300).double() / draws
    # f32 scores of magnitude up to 15: 15 * 2^-23 relative on each weight
    assert float((count - share).abs().max()) <= 1.5 / draws
    assert float((prob.cpu().double() - share[token.cpu().long()]).abs().max()) <= 4e-6


def test_repeats_and_streams(cuda):
    import torch
    from hy_mt_rs_b200 import sampling
    g = torch.Generator(device=cuda).manual_seed(0)
    x = torch.randn(64, 20001, generator=g, device=cuda) * 2
    u = torch.rand(64, generator=g, device=cuda)
    first = sampling.sample(x, u, 1.0, 0, 0.95)[0].clone()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        again = sampling.sample(x, u, 1.0, 0, 0.95)[0]
    st.synchronize()
    assert torch.equal(first, again)
    one = torch.cat([sampling.sample(x[i:i + 1], u[i:i + 1], 1.0, 0, 0.95)[0] for i in range(64)])
    assert torch.equal(first, one)      # a row's token does not depend on the batch


@pytest.mark.parametrize("rows", [3, 40, 150])
def test_launch_overlap(cuda, rows):
    """With kernels launched before their predecessors have ended, what follows
    a call still sees its tokens, and a call what precedes it."""
    import torch
    from hy_mt_rs_b200 import quant, sampling
    g = torch.Generator(device=cuda).manual_seed(rows)
    logits = torch.randn(rows, 30011, generator=g, device=cuda) * 3
    u = torch.rand(rows, generator=g, device=cuda)
    i = torch.arange(rows, device=cuda)
    temperature = torch.tensor([0.0, 0.8, 1.2, 1.0], device=cuda)[i % 4]
    top_k = torch.tensor([0, 40, 500], dtype=torch.int32, device=cuda)[i % 3]
    top_p = torch.tensor([1.0, 0.9], device=cuda)[i % 2]
    want, _ = sampling.sample(logits, u, temperature, top_k, top_p)
    second, _ = sampling.sample(logits.roll(1, 0).contiguous(), u, temperature, top_k, top_p)
    x, token, again = torch.empty_like(logits), torch.empty_like(want), torch.empty_like(want)
    quant.set_launch_overlap(True)
    try:
        for _ in range(10):
            token.fill_(-1)
            x.copy_(logits)
            sampling.sample(x, u, temperature, top_k, top_p, token=token)
            sampling.sample(x, u, temperature, top_k, top_p, token=again)
            x.copy_(logits.roll(1, 0))
            assert torch.equal(token, want) and torch.equal(again, want)
            sampling.sample(x, u, temperature, top_k, top_p, token=token)
            assert torch.equal(token, second)
    finally:
        quant.set_launch_overlap(False)
