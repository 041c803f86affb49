"""GPU parity of sampling.adjust (penalties, biases, masks on logits) with the
rule written out token by token.  Every step is one f32 operation, rounded once,
in a stated order: the outputs are equal bit for bit."""
import math
import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _int(v, dev):
    import torch
    return torch.tensor(v, dtype=torch.int32).to(dev)


def _expected(x, c):
    """The rule in numpy float32, one operation at a time."""
    f = np.float32
    out = x.astype(f).copy()
    n = x.shape[1]
    with np.errstate(all="ignore"):
        for r in range(x.shape[0]):
            y = out[r]
            slot = c["slot"][r] if c.get("slot") is not None else r
            if c.get("history") is not None and slot >= 0:
                past = c["history"][slot][:c["length"][slot]]
                prompt = c["prompt"][slot] if c.get("prompt") is not None else 0
                value = lambda name, default: f(c[name][r]) if c.get(name) is not None else f(default)  # noqa: E731
                rep, presence, frequency = value("repetition", 1), value("presence", 0), value("frequency", 0)
                if not rep > 0:
                    rep = f(1)
                made = {}
                for t in past[prompt:]:
                    made[t] = made.get(t, 0) + 1
                for t in set(past):
                    if 0 <= t < n:
                        y[t] = y[t] / rep if y[t] > 0 else y[t] * rep
                        if t in made:
                            y[t] = y[t] - f(f(frequency * f(made[t])) + presence)
            if c.get("bias") is not None:
                start, token, bias = c["bias"]
                last = {token[i]: i for i in range(start[r], start[r + 1])}
                for t, i in last.items():
                    if 0 <= t < n:
                        y[t] = y[t] + f(bias[i])
            if c.get("mask") is not None:
                m = c["mask_row"][r] if c.get("mask_row") is not None else r
                if m >= 0:
                    t = np.arange(n)
                    y[((c["mask"][m][t // 32].astype(np.int64) >> (t % 32)) & 1) == 0] = -np.inf
    return out


def _case(rows, n, width, seed, biases=5, masks=2, slots=None):
    rng = random.Random(seed)
    slots = slots or rows + 2
    length = [rng.choice([0, 1, width, rng.randint(0, width)]) for _ in range(slots)]
    hot = [rng.randrange(n) for _ in range(9)] + [0, n - 1]
    token = lambda: rng.choice(hot) if rng.random() < 0.5 else rng.randrange(n)  # noqa: E731
    counts = [rng.randint(0, biases) for _ in range(rows)]
    start = [sum(counts[:i]) for i in range(rows + 1)]
    pick = lambda *v: [rng.choice(v) for _ in range(rows)]  # noqa: E731
    words = np.random.RandomState(seed).randint(-2 ** 31, 2 ** 31, (masks, (n + 31) // 32)).astype(np.int32)
    return dict(history=[[token() for _ in range(width)] for _ in range(slots)], length=length,
                prompt=[rng.randint(0, n_) for n_ in length], slot=[rng.choice([-1, s]) if rng.random() < 0.2 else s
                                                                      for s in rng.sample(range(slots), rows)],
                repetition=pick(1.05, 1.0, 1.3, 0.8), presence=pick(0.0, 0.5, -0.25), frequency=pick(0.0, 0.1, 0.7),
                bias=(start, [token() for _ in range(start[-1])], [rng.uniform(-5, 5) for _ in range(start[-1])]),
                mask=words, mask_row=[rng.randint(-1, masks - 1) for _ in range(rows)])


def _logits(rows, n, seed):
    x = np.random.RandomState(seed).randn(rows, n).astype(np.float32) * 4
    x[0, 0] = 0.0
    return x


def _args(c, dev):
    import torch
    out = {}
    for k, v in c.items():
        if v is None:
            continue
        if k == "bias":
            out[k] = (_int(v[0], dev), _int(v[1], dev), torch.tensor(v[2], dtype=torch.float32).to(dev))
        elif k == "mask":
            out[k] = torch.from_numpy(v).to(dev)
        elif k in ("repetition", "presence", "frequency"):
            out[k] = torch.tensor(v, dtype=torch.float32).to(dev)
        else:
            out[k] = _int(v, dev)
    return out


def _check(dev, x, c, **kw):
    import torch
    from hy_mt_rs_b200 import quant, sampling
    got = sampling.adjust(torch.from_numpy(x).to(dev), **_args(c, dev), **kw)
    np.testing.assert_array_equal(got.cpu().numpy(), _expected(x, c))
    assert quant.device_status() == 0
    return got


# a slice is 4,096 logits: sizes around its ends, odd rows (unaligned), one token
@pytest.mark.parametrize("rows,n,width", [(1, 1, 3), (3, 31, 7), (5, 32, 1), (2, 33, 40), (4, 1000, 300), (3, 4095, 64), (3, 4096, 64),
                                          (2, 4097, 1000), (7, 8191, 129), (2, 12288, 2000), (1, 120832, 4000), (3, 120833, 513)])
def test_sizes(cuda, rows, n, width):
    _check(cuda, _logits(rows, n, n), _case(rows, n, width, n))


@pytest.mark.parametrize("leave", ["history", "prompt", "slot", "repetition", "presence", "frequency", "bias", "mask", "mask_row"])
def test_parts_left_out(cuda, leave):
    c = _case(4, 5000, 90, 3, masks=4)
    gone = ["history", "length", "prompt", "slot", "repetition", "presence", "frequency"] if leave == "history" else [leave]
    gone += ["mask_row"] if leave == "mask" else []
    _check(cuda, _logits(4, 5000, 3), {k: v for k, v in c.items() if k not in gone})


@pytest.mark.parametrize("only", ["repetition", "presence", "frequency", "bias", "mask"])
def test_one_part_alone(cuda, only):
    c = _case(4, 5000, 90, 4)
    keep = {"bias": ["bias"], "mask": ["mask", "mask_row"]}.get(only, ["history", "length", "prompt", "slot", only])
    _check(cuda, _logits(4, 5000, 4), {k: v for k, v in c.items() if k in keep})


def test_numbers_for_all_rows(cuda):
    import torch
    from hy_mt_rs_b200 import sampling
    c = _case(3, 700, 50, 5)
    c.update(repetition=[1.1] * 3, presence=[0.25] * 3, frequency=[0.5] * 3)
    x = _logits(3, 700, 5)
    a = _args(c, cuda)
    a.update(repetition=1.1, presence=0.25, frequency=0.5)
    got = sampling.adjust(torch.from_numpy(x).to(cuda), **a)
    np.testing.assert_array_equal(got.cpu().numpy(), _expected(x, c))


@pytest.mark.parametrize("n", [5000, 5001])
def test_strides_in_place_and_given_outputs(cuda, n):
    import torch
    from hy_mt_rs_b200 import sampling
    c, x = _case(3, n, 70, 6), _logits(3, n, 6)
    want, a = _expected(x, c), _args(c, cuda)
    wide = torch.full((3, n + 37), 7.0, device=cuda)
    wide[:, 1:n + 1] = torch.from_numpy(x).to(cuda)
    view = wide[:, 1:n + 1]
    a["history"] = torch.cat([a["history"], a["history"]], 1)[:, :70]     # rows 140 apart
    out = torch.full((3, n + 8), 8.0, device=cuda)
    got = sampling.adjust(view, **a, out=out[:, 4:n + 4])
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    assert (out[:, :4] == 8).all() and (out[:, n + 4:] == 8).all()
    sampling.adjust(view, **a, out=view)
    np.testing.assert_array_equal(view.cpu().numpy(), want)
    assert (wide[:, 0] == 7).all() and (wide[:, n + 1:] == 7).all()


def test_values_at_the_edges(cuda):
    """Infinities, NaN and the lowest value; a row whose mask leaves nothing;
    penalties that are off or not numbers above zero; tokens outside the
    vocabulary, repeated ones, 70,000 times the same."""
    import torch
    from hy_mt_rs_b200 import sampling
    n = 200
    x = _logits(8, n, 7)
    x[:, 3], x[:, 4], x[:, 5], x[:, 6], x[:, 7] = np.inf, -np.inf, np.nan, np.finfo(np.float32).min, -0.0
    past = [[3, 4, 5, 6, 7, -1, n, n + 5, 2 ** 31 - 1, -2 ** 31] + [9] * 70000 for _ in range(8)]
    c = dict(history=past, length=[len(past[0])] * 8, prompt=[0, 2, 4, 6, 10, 11, 70010, 100000], slot=list(range(8)),
             repetition=[1.5, 0.0, -1.0, math.nan, math.inf, 1.5, 1.5, 1.5], presence=[0.5] * 8, frequency=[0.001] * 8,
             bias=([0, 3, 3, 5, 5, 5, 5, 5, 5], [1, 1, 1, -4, n], [1.0, 2.0, math.inf, 3.0, 3.0]),
             mask=np.array([[0] * 7, [-1] * 7], dtype=np.int32), mask_row=[-1, -1, 0, 1, 1, -7, 1, 1])
    got = _check(cuda, x, c)
    assert (got[2] == -math.inf).all()
    token, prob = sampling.sample(got, torch.full((8,), 0.5, device=cuda))
    assert int(token[2]) == 0 and float(prob[2]) == 0


def test_bad_indexes_leave_their_part_out(cuda):
    """Slots and mask rows past the last, lengths and bias ranges outside their
    arrays: the row without that part, and the device status raised."""
    import torch
    from hy_mt_rs_b200 import quant, sampling
    c, x = _case(2, 300, 20, 8, slots=2), _logits(2, 300, 8)
    c.update(slot=[0, 1], length=[20, 20], mask_row=[0, 1], repetition=[2.0, 2.0])
    rows = lambda **kw: {**c, **kw}  # noqa: E731
    for given, as_if in ((rows(slot=[2, 1]), rows(slot=[-1, 1])), (rows(length=[21, 20]), rows(length=[0, 20])),
                         (rows(length=[-1, 20]), rows(length=[0, 20])), (rows(mask_row=[0, 2]), rows(mask_row=[0, -1])),
                         (rows(bias=([0, -1, 2], *c["bias"][1:])), rows(bias=([0, 0, 0], *c["bias"][1:]))),
                         (rows(bias=([0, 2, 2 ** 30], *c["bias"][1:])), rows(bias=([0, 2, 2], *c["bias"][1:])))):
        if len(given["bias"][1]) < 2:
            continue
        got = sampling.adjust(torch.from_numpy(x).to(cuda), **_args(given, cuda))
        np.testing.assert_array_equal(got.cpu().numpy(), _expected(x, as_if))
        assert quant.device_status() != 0


def test_captured_and_replayed_with_sampling(cuda):
    """adjust and sample captured in a graph, replayed as the history grows: greedy
    tokens as the rule gives them."""
    import torch
    from hy_mt_rs_b200 import sampling
    n, rows = 3000, 4
    x = _logits(rows, n, 9)
    dx = torch.from_numpy(x).to(cuda)
    history, length = torch.zeros(rows, 30, dtype=torch.int32, device=cuda), _int([0] * rows, cuda)
    u, token = torch.zeros(rows, device=cuda), torch.zeros(rows, dtype=torch.int32, device=cuda)
    rep, freq = torch.full((rows,), 1.2, device=cuda), torch.full((rows,), 0.3, device=cuda)
    zero = torch.zeros(rows, device=cuda)

    def step():
        y = sampling.adjust(dx, history, length, repetition=rep, frequency=freq)
        sampling.sample(y, u, temperature=zero, token=token)
        history.scatter_(1, length.long()[:, None], token[:, None])
        length.add_(1)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        step()
        length.zero_()
        with torch.cuda.graph(graph, stream=stream):
            step()
    torch.cuda.current_stream().wait_stream(stream)
    length.zero_()
    made = [[] for _ in range(rows)]
    for _ in range(25):
        graph.replay()
        want = _expected(x, dict(history=made, length=[len(m) for m in made], repetition=[1.2] * rows, frequency=[0.3] * rows))
        got = token.tolist()
        assert got == want.argmax(1).tolist()
        for m, t in zip(made, got):
            m.append(t)
