"""sampling.adjust on batches: from 148 slices of 8,192 logits on a CTA takes such a
slice instead of 2,048.  Bit for bit the rule written out token by token."""
import numpy as np
import pytest

from test_gpu_adjust import _args, _case, _check, _expected, _logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,n,width", [(150, 8191, 40), (150, 8192, 300), (80, 8193, 64), (75, 16384, 3000), (50, 20001, 100),
                                          (10, 120832, 4000), (20, 120833, 513), (148, 1, 3), (200, 33, 70), (300, 2049, 5)])
def test_sizes(cuda, rows, n, width):
    """Around a slice's end, odd rows (unaligned), rows shorter than one."""
    assert rows * -(-n // 8192) >= 148
    _check(cuda, _logits(rows, n, n), _case(rows, n, width, n, masks=5))


@pytest.mark.parametrize("rows,n", [(147, 8192), (49, 24576), (9, 120832), (2, 2047), (2, 2048), (2, 2049), (3, 6145)])
def test_sizes_below(cuda, rows, n):
    assert rows * -(-n // 8192) < 148
    _check(cuda, _logits(rows, n, n), _case(rows, n, 200, n))


@pytest.mark.parametrize("rows,n", [(150, 8192), (150, 8000), (40, 32769)])
def test_long_histories(cuda, rows, n):
    """More than 4,096 tokens of a history in one slice (noted down no further), next to
    rows with fewer, and the same token again and again."""
    c, rng = _case(rows, n, 5000, 1), np.random.RandomState(5)
    history = rng.randint(0, min(n, 8192), (rows + 2, 9000)).astype(np.int32)
    history[1] = 7
    history[2, :4096] = rng.randint(0, n, 4096)
    length = [9000, 9000, 4096, 4097, 0] + rng.randint(0, 9001, rows - 3).tolist()
    c.update(history=history.tolist(), length=length, prompt=[v // 3 for v in length])
    _check(cuda, _logits(rows, n, 3), c)


@pytest.mark.parametrize("n", [8300, 8301])
def test_strides_in_place_and_replayed(cuda, n):
    """Rows with a stride, into themselves; captured, and replayed over other logits beside
    another stream's call."""
    import torch
    from hy_mt_rs_b200 import sampling
    rows = 80
    c, x = _case(rows, n, 400, 6, masks=3), _logits(rows, n, 6)
    a = _args(c, cuda)
    wide = torch.full((rows, n + 37), 7.0, device=cuda)
    view = wide[:, 1:n + 1]
    view.copy_(torch.from_numpy(x))
    sampling.adjust(view, **a, out=view)
    np.testing.assert_array_equal(view.cpu().numpy(), _expected(x, c))
    assert (wide[:, 0] == 7).all() and (wide[:, n + 1:] == 7).all()
    src, out = torch.from_numpy(x).to(cuda), torch.zeros(rows, n, device=cuda)
    graph, stream, other = torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        sampling.adjust(src, **a, out=out)
    for seed in (7, 8):
        y = _logits(rows, n, seed)
        src.copy_(torch.from_numpy(y))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(other):
            beside = sampling.adjust(src, **a)
        torch.cuda.synchronize()
        np.testing.assert_array_equal(out.cpu().numpy(), _expected(y, c))
        assert torch.equal(beside, out)


def test_histories_of_width_zero(cuda):
    """Rows that can hold no token: penalties change nothing, biases and masks do."""
    import torch
    from hy_mt_rs_b200 import quant, sampling
    from hy_mt_rs_b200._native import HyqError
    c, x = _case(4, 700, 5, 2), _logits(4, 700, 2)
    a = _args(c, cuda)
    a.update(history=torch.empty(6, 0, dtype=torch.int32, device=cuda), length=torch.zeros(6, dtype=torch.int32, device=cuda))
    a.pop("prompt")
    got = sampling.adjust(torch.from_numpy(x).to(cuda), **a)
    np.testing.assert_array_equal(got.cpu().numpy(), _expected(x, {k: c[k] for k in ("bias", "mask", "mask_row")}))
    got = sampling.adjust(torch.from_numpy(x).to(cuda), a["history"], a["length"], repetition=1.5, frequency=0.5)
    np.testing.assert_array_equal(got.cpu().numpy(), x)
    with pytest.raises(HyqError):
        sampling.adjust(torch.from_numpy(x).to(cuda), a["history"], a["length"][:5], repetition=1.5)
    assert quant.device_status() == 0
