"""A call's tensors are on one device.  Fake tensors stand in for those of a
second GPU: every call here is refused before it reads an address."""
import pytest

_ON = "cuda:0", "cuda:1"


@pytest.fixture
def fake():
    """fake(shape, type, device index): a CUDA tensor without memory."""
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode
    mode = FakeTensorMode()

    def make(shape, dtype=None, on=0):
        with mode:
            return torch.empty(shape, dtype=dtype or torch.float32, device=_ON[on])
    return make


def _refused(call, name):
    from hy_mt_rs_b200._native import HyqError
    with pytest.raises(HyqError, match=name + ": on another device"):
        call()


@pytest.mark.parametrize("name", ["u", "temperature", "top_k", "top_p", "min_p", "token", "prob"])
def test_sample(fake, name):
    import torch
    from hy_mt_rs_b200 import sampling
    ints = ("top_k", "token")
    x = fake((3, 100))
    kw = {n: fake((3,), torch.int32 if n in ints else torch.float32, int(n == name)) for n in ("u", "token", name)}
    _refused(lambda: sampling.sample(x, **kw), name)


def _cache_args(fake, **there):
    import torch
    i32 = torch.int32
    shapes = dict(q=((4, 8, 64), None), k_pages=((6, 2, 16, 64), None), v_pages=((6, 2, 16, 64), None), table=((2, 3), i32),
                  row_start=((3,), i32), pos=((2,), i32), slot=((2,), i32), k=((4, 2, 64), None), v=((4, 2, 64), None),
                  cos=((48, 32), None), sin=((48, 32), None), q_norm=((64,), None), k_norm=((64,), None),
                  out=((4, 8, 64), None), workspace=((1 << 26,), torch.uint8))
    return {n: fake(s, t, 1 if n in there else 0) for n, (s, t) in shapes.items()}


@pytest.mark.parametrize("name", ["k_pages", "v_pages", "table", "row_start", "pos", "slot", "out", "workspace"])
def test_attention(fake, name):
    from hy_mt_rs_b200 import paged
    a = _cache_args(fake, **{name: 1})
    _refused(lambda: paged.attention(a["q"], a["k_pages"], a["v_pages"], a["table"], a["row_start"], a["pos"], 3,
                                     slot=a["slot"], out=a["out"], workspace=a["workspace"]), name)


@pytest.mark.parametrize("name", ["k_pages", "v_pages", "table", "row_start", "pos", "slot", "out", "k", "v", "cos", "sin",
                                  "q_norm", "k_norm"])
def test_rope_append(fake, name):
    from hy_mt_rs_b200 import paged
    a = _cache_args(fake, **{name: 1})
    _refused(lambda: paged.rope_append(a["q"], a["k"], a["v"], a["k_pages"], a["v_pages"], a["table"], a["row_start"],
                                       a["pos"], a["cos"], a["sin"], a["q_norm"], a["k_norm"], slot=a["slot"],
                                       out=a["out"]), name)


@pytest.mark.parametrize("name", ["table", "length", "refs"])
def test_cache(fake, name):
    import torch
    from hy_mt_rs_b200.paged import PagedCache
    t = {n: fake(s, torch.int32, int(n == name)) for n, s in dict(table=(3, 2), length=(3,), refs=(6,)).items()}
    pool = fake((1, 2, 6, 2, 16, 64))
    _refused(lambda: PagedCache.over(pool, t["table"], t["length"], t["refs"]), name)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_page_calls(fake, which):
    import torch
    from hy_mt_rs_b200.paged import PagedCache
    cache = PagedCache.__new__(PagedCache)
    cache.pool = fake((1, 2, 6, 2, 16, 64))
    a = [fake((2,), torch.int32, int(i == which)) for i in range(3)]
    if which < 2:
        _refused(lambda: cache.fork(a[0], a[1]), "slots")
    if which == 0:
        _refused(lambda: cache.free(a[0]), "slots")
    _refused(lambda: cache.reserve(a[0], a[1], pos=a[2]), "slots")
