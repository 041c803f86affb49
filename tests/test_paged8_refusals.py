"""Host checks of the 8-bit, shared-prefix, gather and adjust entry points: bad
arguments are refused with a negative code and a reason before any GPU work."""
import ctypes as C
import struct

import pytest

from test_paged_devices import _refused, fake  # noqa: F401
from test_paged_refusals import ALIGN, BATCH, INVALID, KV, PTR, SHAPE, _batch, _kv

_KV8 = struct.Struct("PPqqq")                                  # behind hyq_paged_kv
_ADJUST = struct.Struct("PqqqPPPPPPPPPqPqqP")                  # hyq_adjust


def _kv8(k_scale=PTR, v_scale=PTR, page=32, head=16, row=1, **kw):
    return _kv(**{"dtype": 2, **kw}) + _KV8.pack(k_scale or 0, v_scale or 0, page, head, row)


def _attention(kv, b, q=PTR, q_stride=512, heads=4, out=PTR, out_stride=512, ws=PTR):
    from hy_mt_rs_b200._native import lib
    return lib.hyq_paged_attention_kv8(kv, b, q, q_stride, heads, out, out_stride, ws, None)


def _append(kv, b, q=PTR, q_stride=512, heads=4, k=PTR, k_stride=256, cos=PTR, positions=64, out=PTR):
    from hy_mt_rs_b200._native import lib
    return lib.hyq_paged_rope_append_kv8(kv, b, q, q_stride, heads, k, k_stride, PTR, 256, cos, PTR, positions, None, None, 1e-5, 0,
                                         out, 512, None)


def _shared(kv, b, start=PTR, shared=PTR, groups=1, max_shared=50, heads=4, out=PTR, ws=PTR):
    from hy_mt_rs_b200._native import lib
    return lib.hyq_paged_attention_shared(kv, b, start, shared, groups, max_shared, PTR, 512, heads, out, 512, ws, None)


def _gather(kv, b, f16=1, k=PTR, k_stride=256, v=PTR, v_stride=256):
    from hy_mt_rs_b200._native import lib
    return lib.hyq_paged_gather(kv, b, f16, k, k_stride, v, v_stride, None)


@pytest.mark.parametrize("call", [_attention, _append, _shared, _gather])
def test_cache_and_batch_checks(call):
    from hy_mt_rs_b200._native import last_error
    assert call(None, _batch()) == INVALID
    assert call(_kv8(), None) == INVALID
    for kw, code in KV:
        if kw == dict(dtype=2) or (call is _gather and kw == dict(kv_heads=3)):    # fine with these calls
            continue
        assert call(_kv8(**{"dtype": 1, **kw}), _batch()) == code, kw
        assert "paged_" in last_error()
    for dtype in (2, 3):
        for kw, code in ((dict(k_scale=None), INVALID), (dict(v_scale=None), INVALID), (dict(page=0), SHAPE), (dict(head=-1), SHAPE),
                         (dict(row=0), SHAPE), (dict(k_scale=PTR + 2), ALIGN), (dict(v_scale=PTR + 1), ALIGN), (dict(head_dim=257), SHAPE),
                         (dict(slots=1), SHAPE)):
            assert call(_kv8(dtype=dtype, **kw), _batch()) == code, kw
    for dtype in (4, -1):
        assert call(_kv8(dtype=dtype), _batch()) == INVALID
    for kw, code in BATCH:
        assert call(_kv8(), _batch(**kw)) == code, kw


def test_scales_are_not_for_the_plain_calls():
    from hy_mt_rs_b200._native import lib
    for dtype in (2, 3):
        assert lib.hyq_paged_attention(_kv8(dtype=dtype), _batch(), PTR, 512, 4, PTR, 512, PTR, None) == INVALID


def test_shared_checks():
    from hy_mt_rs_b200._native import lib
    import torch
    n = C.c_size_t()
    f = lib.hyq_paged_attention_shared_workspace_bytes
    assert f(16, 128, 64, C.byref(n)) == 0
    small = n.value
    assert f(16, 128, 6400, C.byref(n)) == 0 and n.value >= small + 6336 * 16 * 128 * 4
    assert f(16, 128, 64, None) == INVALID
    for bad in ((0, 128, 64), (16, 0, 64), (16, 257, 64), (16, 128, -1), (16, 128, 1 << 31), (1 << 17, 128, 1)):
        assert f(*bad, C.byref(n)) == SHAPE, bad
    if not torch.cuda.is_available():
        return      # the status word comes first and needs a device
    for kw, code in ((dict(groups=-1), SHAPE), (dict(groups=4097), SHAPE), (dict(max_shared=-1), SHAPE), (dict(max_shared=101), SHAPE),
                     (dict(start=None), INVALID), (dict(shared=None), INVALID), (dict(start=PTR + 2), ALIGN),
                     (dict(shared=PTR + 1), ALIGN), (dict(ws=None), INVALID), (dict(ws=PTR + 4), ALIGN), (dict(out=PTR + 2), ALIGN)):
        assert _shared(_kv8(), _batch(), **kw) == code, kw
    assert _shared(_kv8(), _batch(max_new=9)) == SHAPE      # 18 rows of a sequence
    assert _gather(_kv8(), _batch(), k_stride=255) == SHAPE
    assert _gather(_kv8(), _batch(), k=None) == INVALID
    assert _gather(_kv8(), _batch(), v=PTR + 1) == ALIGN


def _adjust(n=100, stride=100, rows=2, logits=PTR, out=PTR, out_stride=100, given=True, **kw):
    from hy_mt_rs_b200._native import lib
    d = dict(history=PTR, slots=2, width=8, history_stride=8, slot=None, length=PTR, prompt=None, repetition=PTR, presence=None,
             frequency=None, bias_start=PTR, bias_token=PTR, bias_value=PTR, bias_count=5, mask=PTR, masks=2, mask_stride=4,
             mask_row=None)
    d.update(kw)
    return lib.hyq_logits_adjust(logits, n, stride, rows, _ADJUST.pack(*(v or 0 for v in d.values())) if given else None, out,
                                 out_stride, None)


def test_adjust_checks():
    from hy_mt_rs_b200._native import last_error
    assert _adjust(given=False) == INVALID and "logits_adjust" in last_error()
    for kw, code in ((dict(n=0), SHAPE), (dict(n=1 << 31, stride=1 << 31, out_stride=1 << 31), SHAPE), (dict(stride=99), SHAPE),
                     (dict(out_stride=99), SHAPE), (dict(rows=-1), SHAPE), (dict(rows=1 << 31), SHAPE), (dict(logits=None), INVALID),
                     (dict(out=None), INVALID), (dict(length=None), INVALID), (dict(history=None), INVALID),
                     (dict(bias_token=None), INVALID), (dict(bias_value=None), INVALID), (dict(slots=0), SHAPE), (dict(slots=1), SHAPE),
                     (dict(width=-1), SHAPE), (dict(history_stride=7), SHAPE), (dict(bias_count=-1), SHAPE), (dict(masks=0), SHAPE),
                     (dict(masks=1), SHAPE), (dict(mask_stride=3), SHAPE), (dict(stride=101), SHAPE), (dict(logits=PTR + 2), ALIGN),
                     (dict(prompt=PTR + 1), ALIGN), (dict(mask_row=PTR + 3), ALIGN), (dict(bias_value=PTR + 2), ALIGN)):
        assert _adjust(**kw) == code, kw
    assert _adjust(rows=0) == 0


def test_python_entry_points_refuse():
    import torch
    from hy_mt_rs_b200 import paged, sampling
    from hy_mt_rs_b200._native import HyqError
    cpu, ints = torch.zeros(2, 4, 128), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(HyqError):
        paged.attention_shared(cpu, cpu, cpu, ints, ints, ints, ints, ints, 1, workspace=ints)
    with pytest.raises(HyqError):
        paged.attention_shared(None, cpu, cpu, ints, ints, ints, ints, ints, 1)
    with pytest.raises(HyqError):
        paged.gather(cpu, cpu, ints, ints, ints, 2)
    with pytest.raises(HyqError):
        paged.gather(cpu, cpu, ints, ints, ints, 2, dtype=torch.bfloat16)
    with pytest.raises(HyqError):
        sampling.adjust(cpu[0])
    with pytest.raises(HyqError):
        sampling.adjust(None, repetition=1.1)
    with pytest.raises(HyqError):
        sampling.adjust(cpu[0], bias=3)
    with pytest.raises(TypeError):
        paged._ops.gather(cpu)


def _cache(fake, dtype, **there):  # noqa: F811
    import torch
    i32, f32 = torch.int32, torch.float32
    shapes = dict(q=((4, 8, 64), f32), k_pages=((6, 2, 16, 64), dtype), v_pages=((6, 2, 16, 64), dtype), table=((2, 3), i32),
                  row_start=((3,), i32), pos=((2,), i32), slot=((2,), i32), group_start=((2,), i32), shared=((1,), i32),
                  k_scale=((6, 2, 16), f32), v_scale=((6, 2, 16), f32), out=((4, 8, 64), f32), workspace=((1 << 26,), torch.uint8),
                  k_out=((4, 2, 64), f32), v_out=((4, 2, 64), f32))
    return {n: fake(s, t, 1 if n in there else 0) for n, (s, t) in shapes.items()}


@pytest.mark.parametrize("name", ["k_scale", "v_scale", "group_start", "shared", "out", "workspace", "table", "slot"])
def test_shared_is_on_one_device(fake, name):  # noqa: F811
    import torch
    from hy_mt_rs_b200 import paged
    a = _cache(fake, torch.int8, **{name: 1})
    _refused(lambda: paged.attention_shared(a["q"], a["k_pages"], a["v_pages"], a["table"], a["row_start"], a["pos"], a["group_start"],
                                            a["shared"], 1, slot=a["slot"], out=a["out"], workspace=a["workspace"],
                                            k_scale=a["k_scale"], v_scale=a["v_scale"]), name)


@pytest.mark.parametrize("name", ["k_out", "v_out", "k_scale", "row_start", "pos"])
def test_gather_is_on_one_device(fake, name):  # noqa: F811
    import torch
    from hy_mt_rs_b200 import paged
    a = _cache(fake, torch.float8_e4m3fn, **{name: 1})
    _refused(lambda: paged.gather(a["k_pages"], a["v_pages"], a["table"], a["row_start"], a["pos"], 4, k_out=a["k_out"],
                                  v_out=a["v_out"], k_scale=a["k_scale"], v_scale=a["v_scale"]), name)


@pytest.mark.parametrize("name", ["history", "length", "prompt", "slot", "repetition", "presence", "frequency", "mask", "mask_row", "out"])
def test_adjust_is_on_one_device(fake, name):  # noqa: F811
    import torch
    from hy_mt_rs_b200 import sampling
    i32, f32 = torch.int32, torch.float32
    shapes = dict(history=((3, 9), i32), length=((3,), i32), prompt=((3,), i32), slot=((2,), i32), repetition=((2,), f32),
                  presence=((2,), f32), frequency=((2,), f32), mask=((2, 4), i32), mask_row=((2,), i32), out=((2, 100), f32))
    a = {n: fake(s, t, int(n == name)) for n, (s, t) in shapes.items()}
    _refused(lambda: sampling.adjust(fake((2, 100)), **a), name)


def test_scales_that_do_not_fit(fake):  # noqa: F811
    """Missing, of another shape, of different strides, or for pages that have none."""
    import torch
    from hy_mt_rs_b200 import paged
    from hy_mt_rs_b200._native import HyqError
    a = _cache(fake, torch.int8)

    def call(**kw):
        b = {**a, **kw}
        paged.attention(b["q"], b["k_pages"], b["v_pages"], b["table"], b["row_start"], b["pos"], 1, workspace=b["workspace"],
                        k_scale=b["k_scale"], v_scale=b["v_scale"])

    f16 = fake((6, 2, 16, 64), torch.float16)
    for kw in (dict(k_scale=None), dict(v_scale=None), dict(k_scale=fake((6, 2, 15))), dict(k_scale=fake((6, 2))),
               dict(k_scale=fake((6, 16, 2)).transpose(1, 2)), dict(k_scale=fake((6, 2, 16), torch.float16)),
               dict(k_pages=f16, v_pages=f16), dict(v_pages=fake((6, 2, 16, 64), torch.float8_e4m3fn)),
               dict(k_pages=fake((6, 2, 16, 64), torch.uint8), v_pages=fake((6, 2, 16, 64), torch.uint8))):
        with pytest.raises(HyqError):
            call(**kw)
