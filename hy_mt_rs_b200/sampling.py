"""Sampling of next tokens on the device (hyq_sample).

The reference samples on the host (Sampler, generation.rs: temperature, top-k,
top-p); here one launch samples every row of a batch of logits from uniform
numbers the caller provides, so a decode loop needs no host round trip and a
draw can be repeated.
"""
import torch

from ._native import HyqError, check, lib
from .quant import _need_cuda

__all__ = ["sample"]

_current_stream = torch._C._cuda_getCurrentRawStream


def _check(t, name, dtype, rows):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != dtype or not t.is_contiguous():
        _need_cuda(t, name, dtype)
    if t.numel() != rows:
        raise HyqError(-2, f"sample: {name} takes one value per row")
    return t.data_ptr()


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, token=None, prob=None):
    """One token of each row of `logits` [rows, n] (f32, rows any stride) from
    the uniform numbers u [rows] in [0, 1): (token int32 [rows], prob f32
    [rows], the token's share of what the filters keep).

    temperature, top_k, top_p and min_p are device tensors of one value per
    row, numbers for all rows, or None.  temperature <= 0 is greedy; top_k <= 0,
    top_p >= 1 and min_p <= 0 are off.  The filters apply in that order; ties
    go to the lower index (include/hyq.h, hyq_sample, states the rule).
    token and prob may be given to be written."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dtype != torch.float32:
        raise HyqError(-1, "sample: logits are a CUDA float32 tensor")
    shape, strides = logits.shape, logits.stride()
    if len(shape) != 2 or (shape[1] > 1 and strides[1] != 1):
        raise HyqError(-2, "sample: logits are [rows, n] with contiguous rows")
    rows, n = shape
    dev = logits.device
    kept = []   # tensors made here live until the launch

    def per_row(value, name, dtype):
        if value is None:
            return None
        if not isinstance(value, torch.Tensor):
            kept.append(torch.full((rows,), value, dtype=dtype, device=dev))
            return kept[-1].data_ptr()
        return _check(value, name, dtype, rows)

    if token is None:
        token = torch.empty(rows, dtype=torch.int32, device=dev)
    if prob is None:
        prob = torch.empty(rows, dtype=torch.float32, device=dev)
    check(lib.hyq_sample(logits.data_ptr(), n, strides[0] if rows > 1 else n, rows,
                         per_row(temperature, "temperature", torch.float32), per_row(top_k, "top_k", torch.int32),
                         per_row(top_p, "top_p", torch.float32), per_row(min_p, "min_p", torch.float32),
                         _check(u, "u", torch.float32, rows), _check(token, "token", torch.int32, rows),
                         _check(prob, "prob", torch.float32, rows), _current_stream(logits.get_device())))
    return token, prob
