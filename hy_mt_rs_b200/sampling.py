"""Sampling of next tokens on the device (hyq_sample).

The reference samples on the host (Sampler, generation.rs: temperature, top-k,
top-p); here one launch samples every row of a batch of logits from uniform
numbers the caller provides, so a decode loop needs no host round trip and a
draw can be repeated.
"""
import ctypes as C

import torch

from ._native import HyqError, check, lib
from .quant import _need_cuda, _ptr, _stream

__all__ = ["sample"]


def _per_row(value, rows, dtype, name, device):
    """A parameter as a device array of one value per row (None: off)."""
    if value is None:
        return None
    if not isinstance(value, torch.Tensor):
        return torch.full((rows,), value, dtype=dtype, device=device)
    _need_cuda(value, name, dtype)
    if value.numel() != rows:
        raise HyqError(-2, f"sample: {name} takes one value per row")
    return value


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
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise HyqError(-2, "sample: logits are [rows, n] with contiguous rows")
    rows, n = logits.shape
    dev = logits.device
    _need_cuda(u, "u", torch.float32)
    if u.numel() != rows:
        raise HyqError(-2, "sample: u takes one number per row")
    token = torch.empty(rows, dtype=torch.int32, device=dev) if token is None else token
    prob = torch.empty(rows, dtype=torch.float32, device=dev) if prob is None else prob
    _need_cuda(token, "token", torch.int32)
    _need_cuda(prob, "prob", torch.float32)
    if token.numel() != rows or prob.numel() != rows:
        raise HyqError(-2, "sample: invalid output buffer")
    params = [_per_row(temperature, rows, torch.float32, "temperature", dev),
              _per_row(top_k, rows, torch.int32, "top_k", dev), _per_row(top_p, rows, torch.float32, "top_p", dev),
              _per_row(min_p, rows, torch.float32, "min_p", dev)]
    opt = lambda t: C.c_void_p(None) if t is None else _ptr(t)  # noqa: E731
    check(lib.hyq_sample(_ptr(logits), n, max(logits.stride(0), n), rows, *(opt(t) for t in params), _ptr(u),
                         _ptr(token), _ptr(prob), _stream(dev)))
    return token, prob
