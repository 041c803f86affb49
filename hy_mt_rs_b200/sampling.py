"""Sampling of next tokens on the device (hyq_sample).

The reference samples on the host (Sampler, generation.rs: temperature, top-k,
top-p); here one launch samples every row of a batch of logits from uniform
numbers the caller provides, so a decode loop needs no host round trip and a
draw can be repeated.
"""
import torch

from ._native import HyqError, load_ops

__all__ = ["sample"]

_ops = load_ops()


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, token=None, prob=None):
    """One token of each row of `logits` [rows, n] (f32, rows any stride) from
    the uniform numbers u [rows] in [0, 1): (token int32 [rows], prob f32
    [rows], the token's share of what the filters keep).

    temperature, top_k, top_p and min_p are device tensors of one value per
    row, numbers for all rows, or None.  temperature <= 0 is greedy; top_k <= 0,
    top_p >= 1 and min_p <= 0 are off.  The filters apply in that order; ties
    go to the lower index (include/hyq.h, hyq_sample, states the rule).
    token and prob may be given to be written."""
    def per_row(value, dtype):
        if value is None or isinstance(value, torch.Tensor):
            return value
        if not isinstance(logits, torch.Tensor):
            raise HyqError(-1, "logits: expected a CUDA tensor")
        return torch.full((logits.shape[0],), value, dtype=dtype, device=logits.device)

    return _ops.sample(logits, u, per_row(temperature, torch.float32), per_row(top_k, torch.int32),
                       per_row(top_p, torch.float32), per_row(min_p, torch.float32), token, prob)
