"""Sampling of next tokens on the device (hyq_sample).

The reference samples on the host (Sampler, generation.rs: temperature, top-k,
top-p); here one launch samples every row of a batch of logits from uniform
numbers the caller provides, so a decode loop needs no host round trip and a
draw can be repeated.
"""
import torch

from ._native import HyqError, load_ops

__all__ = ["adjust", "sample"]

_ops = load_ops()


def _per_row(logits, value, dtype):
    if value is None or isinstance(value, torch.Tensor):
        return value
    if not isinstance(logits, torch.Tensor):
        raise HyqError(-1, "logits: expected a CUDA tensor")
    return torch.full((logits.shape[0],), value, dtype=dtype, device=logits.device)


def adjust(logits, history=None, length=None, prompt=None, slot=None, repetition=None, presence=None, frequency=None,
           bias=None, mask=None, mask_row=None, out=None):
    """hyq_logits_adjust: penalties for repeated tokens, biases and a mask on
    `logits` [rows, n] (f32, rows any stride), in this order, before sample();
    into `out` when given (logits itself is allowed).

    history [slots, width] (int32) holds token ids: of the first length[slot] of
    row slot[r] (row r without slots; a negative slot: none) the first
    prompt[slot] are the prompt's (none without), the others were made.  Tokens
    of the history are divided by `repetition` where the logit is above zero and
    multiplied by it elsewhere; made ones then lose frequency * count + presence.
    The three are device tensors of one value per row, numbers for all rows, or
    None.  bias: (start [rows + 1], token, value): entries start[r] .. start[r +
    1] - 1 are row r's, the last of several for a token counts.  mask [masks,
    (n + 31) // 32] (int32): where bit token % 32 of word token // 32 of row
    mask_row[r] (row r without; negative: no mask) is 0, the logit becomes -inf."""
    if bias is None:
        bias = None, None, None
    elif not isinstance(bias, (tuple, list)) or len(bias) != 3:
        raise HyqError(-1, "bias: expected (start, token, value)")
    penalties = (_per_row(logits, p, torch.float32) for p in (repetition, presence, frequency))
    return _ops.adjust(logits, history, length, prompt, slot, *penalties, *bias, mask, mask_row, out)


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
        return _per_row(logits, value, dtype)

    return _ops.sample(logits, u, per_row(temperature, torch.float32), per_row(top_k, torch.int32),
                       per_row(top_p, torch.float32), per_row(min_p, torch.float32), token, prob)
