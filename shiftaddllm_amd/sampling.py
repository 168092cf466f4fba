"""Choosing next tokens from logits with temperature, top-k, top-p and min-p, from given random numbers.

The reference's benchmark feeds given tokens (model/opt.py:367-423) and the decode harness took the most likely one; this is
what a server needs next to that.  The rules, to the treatment of ties, infinities and empty rows, are those of lutgemm_sample_tokens in
include/lutgemm_gfx950.h: largest logits first, equal ones by index, each filter keeps a first part of that order.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import native


def sample(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
    """(ids int64 [rows], logprob float32 [rows]) of logits [rows, vocab] (fp16, bf16 or fp32; rows any distance apart).

    uniform: float32 [rows], one number in [0, 1) per row.  temperature, top_p, min_p (float32) and top_k (int32): a tensor of one value
    per row, a number for all rows, or None (temperature 1, filter off).  temperature <= 0 takes the first of the largest logits.
    logprob is the logarithm of the drawn token's share of what the filters left.  A row of -inf or NaN only: id -1, logprob -inf."""
    rows = logits.shape[0] if logits.dim() == 2 else 0

    def per_row(value, dtype):
        if value is None or isinstance(value, torch.Tensor):
            return value
        return torch.full((rows,), value, dtype=dtype, device=logits.device)
    f32 = torch.float32
    return native.lutgemm.sample_tokens(logits, uniform, per_row(temperature, f32), per_row(top_k, torch.int32), per_row(top_p, f32),
                                        per_row(min_p, f32))


@dataclass
class SamplingOptions:
    """How a decoder chooses its tokens: the filters, and the seed of the random numbers."""
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int = 0
