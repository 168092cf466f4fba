"""A cache of keys and values held in 4 bits, and the attention that appends to it and reads it.

The fp16 cache of the decode harness takes 512 bytes a position of a kv head of 128 numbers, this one 160: groups of 32
numbers along the head share a scale and a minimum (lutgemm_q4_attention_f16 of include/lutgemm_gfx950.h states layout and
rounding).  One call serves single tokens, several at once and prompts, every sequence at its own position.  The reference has
no counterpart: it decodes through the framework's fp16 cache (model/opt.py:367-423).
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import native

GROUP = 32
BLOCK = 32


class Q4Cache(nn.Module):
    """Keys and values of `batch` sequences, `kv_heads` heads of `head_dim` numbers (a multiple of 32, at most 256), up to
    `max_positions` positions.  `data` is the memory: uint8 [batch, kv_heads, blocks of 32 positions, 40 * head_dim], given or allocated;
    a buffer, so that a module's caches move with it, but none of its state."""

    def __init__(self, batch: int, kv_heads: int, max_positions: int, head_dim: int, device="cuda:0", data: torch.Tensor | None = None):
        super().__init__()
        size = native.cabi().lutgemm_q4_cache_bytes(batch, kv_heads, max_positions, head_dim)
        if size == 0:
            raise ValueError(f"no 4-bit cache for batch={batch}, kv_heads={kv_heads}, max_positions={max_positions}, head_dim={head_dim} "
                             "(head_dim must be a multiple of 32 up to 256, max_positions 1 to 2^20)")
        self.batch, self.kv_heads, self.max_positions, self.head_dim = batch, kv_heads, max_positions, head_dim
        shape = (batch, kv_heads, -(-max_positions // BLOCK), 40 * head_dim)
        if data is None:
            data = torch.zeros(shape, dtype=torch.uint8, device=device)
        if tuple(data.shape) != shape or data.dtype is not torch.uint8 or not data.is_contiguous():
            raise ValueError(f"data must be contiguous uint8 {shape}, is {data.dtype} {tuple(data.shape)}")
        self.register_buffer("data", data, persistent=False)

    def attend(self, q, k, v, cos, sin, start, counts=None, out=None, held=False):
        """Appends the new tokens' keys (rotated) and values and returns attention over each sequence's positions up to each token.

        q [batch, tokens, heads * head_dim] or, for one token each, [batch, heads * head_dim], k and v alike with kv_heads; fp16, any strides.
        cos, sin: fp16 tables [max_positions, head_dim], rotate-half convention.  start int64 [batch]: position of each sequence's first
        new token, negative for an idle slot; counts int32 [batch]: how many of its tokens are there (None: all).  Tokens beyond the count or
        outside the cache are passed over, their rows are zeros.  With `held` also returns the values the cache holds for the
        new tokens' keys and values."""
        return native.lutgemm.q4_attend(self._buffers["data"], q, k, v, cos, sin, start, counts, out, held, self.max_positions)

    def values(self, sequence: int, positions: int):
        """What the cache holds of the first `positions` positions of a sequence: keys and values, fp16 [positions, kv_heads, head_dim].
        (For looking at a cache; attention reads it as it is.)"""
        if not 0 <= positions <= self.max_positions:
            raise ValueError(f"{positions} positions of a cache of {self.max_positions}")
        G, n = self.head_dim // GROUP, -(-positions // BLOCK)
        block = self.data[sequence, :, :n].contiguous()
        words, half = block.view(torch.int32), block.view(torch.float16)
        shift = torch.tensor([4 * (e // 2) + 16 * (e % 2) for e in range(8)], device=block.device, dtype=torch.int32)

        def codes(first):
            return (words[..., first:first + 128 * G].unsqueeze(-1) >> shift) & 15
        k = codes(0).view(self.kv_heads, n, 32, 4, G, 8).transpose(-3, -2).reshape(self.kv_heads, n * 32, G, 32)
        ks = half[..., 256 * G:320 * G].reshape(self.kv_heads, n * 32, G, 2)
        v = codes(160 * G).view(self.kv_heads, n, 4, 16, 2 * G, 2, 4).permute(0, 1, 5, 2, 6, 4, 3).reshape(self.kv_heads, n * 32, G, 32)
        vs = half[..., 576 * G:640 * G].view(self.kv_heads, n, G, 2, 4, 2, 4).permute(0, 1, 5, 4, 6, 2, 3).reshape(self.kv_heads, n * 32, G, 2)
        return tuple((s[..., 1:].float() + s[..., :1].float() * c.float()).half().flatten(2)[:, :positions].transpose(0, 1).contiguous()
                     for c, s in ((k, ks), (v, vs)))
