"""Low-rank adapters of many requests beside one shared quantised projection.

A binary-coded weight cannot take up an adapter's product, and requests that are decoded together may each want another one.
`AdapterBank` holds the adapters of one projection, `LutLinear.adapters` hangs it beside a layer, and every row names its
adapter.  The reference has no counterpart.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .. import native


class AdapterBank(nn.Module):
    """`count` adapters of a projection of infeatures -> outfeatures: out = base + scale * up (down x).

    Buffers
      down   fp16 [count, rank, infeatures]
      up     fp16 [count, outfeatures, rank]
      scale  fp32 [count]
    `rank` is filled up to a multiple of 8 with zeros; adapters of lower rank likewise (`set`)."""

    def __init__(self, infeatures: int, outfeatures: int, rank: int, count: int):
        super().__init__()
        if infeatures < 32 or infeatures % 32 or outfeatures < 4 or outfeatures % 4:
            raise ValueError("infeatures must be a multiple of 32, outfeatures a multiple of 4")
        if not 1 <= rank <= 256 or not 1 <= count <= native.MAX_ADAPTERS:
            raise ValueError(f"rank must be 1 to 256, count 1 to {native.MAX_ADAPTERS}")
        self.K, self.N, self.count, self.rank = infeatures, outfeatures, count, -(-rank // 8) * 8
        self.register_buffer("down", torch.zeros((count, self.rank, infeatures), dtype=torch.float16))
        self.register_buffer("up", torch.zeros((count, outfeatures, self.rank), dtype=torch.float16))
        self.register_buffer("scale", torch.ones(count, dtype=torch.float32))

    @classmethod
    def from_tensors(cls, down, up, scale=None):
        """A bank of down [count, rank, infeatures], up [count, outfeatures, rank] and scale [count], on their device."""
        count, rank, K = down.shape
        if up.dim() != 3 or up.shape[0] != count or up.shape[2] != rank:
            raise ValueError(f"down is {tuple(down.shape)}, up {tuple(up.shape)}: not the same adapters")
        with torch.device("meta"):
            bank = cls(K, up.shape[1], rank, count)
        pad = bank.rank - rank
        bank.down = nn.functional.pad(down.detach().half(), (0, 0, 0, pad)).contiguous()
        bank.up = nn.functional.pad(up.detach().half(), (0, pad)).contiguous()
        bank.scale = torch.ones(count, dtype=torch.float32, device=down.device) if scale is None else scale.detach().float().contiguous()
        return bank

    @torch.no_grad()
    def set(self, index: int, down, up, scale: float = 1.0):
        """Fills adapter `index` from down [r, infeatures] and up [outfeatures, r], r at most the bank's rank."""
        r = down.shape[0]
        if not 0 <= index < self.count:
            raise IndexError(f"adapter {index} of {self.count}")
        if r > self.rank or tuple(down.shape) != (r, self.K) or tuple(up.shape) != (self.N, r):
            raise ValueError(f"expected down [r, {self.K}] and up [{self.N}, r], r <= {self.rank}; got {tuple(down.shape)}, {tuple(up.shape)}")
        self.down[index].zero_()
        self.up[index].zero_()
        self.down[index, :r] = down
        self.up[index, :, :r] = up
        self.scale[index] = scale

    def forward(self, x, ids, base, out=None):
        """base + scale[id] * up[id] (down[id] x), row by row: x [..., infeatures], base [..., outfeatures] fp16, ids int32, one per row;
        rows whose id is not in 0 .. count - 1 are base's.  `out` may be base itself."""
        b = self._buffers
        return native.lutgemm.adapters_apply(x, ids, base, out, b["down"], b["up"], b["scale"])

    def extra_repr(self):
        return f"in_features={self.K}, out_features={self.N}, rank={self.rank}, count={self.count}"
