"""What a hyper-connection layer may do between its read and its write, besides
calling the wrapped module.

The reference's layers leave all of this to the module they wrap. Given a
``BlockOptions``, the layers of this package (``cghc``, ``ghc``, ``mhc``) do it
in the read and the write themselves, where it costs no pass of its own over
the block's tensors:

    y  = pre_norm(R x)                                  ops.hc_read_norm
    f  = module(y)
    z  = dropout(scale * sigmoid(gate(y)) * post_norm(f))
    x' = H x [+ projection] + W z                       ops.hc_mix_write_norm

and the wrapped module is then the block without its norm, dropout and
residual scale. Without options (the default) a layer is the reference's, in
its parameters, ``state_dict`` keys and results.
"""

from __future__ import annotations

from contextlib import nullcontext
from dataclasses import dataclass
from typing import Literal, Optional

import torch
import torch.nn as nn

from .drop_state import DropState
from .ops import hc_mix_write, hc_mix_write_norm, hc_read, hc_read_norm

NormKind = Literal["rms", "layer"]


@dataclass(frozen=True)
class BlockOptions:
    """pre_norm / post_norm: "rms" or "layer" over a token's embed_dim values
    (affine; LayerNorm with a bias), or None. gate: an elementwise sigmoid gate
    on the block's output, from a Linear(embed_dim, embed_dim) of its input.
    residual_scale: the initial value of a learnt scale a channel, or None.
    dropout: the probability that an element of z is dropped in training."""

    pre_norm: Optional[NormKind] = None
    post_norm: Optional[NormKind] = None
    gate: bool = False
    residual_scale: Optional[float] = None
    dropout: float = 0.0
    eps: float = 1e-6

    def __post_init__(self):
        for kind in (self.pre_norm, self.post_norm):
            if kind not in (None, "rms", "layer"):
                raise ValueError(f"a norm must be 'rms', 'layer' or None, got {kind!r}")
        if not 0.0 <= self.dropout <= 1.0:
            raise ValueError(f"dropout must lie in [0, 1], got {self.dropout}")


class _Norm(nn.Module):
    def __init__(self, dim: int, kind: NormKind):
        super().__init__()
        self.kind = kind
        self.weight = nn.Parameter(torch.ones(dim))
        self.bias = nn.Parameter(torch.zeros(dim)) if kind == "layer" else None


class BlockParts(nn.Module):
    """The parameters of a layer's ``BlockOptions`` and its read and write.

    Dropout's bits come from ``drop_state``, an int64 tensor (seed, offset) on
    the layer's device (seeded from torch's generator, not part of the
    ``state_dict``): every training step's write draws with the next offset, also
    when a graph that holds it is replayed, and a write that a checkpoint runs
    again with the offset of its first run (``drop_state.py``)."""

    def __init__(self, options: BlockOptions, embed_dim: int):
        super().__init__()
        self.options, self.embed_dim = options, embed_dim
        self.pre_norm = _Norm(embed_dim, options.pre_norm) if options.pre_norm else None
        self.post_norm = _Norm(embed_dim, options.post_norm) if options.post_norm else None
        self.gate = nn.Linear(embed_dim, embed_dim) if options.gate else None
        self.scale = None if options.residual_scale is None else nn.Parameter(
            torch.full((embed_dim,), float(options.residual_scale)))
        self.bits = DropState(seeded=options.dropout > 0)

    @property
    def drop_state(self) -> torch.Tensor:
        return self.bits.state

    @drop_state.setter
    def drop_state(self, state: torch.Tensor) -> None:
        self.bits.state = state

    def read(self, R: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
        """The block's input [T, m, D] from the streams x [T, n, D]."""
        if self.pre_norm is None:
            return hc_read(R, x)
        p = self.pre_norm
        return hc_read_norm(R, x, p.weight, p.bias, norm=p.kind, eps=self.options.eps)

    def write(self, H, x, W, f, v, u) -> torch.Tensor:
        """The new streams from the block's output f [T, m, D] and input u."""
        o, p = self.options, self.post_norm
        drop = o.dropout if self.training else 0.0
        if p is None and self.gate is None and self.scale is None and drop == 0.0:
            return hc_mix_write(H, x, W, f, v)
        gate = None if self.gate is None else self.gate(u.reshape(-1, self.embed_dim)).view(f.shape)
        with self.bits.drawn(x.device) if drop else nullcontext() as seed:
            return hc_mix_write_norm(H, x, W, f, v, norm="none" if p is None else p.kind,
                                     weight=None if p is None else p.weight, bias=None if p is None else p.bias, eps=o.eps,
                                     gate=gate, gate_activation="sigmoid", scale=self.scale, dropout_p=drop, seed=seed)


def read_block(parts: Optional[BlockParts], R, x):
    return hc_read(R, x) if parts is None else parts.read(R, x)


def write_block(parts: Optional[BlockParts], H, x, W, f, v, u):
    return hc_mix_write(H, x, W, f, v) if parts is None else parts.write(H, x, W, f, v, u)
