"""Dropout whose bits come from a counter, so that no mask is stored.

    y = hc_dropout(x, p, seed, offset)     y_i = x_i / (1 - p) where kept, else 0

Element i (its row-major index in x) is kept when word i mod 4 of Philox
4x32-10 (Salmon, Moraes, Dror and Shaw, SC 2011) with counter (i div 4,
offset) and key seed is at least floor(p 2^32). The bits depend on p, seed,
offset and the element's place alone: the backward draws the same ones again,
and two calls with the same seed and offset on tensors of one size drop the
same places. Give every call of a step its own offset (or seed).

seed and offset are whole numbers (taken modulo 2^64), or seed is an int64
CUDA tensor of two elements (seed, offset), which the kernel reads when it
runs: a step captured into a CUDA graph draws new bits at each replay when the
step also moves that tensor on. ``drop_state.DropState`` does that for a module,
with checkpoints and several ranks in mind.
"""

from __future__ import annotations

import torch

from .. import _lib


def drop_state(name: str, seed, offset, x: torch.Tensor):
    """(state tensor or None, seed, offset) of a caller's seed and offset."""
    if seed is None:
        raise ValueError(f"{name} needs a seed for its dropout")
    if not torch.is_tensor(seed):
        return None, int(seed), int(offset)
    if offset:
        raise ValueError(f"{name}: a seed tensor holds the offset too (its second element)")
    if seed.dtype != torch.int64 or seed.shape != (2,):
        raise ValueError(f"{name}: a seed tensor must be int64 of shape (2,), got {seed.dtype} {tuple(seed.shape)}")
    if seed.device != x.device:
        raise RuntimeError(f"{name} requires tensors on one device (x is on {x.device}, seed on {seed.device})")
    return seed.contiguous(), 0, 0


def drop_words(seed: int, offset: int):
    """Both modulo 2^64, as the signed words of the C call."""
    return tuple((k + (1 << 63)) % (1 << 64) - (1 << 63) for k in (seed, offset))


def hc_dropout(x: torch.Tensor, p: float, seed, offset: int = 0) -> torch.Tensor:
    """x with each element kept (times 1 / (1 - p)) or zeroed (see module doc)."""
    if not x.is_cuda or (torch.is_tensor(seed) and not seed.is_cuda):
        raise RuntimeError("hc_dropout requires CUDA tensors")
    state, seed, offset = drop_state("hc_dropout", seed, offset, x)
    out = _lib.torch_ext().dropout(x, state, p, *drop_words(seed, offset))
    if out is None:
        _lib.dtype_code(x.dtype)
        raise ValueError(f"p must lie in [0, 1], got {p}")
    return out
