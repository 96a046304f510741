"""Error bounds of the operators around a layer's block, counted from the
roundings that they make (half a step of a type t is finfo(t).eps / 2 relative
to the value).

An output of a norm operator is float32 arithmetic rounded once to its type:

    |got - ref| <= half_step(t) |ref| + tiny(t) + C 2^-24 amp

where amp bounds the sum of the absolute values of the terms that the output
is made of (the same formula on absolute values), and C counts the float32
roundings along the longest chain: a sum over a token's E <= 8192 values is 32
serial additions a thread and 10 levels of a tree (42), twice for a gradient
(the norm's sums, then the outer product's); a row of at most 8 + 4 products;
the root, the quotient and a handful of products (about 20). That is below
128, and a sum over T tokens adds T / rows + rows for `rows` partial sums.
"""

from __future__ import annotations

import numpy as np
import torch

U = 2.0**-24
CHAIN = 128


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype) -> float:
    """Half the spacing of the type's subnormals."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def np64(t):
    return t.detach().double().cpu().numpy()


def assert_bounded(got, ref, amp, what: str, chain: float = CHAIN) -> None:
    """|got - ref| <= half_step |ref| + tiny + chain 2^-24 amp, elementwise."""
    dtype = got.dtype
    got, ref = np64(got), np.asarray(ref, np.float64)
    assert got.shape == ref.shape, f"{what}: shape {got.shape}, expected {ref.shape}"
    if not ref.size:
        return
    bound = half_step(dtype) * np.abs(ref) + tiny(dtype) + chain * U * np.broadcast_to(amp, ref.shape)
    err = np.abs(got - ref)
    worst = np.unravel_index(np.argmax(np.where(np.isnan(err), np.inf, err - bound)), err.shape)
    assert (err <= bound).all(), (f"{what} ({dtype}): error {err[worst]:.3e} at {tuple(int(i) for i in worst)} above "
                                  f"{bound[worst]:.3e} (value {ref[worst]:.3e})")
