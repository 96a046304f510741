"""Gated feed-forward block, forward and backward.

    y = gated_ffn(x, w_gate, w_up, w_down, activation="silu")
    y = (act(x w_gate^T) * (x w_up^T)) w_down^T

x [*, D], w_gate and w_up [F, D], w_down [O, F] (the layouts of
``nn.Linear.weight``) -> y [*, O], at most 2^22 rows of x and widths of 2^20; activation "silu" or "gelu_tanh" (the
tanh form of GELU). Both projections, the activation and the product are one
kernel, which writes h = act(a) * b and, when a backward follows, what dh is
multiplied with there: act'(a) b and act(a). The backward does that where it
makes dh = g w_down, and sums dx = da w_gate + db w_up in one product.

Weights are cast to x's dtype (float32, float16 or bfloat16; under autocast
all four tensors to the autocast dtype, as ``F.linear`` does). Products are
summed in float32; h, the two slopes and the gradients da and db are rounded
once to that dtype (h, da and db are operands of the products that follow).
"""

from __future__ import annotations

import torch

from .. import _lib

_ACT = {"silu": 2, "gelu_tanh": 3}


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, *,
              activation: str = "silu") -> torch.Tensor:
    """y = (act(x w_gate^T) * (x w_up^T)) w_down^T (see module doc)."""
    autocast = torch.is_autocast_enabled("cuda")
    if not autocast:
        # tensors as the kernels take them go straight there; whatever else comes is named or converted below
        out = _lib.torch_ext().gated_ffn(x, w_gate, w_up, w_down, _ACT.get(activation, -1))
        if out is not None:
            return out
    for name, t in (("x", x), ("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        if not t.is_cuda:
            raise RuntimeError(f"gated_ffn requires CUDA tensors ({name} is on {t.device})")
        if t.device != x.device:
            raise RuntimeError(f"gated_ffn requires tensors on one device (x is on {x.device}, {name} on {t.device})")
    if activation not in _ACT:
        raise ValueError(f"activation must be 'silu' or 'gelu_tanh', got {activation!r}")
    if x.dim() < 1 or w_gate.dim() != 2:
        raise ValueError("x must be [*, D] and w_gate [F, D]")
    F, D = w_gate.shape
    assert x.shape[-1] == D, f"x must be {('*', D)}, got {tuple(x.shape)}"
    assert w_up.shape == (F, D), f"w_up must be {(F, D)}, got {tuple(w_up.shape)}"
    assert w_down.dim() == 2 and w_down.shape[1] == F, f"w_down must be {('O', F)}, got {tuple(w_down.shape)}"
    dt = torch.get_autocast_dtype("cuda") if autocast else x.dtype
    _lib.dtype_code(dt)
    return _lib.torch_ext().gated_ffn(*[t.to(dt) for t in (x, w_gate, w_up, w_down)], _ACT[activation])
