"""Gated feed-forward block, forward and backward.

    y = gated_ffn(x, w_gate, w_up, w_down, activation="silu")
    y = (act(x w_gate^T) * (x w_up^T)) w_down^T

x [*, D], w_gate and w_up [F, D], w_down [O, F] (the layouts of
``nn.Linear.weight``) -> y [*, O]; activation "silu" or "gelu_tanh" (the
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

import math

import torch
from torch.autograd.function import once_differentiable

from .. import _lib

_ACT = {"silu": 2, "gelu_tanh": 3}


def _scratch(backward: int, T, D, F, O, code, device):
    size = _lib.lib().hc_gated_ffn_scratch_bytes(backward, T, D, F, O, code)
    return (torch.empty(size, dtype=torch.uint8, device=device) if size > 0 else None), max(size, 0)


def _dense(t):
    """t itself, or a copy where it is strided or starts off a 16-byte boundary (the tensor copies need one)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _forward(x, w_gate, w_up, w_down, act, keep):
    D, (O, F) = x.shape[-1], w_down.shape
    lead = x.shape[:-1]
    T = math.prod(lead)
    dense = [_dense(t) for t in (x, w_gate, w_up, w_down)]
    x_c = dense[0]
    dev, dt, code = x.device, x.dtype, _lib.dtype_code(x.dtype)
    Fp = (F + 7) // 8 * 8
    y = torch.empty(*lead, O, dtype=dt, device=dev)
    h = torch.empty(T, Fp, dtype=dt, device=dev)
    slopes = [torch.empty(T, Fp, dtype=dt, device=dev) if keep else None for _ in range(2)]
    with _lib.on_device(x_c):
        scratch, size = _scratch(0, T, D, F, O, code, dev)
        rc = _lib.lib().hc_gated_ffn_fwd(*[t.data_ptr() for t in dense], y.data_ptr(), h.data_ptr(),
                                         *[_lib.ptr(t) for t in slopes], _lib.ptr(scratch), size, T, D, F, O, act, code,
                                         _lib.stream_of(x_c))
    _lib.check(rc, "hc_gated_ffn_fwd")
    return y, dense, h, slopes


class _GatedFfnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, act):
        y, dense, h, slopes = _forward(x, w_gate, w_up, w_down, act, True)
        ctx.save_for_backward(*dense, h, *slopes)
        ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, w_gate, w_up, w_down, h, slope_gate, slope_up = ctx.saved_tensors
        (O, F), D, T = w_down.shape, x.shape[-1], h.shape[0]
        code = _lib.dtype_code(x.dtype)
        g_c = _dense(g.to(x.dtype))
        grads = [torch.empty_like(t) if need else None
                 for t, need in zip((x, w_gate, w_up, w_down), ctx.needs_input_grad)]
        inner = any(t is not None for t in grads[:3])
        d_pre = [torch.empty_like(h) if inner else None for _ in range(2)]
        with _lib.on_device(x):
            scratch, size = _scratch(1, T, D, F, O, code, x.device)
            rc = _lib.lib().hc_gated_ffn_bwd(
                *[t.data_ptr() for t in (g_c, x, w_gate, w_up, w_down, h, slope_gate, slope_up)],
                *[_lib.ptr(t) for t in (*d_pre, *grads, scratch)], size, T, D, F, O, ctx.act, code, _lib.stream_of(x))
        _lib.check(rc, "hc_gated_ffn_bwd")
        return (*grads, None)


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, *,
              activation: str = "silu") -> torch.Tensor:
    """y = (act(x w_gate^T) * (x w_up^T)) w_down^T (see module doc)."""
    if not _lib.available():
        raise RuntimeError("gated_ffn requires the hyperconnections_b200 CUDA kernels (libhcops.so)")
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
    dt = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype
    _lib.dtype_code(dt)
    tensors = [t.to(dt) for t in (x, w_gate, w_up, w_down)]
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        return _GatedFfnFn.apply(*tensors, _ACT[activation])
    return _forward(*tensors, _ACT[activation], False)[0]
