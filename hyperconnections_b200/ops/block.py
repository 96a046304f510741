"""The two halves of a hyper-connection layer with the norms, gate, residual
scale and dropout of the block between them.

    y  = hc_read_norm(R, x, weight, bias)             the block's input
    x' = hc_mix_write_norm(H, x, W, f, v, ...)        from the block's output f

    u[t,k,:]  = sum_j R[t,k,j] x[t,j,:]
    y[t]      = weight * norm(u[t]) + bias            over the E = m D values of a token

    z[t]      = dropout(scale * act(gate[t]) * (weight * norm(f[t]) + bias))
    x'[t,i,:] = sum_j H_ij x_j [+ (v_i - (H v)_i) v^T x] + sum_k W_ik z_k

``hc_read_norm`` is ``hc_read`` followed by the pre-norm that a block starts
with, in one pass over x: u is not stored, and the backward makes it again
from x. ``hc_mix_write_norm`` is ``hc_mix_write`` of a block's output after
its post-norm, an elementwise gate, a residual scale per channel and dropout;
neither z nor the dropout mask is stored.

Shapes: x [*, n, D]; R [*, m, n]; H [*, n, n]; W [*, n, m]; f [*, m, D]; gate
broadcasts to f's shape; weight and bias [m D] or [m, D]; scale the same, or a
number or one-element tensor; v [*, n], or [n] / [1, n] broadcast over the
tokens. 1 <= m <= 4, n <= 8. x, f and gate travel in x's dtype (float32, float16
or bfloat16); the rest in float32, and every gradient comes back in its
tensor's own dtype. norm is "rms" (x / sqrt(mean x^2 + eps)) or "layer"
((x - mean) / sqrt(var + eps)), and for ``hc_mix_write_norm`` also "none".
Dropout's bits are those of ``hc_dropout`` on z as a tensor [*, m, D].

With one stream and one block the norm takes R's size out of y: R's gradient is
then 0 but for eps, and what comes out is mostly rounding.
"""

from __future__ import annotations

import torch

from .. import _lib
from .dropout import drop_state, drop_words
from .rw import _check_width, _require_cuda

_NORM = {"none": 0, "rms": 1, "layer": 2}
_GATE = {"linear": 0, "sigmoid": 1}


def _require_one_device(name: str, x: torch.Tensor, tensors) -> None:
    for tname, t in tensors:
        if t is not None and t.device != x.device:
            raise RuntimeError(f"{name} requires tensors on one device (x is on {x.device}, {tname} on {t.device})")


def _f32(t):
    return None if t is None else t.to(torch.float32)


def _param(name: str, t, m: int, D: int):
    """A [m D] parameter in float32, or None."""
    if t is None:
        return None
    assert t.shape in ((m * D,), (m, D)), f"{name} must be {(m * D,)} or {(m, D)}, got {tuple(t.shape)}"
    return t.to(torch.float32)


def hc_read_norm(R: torch.Tensor, x: torch.Tensor, weight=None, bias=None, *, norm: str = "rms",
                 eps: float = 1e-6) -> torch.Tensor:
    """y = weight * norm(R x) + bias per token: R [*, m, n], x [*, n, D] ->
    y [*, m, D], the norm over a token's m D values (see module doc)."""
    # tensors as the kernels take them go straight there; whatever else comes is named or converted below
    out = _lib.torch_ext().read_norm(R, x, weight, bias, _NORM.get(norm, -1), eps)
    if out is not None:
        return out
    _require_cuda("hc_read_norm", (("R", R), ("x", x), ("weight", weight), ("bias", bias)))
    _require_one_device("hc_read_norm", x, (("R", R), ("weight", weight), ("bias", bias)))
    if x.dim() < 2:
        raise ValueError("x must be [*, n, D]")
    if norm not in ("rms", "layer"):
        raise ValueError(f"norm must be 'rms' or 'layer', got {norm!r}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    n, D = x.shape[-2], x.shape[-1]
    lead = x.shape[:-2]
    assert R.dim() == x.dim() and R.shape[:-2] == lead and R.shape[-1] == n, (
        f"R must be {(*lead, 'm', n)}, got {tuple(R.shape)}")
    m = R.shape[-2]
    _check_width("hc_read_norm", n, m)
    _lib.dtype_code(x.dtype)
    out = _lib.torch_ext().read_norm(_f32(R), x, _param("weight", weight, m, D), _param("bias", bias, m, D), _NORM[norm],
                                     float(eps))
    assert out is not None, f"x must be [*, n, D] with n >= 1, got {tuple(x.shape)}"
    return out


def hc_mix_write_norm(H: torch.Tensor, x: torch.Tensor, W: torch.Tensor, f: torch.Tensor, v=None, *,
                      norm: str = "rms", weight=None, bias=None, eps: float = 1e-6, gate=None,
                      gate_activation: str = "linear", scale=None, dropout_p: float = 0.0, seed=None,
                      offset: int = 0) -> torch.Tensor:
    """x' = H x [+ projection] + W z per token, z = dropout(scale *
    act(gate) * (weight * norm(f) + bias)); gate_activation "linear" or
    "sigmoid"; seed and offset as for ``hc_dropout`` (see module doc)."""
    name = "hc_mix_write_norm"
    if dropout_p == 0:
        state, words = None, (0, 0)
    else:
        state, *words = drop_state(name, seed, offset, x)
        words = drop_words(*words)
    run = _lib.torch_ext().mix_write_norm
    codes = (_NORM.get(norm, -1), _GATE.get(gate_activation, -1))
    if scale is None or torch.is_tensor(scale):  # as in hc_read_norm
        out = run(H, x, W, f, v, weight, bias, gate, scale, state, *codes, eps, dropout_p, *words)
        if out is not None:
            return out
    scale_t = scale if torch.is_tensor(scale) else None
    named = (("H", H), ("x", x), ("W", W), ("f", f), ("v", v), ("weight", weight), ("bias", bias), ("gate", gate),
             ("scale", scale_t))
    _require_cuda(name, named)
    _require_one_device(name, x, named)
    if x.dim() < 2:
        raise ValueError("x must be [*, n, D]")
    if norm not in _NORM:
        raise ValueError(f"norm must be 'rms', 'layer' or 'none', got {norm!r}")
    if gate_activation not in _GATE:
        raise ValueError(f"gate_activation must be 'linear' or 'sigmoid', got {gate_activation!r}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if not 0.0 <= dropout_p <= 1.0:
        raise ValueError(f"dropout_p must lie in [0, 1], got {dropout_p}")
    n, D = x.shape[-2], x.shape[-1]
    lead = x.shape[:-2]
    m = W.shape[-1]
    assert H.shape == (*lead, n, n), f"H must be {(*lead, n, n)}, got {tuple(H.shape)}"
    assert W.shape == (*lead, n, m), f"W must be {(*lead, n, 'm')}, got {tuple(W.shape)}"
    assert f.shape == (*lead, m, D), f"f must be {(*lead, m, D)}, got {tuple(f.shape)}"
    _check_width(name, n, m)
    _lib.dtype_code(x.dtype)
    if v is not None:
        assert v.shape[-1] == n and v.dim() <= len(lead) + 1, f"v must broadcast to {(*lead, n)}"
        v = _f32(v).expand(*lead, n)
    if gate is not None:
        gate = gate.to(x.dtype).expand(f.shape)
    H, W = _f32(H), _f32(W)
    if scale is not None and (scale_t is None or scale_t.numel() == 1 and scale_t.shape not in ((m * D,), (m, D))):
        W = W * (scale if scale_t is None else _f32(scale).reshape(()))  # one number: W z scale = (W scale) z
        scale = None
    weight, bias, scale = (_param(k, t, m, D) for k, t in (("weight", weight), ("bias", bias), ("scale", scale)))
    out = run(H, x, W, f.to(x.dtype), v, weight, bias, gate, scale, state, *codes, float(eps), float(dropout_p), *words)
    assert out is not None, f"x must be [*, n, D] with n >= 1, got {tuple(x.shape)}"
    return out
