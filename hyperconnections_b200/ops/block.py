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
"""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .dropout import drop_state, drop_words
from .rw import _check_width, _require_cuda

_NORM = {"none": 0, "rms": 1, "layer": 2}
_GATE = {"linear": 0, "sigmoid": 1}


def _require_one_device(name: str, x: torch.Tensor, tensors) -> None:
    for tname, t in tensors:
        if t is not None and t.device != x.device:
            raise RuntimeError(f"{name} requires tensors on one device (x is on {x.device}, {tname} on {t.device})")


def _needs_grad(tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _f32(t):
    return None if t is None else t.to(torch.float32)


def _param(name: str, t, m: int, D: int):
    """A [m D] parameter in float32, or None."""
    if t is None:
        return None
    assert t.shape in ((m * D,), (m, D)), f"{name} must be {(m * D,)} or {(m, D)}, got {tuple(t.shape)}"
    return t.to(torch.float32).reshape(m * D)


def _scratch(T, n, m, D, code, device):
    words = _lib.lib().hc_norm_scratch_words(T, n, m, D, code)
    return torch.empty(max(words, 1), dtype=torch.float32, device=device), words


def _read_fwd(R, x, weight, bias, norm, eps, with_stats):
    n, D = x.shape[-2], x.shape[-1]
    m = R.shape[-2]
    lead = x.shape[:-2]
    T = math.prod(lead)
    x_c = x.contiguous()
    R_c = R.contiguous()
    w_c = None if weight is None else weight.contiguous()
    b_c = None if bias is None else bias.contiguous()
    y = torch.empty(*lead, m, D, dtype=x.dtype, device=x.device)
    stats = torch.empty(T, 2, dtype=torch.float32, device=x.device) if with_stats else None
    with _lib.on_device(x_c):
        rc = _lib.lib().hc_read_norm_fwd(R_c.data_ptr(), x_c.data_ptr(), _lib.ptr(w_c), _lib.ptr(b_c), y.data_ptr(),
                                         _lib.ptr(stats), T, n, m, D, norm, eps, _lib.dtype_code(x.dtype),
                                         _lib.stream_of(x_c))
    _lib.check(rc, "hc_read_norm_fwd")
    return y, R_c, x_c, w_c, stats


class _ReadNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, R, x, weight, bias, norm, eps):
        y, R_c, x_c, w_c, stats = _read_fwd(R, x, weight, bias, norm, eps, True)
        ctx.save_for_backward(R_c, x_c, w_c, stats)
        ctx.norm = norm
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        R_c, x_c, w_c, stats = ctx.saved_tensors
        n, D = x_c.shape[-2], x_c.shape[-1]
        m = R_c.shape[-2]
        T = stats.shape[0]
        need_R, need_x, need_w, need_b = ctx.needs_input_grad[:4]
        dev, code = x_c.device, _lib.dtype_code(x_c.dtype)
        g_c = g.to(x_c.dtype).contiguous()
        grad_x = torch.empty_like(x_c) if need_x else None
        grad_R = torch.empty_like(R_c) if need_R else None
        grad_w = torch.empty(m * D, dtype=torch.float32, device=dev) if need_w else None
        grad_b = torch.empty(m * D, dtype=torch.float32, device=dev) if need_b else None
        with _lib.on_device(x_c):
            scratch, words = _scratch(T, n, m, D, code, dev) if need_w or need_b else (None, 0)
            rc = _lib.lib().hc_read_norm_bwd(
                g_c.data_ptr(), R_c.data_ptr(), x_c.data_ptr(), _lib.ptr(w_c), stats.data_ptr(), _lib.ptr(grad_x),
                _lib.ptr(grad_R), _lib.ptr(grad_w), _lib.ptr(grad_b), _lib.ptr(scratch), words, T, n, m, D, ctx.norm,
                code, _lib.stream_of(x_c))
        _lib.check(rc, "hc_read_norm_bwd")
        return grad_R, grad_x, grad_w, grad_b, None, None


def hc_read_norm(R: torch.Tensor, x: torch.Tensor, weight=None, bias=None, *, norm: str = "rms",
                 eps: float = 1e-6) -> torch.Tensor:
    """y = weight * norm(R x) + bias per token: R [*, m, n], x [*, n, D] ->
    y [*, m, D], the norm over a token's m D values (see module doc)."""
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
    R, weight, bias = _f32(R), _param("weight", weight, m, D), _param("bias", bias, m, D)
    if _needs_grad((R, x, weight, bias)):
        return _ReadNormFn.apply(R, x, weight, bias, _NORM[norm], float(eps))
    return _read_fwd(R, x, weight, bias, _NORM[norm], float(eps), False)[0]


def _write_fwd(H, x, W, f, v, weight, bias, gate, scale, state, meta, with_stats):
    norm, act, eps, p, seed, offset = meta
    n, D = x.shape[-2], x.shape[-1]
    m = W.shape[-1]
    T = math.prod(x.shape[:-2])
    dense = [None if t is None else t.contiguous() for t in (H, x, W, f, v, weight, bias, gate, scale)]
    x_c = dense[1]
    out = torch.empty_like(x_c)
    stats = torch.empty(T, 2, dtype=torch.float32, device=x.device) if with_stats and norm else None
    with _lib.on_device(x_c):
        rc = _lib.lib().hc_mix_write_norm_fwd(*[_lib.ptr(t) for t in dense], out.data_ptr(), _lib.ptr(stats), T, n, m, D,
                                              norm, act, eps, p, _lib.ptr(state), seed, offset,
                                              _lib.dtype_code(x.dtype), _lib.stream_of(x_c))
    _lib.check(rc, "hc_mix_write_norm_fwd")
    return out, dense, stats


class _MixWriteNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, H, x, W, f, v, weight, bias, gate, scale, state, meta):
        out, dense, stats = _write_fwd(H, x, W, f, v, weight, bias, gate, scale, state, meta, True)
        ctx.save_for_backward(*dense, stats, state)
        ctx.meta = meta
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        *dense, stats, state = ctx.saved_tensors
        H, x, W, f, v, weight, bias, gate, scale = dense
        norm, act, _, p, seed, offset = ctx.meta
        n, D = x.shape[-2], x.shape[-1]
        m = W.shape[-1]
        T = math.prod(x.shape[:-2])
        code = _lib.dtype_code(x.dtype)
        g_c = g.to(x.dtype).contiguous()
        grads = [torch.empty_like(t) if need and t is not None else None
                 for t, need in zip(dense, ctx.needs_input_grad)]
        gH, gx, gW, gf, gv, gw, gb, ggate, gs = grads
        # weight and bias may be absent while their sums are still needed for scale
        params = any(t is not None for t in (gw, gb, gs))
        with _lib.on_device(x):
            scratch, words = _scratch(T, n, m, D, code, x.device) if params else (None, 0)
            rc = _lib.lib().hc_mix_write_norm_bwd(
                g_c.data_ptr(), *[_lib.ptr(t) for t in dense], _lib.ptr(stats),
                *[_lib.ptr(t) for t in (gx, gf, ggate, gH, gW, gv, gw, gb, gs)], _lib.ptr(scratch), words, T, n, m, D,
                norm, act, p, _lib.ptr(state), seed, offset, code, _lib.stream_of(x))
        _lib.check(rc, "hc_mix_write_norm_bwd")
        return (*grads, None, None)


def hc_mix_write_norm(H: torch.Tensor, x: torch.Tensor, W: torch.Tensor, f: torch.Tensor, v=None, *,
                      norm: str = "rms", weight=None, bias=None, eps: float = 1e-6, gate=None,
                      gate_activation: str = "linear", scale=None, dropout_p: float = 0.0, seed=None,
                      offset: int = 0) -> torch.Tensor:
    """x' = H x [+ projection] + W z per token, z = dropout(scale *
    act(gate) * (weight * norm(f) + bias)); gate_activation "linear" or
    "sigmoid"; seed and offset as for ``hc_dropout`` (see module doc)."""
    name = "hc_mix_write_norm"
    scale_t = scale if torch.is_tensor(scale) else None
    seed_t = seed if torch.is_tensor(seed) else None
    named = (("H", H), ("x", x), ("W", W), ("f", f), ("v", v), ("weight", weight), ("bias", bias), ("gate", gate),
             ("scale", scale_t), ("seed", seed_t))
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
    n, D = x.shape[-2], x.shape[-1]
    lead = x.shape[:-2]
    m = W.shape[-1]
    assert H.shape == (*lead, n, n), f"H must be {(*lead, n, n)}, got {tuple(H.shape)}"
    assert W.shape == (*lead, n, m), f"W must be {(*lead, n, 'm')}, got {tuple(W.shape)}"
    assert f.shape == (*lead, m, D), f"f must be {(*lead, m, D)}, got {tuple(f.shape)}"
    if v is not None:
        assert v.shape[-1] == n and v.dim() <= len(lead) + 1, f"v must broadcast to {(*lead, n)}"
        v = _f32(v).expand(*lead, n)
    if gate is not None:
        gate = gate.to(x.dtype).expand(f.shape)
    _check_width(name, n, m)
    H, W = _f32(H), _f32(W)
    if scale is not None and (scale_t is None or scale_t.numel() == 1 and scale_t.shape not in ((m * D,), (m, D))):
        W = W * (scale if scale_t is None else _f32(scale).reshape(()))  # one number: W z scale = (W scale) z
        scale = None
    weight, bias, scale = (_param(k, t, m, D) for k, t in (("weight", weight), ("bias", bias), ("scale", scale)))
    p = float(dropout_p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout_p must lie in [0, 1], got {dropout_p}")
    state, seed, offset = (None, 0, 0) if p == 0.0 else drop_state(name, seed, offset, x)
    meta = (_NORM[norm], _GATE[gate_activation], float(eps), p, *drop_words(seed, offset))
    tensors = (H, x, W, f.to(x.dtype), v, weight, bias, gate, scale)
    if _needs_grad(tensors):
        # the caller may move its seed on before the backward draws the bits again
        return _MixWriteNormFn.apply(*tensors, None if state is None else state.clone(), meta)
    return _write_fwd(*tensors, state, meta, False)[0]
