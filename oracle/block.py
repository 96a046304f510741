"""Oracle for the operators around a layer's block (numpy, float64): the
width-read with the block's pre-norm, the mix-write with its post-norm, gate,
residual scale and dropout, counter-based dropout, and the gated feed-forward.

Test infrastructure only. The reference has no counterpart of these; the
formulas are those of the operators' documentation, each gradient written out
by hand.
"""

from __future__ import annotations

import numpy as np

from .rw import mix_write_bwd, mix_write_fwd, read_fwd

F = np.float64
_U32 = np.uint64(0xFFFFFFFF)


def philox_words(index, seed: int, offset: int):
    """Word index % 4 of Philox 4x32-10 (Salmon et al., SC 2011) at counter
    (index // 4, offset) under key seed, for an array of element indices."""
    index = np.asarray(index, np.uint64)
    block = index >> np.uint64(2)
    c0, c1 = block & _U32, block >> np.uint64(32)
    c2 = np.full_like(block, offset & 0xFFFFFFFF)
    c3 = np.full_like(block, (offset >> 32) & 0xFFFFFFFF)
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        p0, p1 = c0 * np.uint64(0xD2511F53), c2 * np.uint64(0xCD9E8D57)
        c0, c1, c2, c3 = ((p1 >> np.uint64(32)) ^ c1 ^ np.uint64(k0), p1 & _U32,
                          (p0 >> np.uint64(32)) ^ c3 ^ np.uint64(k1), p0 & _U32)
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.choose((index & np.uint64(3)).astype(np.int64), [c0, c1, c2, c3]).astype(np.uint64)


def keep_mask(count: int, p: float, seed: int, offset: int):
    return philox_words(np.arange(count), seed, offset) >= np.uint64(int(np.floor(p * 2.0**32)))


def dropout(x, p: float, seed: int, offset: int = 0):
    x = np.asarray(x, F)
    if p >= 1.0:
        return np.zeros_like(x)
    keep = keep_mask(x.size, p, seed, offset).reshape(x.shape)
    return np.where(keep, x / (1.0 - p), 0.0)


def norm(u, kind: str, eps: float):
    """(xhat, rstd) over the last axis; "none" gives u itself and 1."""
    u = np.asarray(u, F)
    if kind == "none":
        return u, np.ones(u.shape[:-1] + (1,))
    c = u - u.mean(-1, keepdims=True) if kind == "layer" else u
    rstd = 1.0 / np.sqrt((c * c).mean(-1, keepdims=True) + eps)
    return c * rstd, rstd


def norm_bwd(q, xhat, rstd, kind: str):
    """Gradient before the norm from the gradient q of xhat."""
    if kind == "none":
        return q
    d = q - xhat * (q * xhat).mean(-1, keepdims=True)
    if kind == "layer":
        d = d - q.mean(-1, keepdims=True)
    return d * rstd


def _p(t, E, value):
    return np.full(E, value) if t is None else np.asarray(t, F).reshape(E)


def read_norm(R, x, weight=None, bias=None, kind="rms", eps=1e-6, g=None):
    """y, or with the upstream gradient g [T,m,D]: (y, grad_R, grad_x,
    grad_weight, grad_bias)."""
    R, x = np.asarray(R, F), np.asarray(x, F)
    T, m, _ = R.shape
    D = x.shape[-1]
    w, b = _p(weight, m * D, 1.0), _p(bias, m * D, 0.0)
    xhat, rstd = norm(read_fwd(R, x).reshape(T, m * D), kind, eps)
    y = (xhat * w + b).reshape(T, m, D)
    if g is None:
        return y
    g = np.asarray(g, F).reshape(T, m * D)
    du = norm_bwd(g * w, xhat, rstd, kind).reshape(T, m, D)
    return (y, np.einsum("tkd,tjd->tkj", du, x), np.einsum("tkj,tkd->tjd", R, du), (g * xhat).sum(0), g.sum(0))


def mix_write_norm(H, x, W, f, v=None, *, kind="rms", weight=None, bias=None, eps=1e-6, gate=None, act="linear",
                   scale=None, p=0.0, seed=0, offset=0, g=None):
    """x', or with g [T,n,D] also a dict of every gradient."""
    W, f = np.asarray(W, F), np.asarray(f, F)
    T, m, D = f.shape
    E = m * D
    w, b, s = _p(weight, E, 1.0), _p(bias, E, 0.0), _p(scale, E, 1.0)
    xhat, rstd = norm(f.reshape(T, E), kind, eps)
    base = xhat * w + b
    a = np.ones((T, E)) if gate is None else np.asarray(gate, F).reshape(T, E)
    da = np.ones((T, E))
    if act == "sigmoid" and gate is not None:
        a = 1.0 / (1.0 + np.exp(-a))
        da = a * (1.0 - a)
    keep = np.ones((T, E), bool) if p == 0 else keep_mask(T * E, p, seed, offset).reshape(T, E) & (p < 1)
    factor = np.where(keep, 1.0 / (1.0 - p) if p < 1 else 0.0, 0.0)
    z = np.where(keep, s * a * base * factor, 0.0).reshape(T, m, D)
    out = mix_write_fwd(H, x, W, z, v)
    if g is None:
        return out
    gH, gx, gW, gz, gv = mix_write_bwd(g, H, x, W, z, v)
    gz = np.where(keep, gz.reshape(T, E) * factor, 0.0)
    q = gz * a
    return out, {
        "H": gH, "x": gx, "W": gW, "v": gv, "f": norm_bwd(q * s * w, xhat, rstd, kind).reshape(T, m, D),
        "weight": (q * s * xhat).sum(0), "bias": (q * s).sum(0), "scale": (q * base).sum(0),
        "gate": (gz * s * base * da).reshape(T, m, D),
    }


def act(a, kind: str):
    """(act(a), act'(a))"""
    if kind == "silu":
        s = 1.0 / (1.0 + np.exp(-a))
        return a * s, s * (1.0 + a * (1.0 - s))
    c = np.sqrt(2.0 / np.pi)
    t = np.tanh(c * (a + 0.044715 * a**3))
    return 0.5 * a * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * a * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * a * a)


def gated_ffn(x, w_gate, w_up, w_down, kind="silu", g=None):
    """y, or with g: (y, grad_x, grad_w_gate, grad_w_up, grad_w_down)."""
    x, wg, wu, wd = (np.asarray(t, F) for t in (x, w_gate, w_up, w_down))
    a, b = x @ wg.T, x @ wu.T
    val, der = act(a, kind)
    h = val * b
    y = h @ wd.T
    if g is None:
        return y
    g = np.asarray(g, F)
    dh = g @ wd
    da, db = dh * b * der, dh * val
    return y, da @ wg + db @ wu, da.T @ x, db.T @ x, g.T @ h
