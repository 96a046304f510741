"""GPU tests of hc_read_norm and hc_mix_write_norm against the float64 oracle
(oracle.block), every output and gradient, with the bounds of tests/bounds.py.

Shapes: every n and m, row lengths that no vector divides, one token and many,
tokens wider than a CTA, unaligned bases and strided inputs; each norm, gate,
scale, projection and dropout; the special values of a masked place."""

import numpy as np
import pytest
import torch

from oracle import block as ob
from tests.bounds import CHAIN, assert_bounded, np64

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")


def ops():
    from hyperconnections_b200 import ops as o

    return o


def amp_norm(u_abs, xhat, rstd, w, b):
    """Bounds of |xhat|, and of y's terms, from the absolute sums of u."""
    xa = (u_abs + u_abs.mean(-1, keepdims=True)) * rstd
    return xa, xa * np.abs(w) + np.abs(b)


def amp_du(q, xa, rstd):
    """Bound of the terms of rstd (q - mean q - xhat mean(q xhat)) for a row, times (1 + |xhat|) for the error that
    xhat itself carries into the mean."""
    qa = np.abs(q)
    return rstd * (qa + qa.mean(-1, keepdims=True) + xa * (qa * xa).mean(-1, keepdims=True)) * (1 + xa)


SHAPES = [
    # T, n, m, D, type, norm, affine
    (5, 4, 1, 768, "bf16", "rms", "w"),
    (300, 4, 1, 768, "bf16", "layer", "wb"),
    (1, 4, 1, 2048, "bf16", "rms", "w"),
    (8, 4, 1, 2048, "fp16", "rms", ""),
    (7, 1, 1, 64, "fp32", "rms", "w"),
    (33, 2, 2, 96, "fp16", "layer", "wb"),
    (19, 3, 2, 333, "fp32", "layer", "wb"),
    (19, 3, 2, 333, "bf16", "rms", "b"),
    (64, 8, 4, 256, "bf16", "layer", "wb"),
    (10, 8, 1, 1024, "fp32", "rms", "w"),
    (21, 5, 3, 200, "fp16", "rms", "w"),
    (6, 6, 4, 136, "fp32", "layer", "w"),
    (9, 7, 2, 520, "bf16", "rms", "wb"),
    (3, 2, 4, 40, "bf16", "rms", "w"),
    (1, 1, 1, 1, "fp32", "rms", "w"),
    (4, 2, 1, 8, "bf16", "layer", "wb"),
    (2, 4, 2, 4096, "bf16", "rms", "w"),
    (3, 2, 1, 8200, "fp16", "layer", "wb"),
    (700, 4, 1, 384, "bf16", "rms", "w"),
    (2500, 2, 1, 16, "fp32", "layer", "wb"),
]


def read_inputs(T, n, m, D, dt, affine, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, n, D, generator=g) * torch.exp(0.5 * torch.randn(T, 1, 1, generator=g))).to(DT[dt])
    R = torch.sigmoid(torch.randn(T, m, n, generator=g))
    w = 1 + 0.1 * torch.randn(m * D, generator=g) if "w" in affine else None
    b = 0.1 * torch.randn(m * D, generator=g) if "b" in affine else None
    gy = torch.randn(T, m, D, generator=g).to(DT[dt])
    return [None if t is None else t.cuda() for t in (R, x, w, b, gy)]


def leaf(t):
    return None if t is None else t.detach().clone().requires_grad_(True)


def check_read(R, x, w, b, gy, norm, eps, got):
    """got = (y, grad_R, grad_x, grad_w, grad_b), any but y None."""
    T, m, n = R.shape
    D = x.shape[-1]
    E = m * D
    Rn, xn, gn = np64(R), np64(x), np64(gy).reshape(T, E)
    wn, bn = (None if t is None else np64(t).reshape(E) for t in (w, b))
    y, gR, gx, gw, gb = ob.read_norm(Rn, xn, wn, bn, norm, eps, gn)
    w1 = np.ones(E) if wn is None else wn
    u_abs = np.einsum("tkj,tjd->tkd", np.abs(Rn), np.abs(xn)).reshape(T, E)
    xhat, rstd = ob.norm(np.einsum("tkj,tjd->tkd", Rn, xn).reshape(T, E), norm, eps)
    xa, ya = amp_norm(u_abs, xhat, rstd, w1, 0.0 if bn is None else bn)
    dua = amp_du(gn * w1, xa, rstd).reshape(T, m, D)
    assert_bounded(got[0], y, ya.reshape(T, m, D), "y")
    if got[1] is not None:
        assert_bounded(got[1], gR, np.einsum("tkd,tjd->tkj", dua, np.abs(xn)), "grad_R")
    if got[2] is not None:
        assert_bounded(got[2], gx, np.einsum("tkj,tkd->tjd", np.abs(Rn), dua), "grad_x")
    if got[3] is not None:
        assert_bounded(got[3].reshape(E), gw, (np.abs(gn) * xa).sum(0), "grad_weight", CHAIN + T / 64)
    if got[4] is not None:
        assert_bounded(got[4].reshape(E), gb, np.abs(gn).sum(0), "grad_bias", CHAIN + T / 64)


@pytest.mark.parametrize("T,n,m,D,dt,norm,affine", SHAPES)
def test_read_norm(T, n, m, D, dt, norm, affine):
    R, x, w, b, gy = read_inputs(T, n, m, D, dt, affine)
    leaves = [leaf(t) for t in (R, x, w, b)]
    y = ops().hc_read_norm(*leaves, norm=norm, eps=1e-5)
    assert y.dtype == x.dtype and y.shape == (T, m, D)
    y.backward(gy)
    check_read(R, x, w, b, gy, norm, 1e-5, [y] + [None if t is None else t.grad for t in leaves])
    with torch.no_grad():
        assert torch.equal(ops().hc_read_norm(R, x, w, b, norm=norm, eps=1e-5), y)


def write_inputs(T, n, m, D, dt, affine, gate, proj, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = dict(x=r(T, n, D).to(DT[dt]), f=(r(T, m, D) * torch.exp(0.5 * r(T, 1, 1))).to(DT[dt]),
             H=torch.eye(n) + 0.2 * r(T, n, n), W=2 * torch.sigmoid(r(T, n, m)),
             v=torch.nn.functional.normalize(r(T, n), dim=-1) if proj else None,
             weight=1 + 0.1 * r(m * D) if "w" in affine else None, bias=0.1 * r(m * D) if "b" in affine else None,
             gate=r(T, m, D).to(DT[dt]) if gate else None, scale=0.1 + 0.02 * r(m * D) if "s" in affine else None)
    gx = r(T, n, D).to(DT[dt])
    return {k: None if a is None else a.cuda() for k, a in t.items()}, gx.cuda()


def check_write(t, g, norm, eps, act, p, seed, offset, out, grads):
    T, n, D = t["x"].shape
    m = t["W"].shape[-1]
    E = m * D
    a64 = {k: None if a is None else np64(a) for k, a in t.items()}
    gn = np64(g)
    kw = dict(kind=norm, weight=a64["weight"], bias=a64["bias"], eps=eps, gate=a64["gate"], act=act,
              scale=a64["scale"], p=p, seed=seed, offset=offset)
    ref, rg = ob.mix_write_norm(a64["H"], a64["x"], a64["W"], a64["f"], a64["v"], g=gn, **kw)
    # the terms' absolute values
    one = lambda k, d: np.full(E, d) if a64[k] is None else np.abs(a64[k].reshape(E))  # noqa: E731
    w, b, s = one("weight", 1.0), one("bias", 0.0), one("scale", 1.0)
    Ha, xa, Wa, ga = (np.abs(k) for k in (a64["H"], a64["x"], a64["W"], gn))
    if t["v"] is not None:
        va = np.abs(a64["v"])
        c = va + np.einsum("tij,tj->ti", Ha, va)
        Ha = Ha + np.einsum("ti,tj->tij", c, va)
    _, rstd = ob.norm(a64["f"].reshape(T, E), norm, eps)
    fa = np.abs(a64["f"].reshape(T, E))
    xh = fa if norm == "none" else (fa + (fa.mean(-1, keepdims=True) if norm == "layer" else 0)) * rstd
    gt = np.ones((T, E)) if t["gate"] is None else np.abs(a64["gate"].reshape(T, E))
    gate = np.ones((T, E)) if act == "sigmoid" and t["gate"] is not None else gt
    base = xh * w + b
    drop = 1.0 / (1.0 - p) if p < 1 else 0.0
    za = (s * gate * base * drop).reshape(T, m, D)
    # sigmoid(a) from exp(-a): |a| + 2 roundings of its exponent's argument
    oa = np.einsum("tij,tjd->tid", Ha, xa) + np.einsum("tik,tkd->tid", Wa, za * (1 + gt.reshape(T, m, D) / 64))
    assert_bounded(out, ref, oa, "out")
    dz = np.einsum("tik,tid->tkd", Wa, ga).reshape(T, E) * drop * (1 + gt / 64)
    q = dz * gate
    amp = dict(
        H=np.einsum("tid,tjd->tij", ga, xa), x=np.einsum("tij,tid->tjd", Ha, ga),
        W=np.einsum("tid,tkd->tik", ga, za * (1 + gt.reshape(T, m, D) / 64)),
        f=(q * s * w if norm == "none" else amp_du(q * s * w, xh, rstd)).reshape(T, m, D),
        weight=(q * s * xh).sum(0), bias=(q * s).sum(0), scale=(q * base).sum(0), gate=(dz * s * base).reshape(T, m, D))
    if t["v"] is not None:
        G = amp["H"]
        gc = np.einsum("tij,tj->ti", G, va)
        amp["H"] = G + np.einsum("ti,tj->tij", gc, va)
        amp["v"] = np.einsum("ti,tij->tj", c, G) + gc + np.einsum("tij,ti->tj", np.abs(a64["H"]), gc)
    for k, got in grads.items():
        chain = CHAIN + (T / 64 if k in ("weight", "bias", "scale") else 0)
        assert_bounded(got, rg[k].reshape(got.shape), np.asarray(amp[k]).reshape(got.shape), f"grad_{k}", chain)


WRITE = [
    # T, n, m, D, type, norm, affine, gate, proj, p
    (5, 4, 1, 768, "bf16", "rms", "ws", "sigmoid", False, 0.1),
    (300, 4, 1, 768, "bf16", "layer", "wbs", "linear", False, 0.0),
    (1, 4, 1, 2048, "bf16", "rms", "ws", "sigmoid", False, 0.0),
    (8, 4, 1, 2048, "fp16", "rms", "w", "", False, 0.3),
    (7, 1, 1, 64, "fp32", "none", "s", "linear", False, 0.5),
    (33, 2, 2, 96, "fp16", "layer", "wb", "", True, 0.0),
    (19, 3, 2, 333, "fp32", "layer", "wbs", "sigmoid", True, 0.2),
    (19, 3, 2, 333, "bf16", "rms", "b", "linear", False, 0.1),
    (64, 8, 4, 256, "bf16", "layer", "wbs", "sigmoid", True, 0.1),
    (40, 8, 2, 1024, "fp16", "layer", "wbs", "", True, 0.0),
    (10, 8, 1, 1024, "fp32", "rms", "w", "sigmoid", False, 0.0),
    (21, 5, 3, 200, "fp16", "rms", "ws", "linear", True, 0.9),
    (6, 6, 4, 136, "fp32", "none", "", "", True, 0.0),
    (9, 7, 2, 520, "bf16", "rms", "wb", "sigmoid", False, 0.1),
    (3, 2, 4, 40, "bf16", "rms", "w", "linear", True, 0.4),
    (1, 1, 1, 1, "fp32", "rms", "ws", "linear", True, 0.5),
    (4, 2, 1, 8, "bf16", "none", "w", "sigmoid", False, 0.1),
    (2, 4, 2, 4096, "bf16", "rms", "ws", "", False, 0.1),
    (3, 2, 1, 8200, "fp16", "layer", "wb", "sigmoid", False, 0.1),
    (700, 4, 1, 384, "bf16", "rms", "ws", "sigmoid", False, 0.1),
    (6, 4, 1, 96, "bf16", "rms", "ws", "sigmoid", False, 1.0),
]


@pytest.mark.parametrize("T,n,m,D,dt,norm,affine,gate,proj,p", WRITE)
def test_mix_write_norm(T, n, m, D, dt, norm, affine, gate, proj, p):
    t, g = write_inputs(T, n, m, D, dt, affine, gate, proj)
    seed, offset = 0x1234567890ABCDEF, (1 << 40) + 3
    kw = dict(norm=norm, eps=1e-5, gate_activation=gate or "linear", dropout_p=p, seed=seed, offset=offset)
    call = lambda s: ops().hc_mix_write_norm(s["H"], s["x"], s["W"], s["f"], s["v"], weight=s["weight"],  # noqa: E731
                                             bias=s["bias"], gate=s["gate"], scale=s["scale"], **kw)
    leaves = {k: leaf(a) for k, a in t.items()}
    out = call(leaves)
    assert out.dtype == t["x"].dtype and out.shape == (T, n, D)
    out.backward(g)
    check_write(t, g, norm, 1e-5, gate or "linear", p, seed, offset, out,
                {k: a.grad for k, a in leaves.items() if a is not None})
    with torch.no_grad():
        assert torch.equal(call(t), out)


def test_strided_unaligned_and_other_dtypes():
    """Transposed weights, streams that start off a 16-byte boundary or stride through a larger tensor, half-precision
    per-token weights: the values of the dense call on the same numbers, and gradients in each tensor's own dtype."""
    T, n, m, D = 17, 4, 2, 256
    R, x, w, b, gy = read_inputs(T, n, m, D, "bf16", "wb")
    want = ops().hc_read_norm(R, x, w, b, norm="layer")
    flat = torch.zeros(x.numel() + 1, dtype=x.dtype, device="cuda")
    flat[1:] = x.flatten()
    odd = flat[1:].view_as(x)
    wide = torch.zeros(T, 2 * n, D, dtype=x.dtype, device="cuda")
    wide[:, ::2] = x
    for xs in (odd, wide[:, ::2], x.transpose(1, 2).contiguous().transpose(1, 2)):
        got = ops().hc_read_norm(R.transpose(1, 2).contiguous().transpose(1, 2), xs, w.view(m, D), b, norm="layer")
        # the element kernels sum in another order
        check_read(R, x, w, b, gy, "layer", 1e-6, [got, None, None, None, None])
        assert (got.float() - want.float()).abs().max() <= 2 ** -7 * want.float().abs().max()
    Rh = R.half().requires_grad_(True)
    wh = w.bfloat16().requires_grad_(True)
    y = ops().hc_read_norm(Rh, x, wh)
    y.backward(gy)
    assert Rh.grad.dtype == torch.float16 and wh.grad.dtype == torch.bfloat16


def test_broadcast_gate_direction_and_scalar_scale():
    """A gate a sample (summed over its tokens), a shared direction and a one-element scale: gradients in their own shapes."""
    B, S, n, m, D = 3, 5, 4, 1, 64
    t, g = write_inputs(B * S, n, m, D, "fp32", "w", "linear", False)
    sh = lambda a: a.view(B, S, *a.shape[1:])  # noqa: E731
    gate = torch.randn(B, 1, m, D, device="cuda", requires_grad=True)
    v = torch.nn.functional.normalize(torch.randn(n, device="cuda"), dim=0).requires_grad_(True)
    s = torch.tensor([0.3], device="cuda", requires_grad=True)
    out = ops().hc_mix_write_norm(sh(t["H"]), sh(t["x"]), sh(t["W"]), sh(t["f"]), v, weight=t["weight"], gate=gate, scale=s)
    out.backward(sh(g))
    full = {**t, "gate": gate.detach().expand(B, S, m, D).reshape(B * S, m, D), "v": v.detach().expand(B * S, n),
            "scale": torch.full((m * D,), s.item(), device="cuda")}
    a64 = {k: None if a is None else np64(a) for k, a in full.items()}
    ref, rg = ob.mix_write_norm(a64["H"], a64["x"], a64["W"], a64["f"], a64["v"], weight=a64["weight"], gate=a64["gate"],
                                scale=a64["scale"], g=np64(g))
    close = lambda got, want: np.abs(np64(got) - want).max() <= 1e-5 * max(1.0, np.abs(want).max())  # noqa: E731
    assert close(out.reshape(B * S, n, D), ref)
    assert gate.grad.shape == gate.shape and close(gate.grad, rg["gate"].reshape(B, S, m, D).sum(1, keepdims=True))
    assert v.grad.shape == (n,) and close(v.grad, rg["v"].sum(0))
    assert s.grad.shape == (1,) and close(s.grad, rg["scale"].sum(keepdims=True))
    # a number as the scale, and none of the gradients that nobody asked for
    half = ops().hc_mix_write_norm(t["H"], t["x"], t["W"], t["f"], scale=0.5)
    want = ob.mix_write_norm(a64["H"], a64["x"], a64["W"], a64["f"], scale=np.full(m * D, 0.5))
    assert close(half, want)


@pytest.mark.parametrize("only", ["R", "x", "weight", "bias"])
def test_read_norm_single_gradients(only):
    R, x, w, b, gy = read_inputs(40, 4, 2, 128, "bf16", "wb")
    t = dict(R=R, x=x, weight=w, bias=b)
    t[only] = leaf(t[only])
    ops().hc_read_norm(**t, norm="layer").backward(gy)
    full = {k: leaf(a) for k, a in dict(R=R, x=x, weight=w, bias=b).items()}
    ops().hc_read_norm(**full, norm="layer").backward(gy)
    assert torch.equal(t[only].grad, full[only].grad)


@pytest.mark.parametrize("only", ["H", "x", "W", "f", "v", "weight", "bias", "gate", "scale"])
def test_mix_write_norm_single_gradients(only):
    t, g = write_inputs(40, 4, 2, 128, "bf16", "wbs", "sigmoid", True)
    kw = dict(norm="layer", gate_activation="sigmoid", dropout_p=0.2, seed=3)
    one = {k: leaf(a) if k == only else a for k, a in t.items()}
    ops().hc_mix_write_norm(**one, **kw).backward(g)
    full = {k: leaf(a) for k, a in t.items()}
    ops().hc_mix_write_norm(**full, **kw).backward(g)
    assert torch.equal(one[only].grad, full[only].grad)


@pytest.mark.parametrize("D", [256, 333])
def test_empty_batch(D):
    R, x, w, b, gy = read_inputs(0, 4, 2, D, "bf16", "wb")
    leaves = [leaf(t) for t in (R, x, w, b)]
    y = ops().hc_read_norm(*leaves)
    assert y.shape == (0, 2, D)
    y.backward(gy)
    assert all((t.grad == 0).all() for t in leaves)
    t, g = write_inputs(0, 4, 2, D, "bf16", "wbs", "sigmoid", True)
    ls = {k: leaf(a) for k, a in t.items()}
    ops().hc_mix_write_norm(**ls, dropout_p=0.1, seed=1).backward(g)
    assert all((a.grad == 0).all() for a in ls.values())


@pytest.mark.parametrize("D", [256, 333])
def test_special_values_stay_in_their_token(D):
    """An infinity or a NaN in one token reaches that token's outputs only, and a dropped place is 0 whatever it held."""
    T, n, m = 6, 4, 1
    R, x, w, b, gy = read_inputs(T, n, m, D, "bf16", "wb")
    bad = x.clone()
    bad[2, 1, 3] = float("nan")
    bad[4, 0, 0] = float("inf")
    clean, dirty = ops().hc_read_norm(R, x, w, b), ops().hc_read_norm(R, bad, w, b)
    keep = [0, 1, 3, 5]
    assert torch.equal(clean[keep], dirty[keep])
    assert dirty[2].isnan().all() and dirty[4].isnan().any()
    # norm none, linear gate: NaN exactly where the mask keeps
    t, g = write_inputs(T, n, m, D, "fp32", "", "linear", False)
    t["f"][:] = float("nan")
    out = ops().hc_mix_write_norm(**t, norm="none", dropout_p=0.5, seed=9, offset=2)
    keep = ob.keep_mask(T * D, 0.5, 9, 2).reshape(T, D)
    assert np.array_equal(np.isnan(np64(out)), np.broadcast_to(keep[:, None], (T, n, D)))
    t["f"].requires_grad_(True)
    g[:] = 1.0
    ops().hc_mix_write_norm(**t, norm="none", dropout_p=0.5, seed=9, offset=2).backward(g)
    assert np.array_equal(np64(t["f"].grad[:, 0]) == 0, ~keep)


def test_zero_rows_and_constant_rows():
    """A token of zeros (nothing to normalise) gives bias; a constant row has no variance."""
    T, n, m, D = 4, 2, 1, 128
    R, x, w, b, gy = read_inputs(T, n, m, D, "fp32", "wb")
    x[1] = 0
    x[2] = 3.0
    for norm in ("rms", "layer"):
        y = ops().hc_read_norm(R, x, w, b, norm=norm, eps=1e-6)
        assert torch.equal(y[1, 0], b)
        assert y.isfinite().all()
    # the row is constant up to the rounding of R's sum, which layer norm at this eps amplifies at most 1e3-fold
    assert (y[2, 0] - b).abs().max() <= 1e3 * 1.1 * 3 * 2 * 8 * 2 ** -24


def test_gradients_against_differences():
    """float32 operators against central differences of the float64 formula along random directions."""
    t, g = write_inputs(5, 3, 2, 24, "fp32", "wbs", "sigmoid", True)
    kw = dict(norm="layer", gate_activation="sigmoid", dropout_p=0.3, seed=11, offset=4, eps=1e-3)
    leaves = {k: leaf(a) for k, a in t.items()}
    ops().hc_mix_write_norm(**leaves, **kw).backward(g)
    rng = np.random.default_rng(0)
    a64 = {k: np64(a) for k, a in t.items()}

    def value(s):
        out = ob.mix_write_norm(s["H"], s["x"], s["W"], s["f"], s["v"], kind="layer", weight=s["weight"], bias=s["bias"],
                                eps=1e-3, gate=s["gate"], act="sigmoid", scale=s["scale"], p=0.3, seed=11, offset=4)
        return (out * np64(g)).sum()

    for k in a64:
        d = rng.standard_normal(a64[k].shape)
        h = 1e-5
        diff = (value({**a64, k: a64[k] + h * d}) - value({**a64, k: a64[k] - h * d})) / (2 * h)
        got = (np64(leaves[k].grad) * d).sum()
        scale = np.abs(np64(leaves[k].grad) * d).sum()
        assert abs(got - diff) <= 1e-5 * scale, k


def test_on_another_stream_and_two_at_once():
    """Two calls on two streams give what each gives alone."""
    a = read_inputs(512, 4, 1, 768, "bf16", "w", seed=1)
    b = read_inputs(512, 4, 1, 768, "bf16", "w", seed=2)

    def step(inp):
        leaves = [leaf(t) for t in inp[:3]]
        y = ops().hc_read_norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, inp[4])]

    want = [step(a), step(b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s, inp in zip(streams, (a, b)):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step(inp))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(g, w))
