"""GPU tests of gated_ffn against the float64 oracle (oracle.block).

Bounds, from the roundings that the operator makes. half = finfo(t).eps / 2 is
the relative error of one rounding to type t, U = 2^-24 that of float32.
Elementwise, an output that is a sum of products |p_k| of rounded operands is
off by at most

    half |ref| + (r half + (2 sqrt(K) + 16 + 40) U) sum_k |p_k|

with r the number of roundings to t on the way to an operand: 1 for y (h), 3
for da and db's products (a, b, then da; 8 for what act'' and the other factor
make of the error of a, since |act''| <= 1.1 and |a| is at most about 6 here),
2 sqrt(K) for a float32 sum of K terms (K / 2 in the worst case, which random
signs do not reach; the tensor cores truncate where the FMA units round), and
40 for the activation's exp. That is the worst case; as a whole the roundings
are independent, so the relative 2-norm is held to (1 + r) half as well (each
rounding's rms is at most half / sqrt(3))."""

import numpy as np
import pytest
import torch

from oracle import block as ob
from tests.bounds import U, half_step, np64, tiny

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")


def ffn(*a, **k):
    from hyperconnections_b200.ops import gated_ffn

    return gated_ffn(*a, **k)


def inputs(T, D, F, O, dt, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, std=1.0: (std * torch.randn(*s, generator=g)).to(DT[dt]).cuda()  # noqa: E731
    return [r(T, D), r(F, D, std=D ** -0.5), r(F, D, std=D ** -0.5), r(O, F, std=F ** -0.5)], r(T, O)


def check(got, ref, terms, K, r, what):
    dtype = got.dtype
    got = np64(got)
    half = 0.0 if dtype == torch.float32 else half_step(dtype)
    bound = half * np.abs(ref) + tiny(dtype) + (r * half + (2 * K ** 0.5 + 56) * U) * terms
    err = np.abs(got - ref)
    assert got.shape == ref.shape and np.isfinite(got).all(), what
    assert (err <= bound).all(), f"{what}: error {err.max():.3e}, worst {(err / bound).max():.2f} of its bound"
    norm = np.linalg.norm(ref)
    rel = np.linalg.norm(err) / norm if norm else 0.0
    most = (1 + r) * half + (2 * K ** 0.5 + 56) * U
    assert rel <= most, f"{what}: relative 2-norm {rel:.3e} above {most:.3e}"


def check_all(t, g, act, y, grads=None):
    x, wg, wu, wd = (np64(k) for k in t)
    (T, D), (O, F) = x.shape, wd.shape
    gn = np64(g)
    ref = ob.gated_ffn(x, wg, wu, wd, act, gn)
    a, b = x @ wg.T, x @ wu.T
    val, der = ob.act(a, act)
    aa, ba = np.abs(x) @ np.abs(wg).T, np.abs(x) @ np.abs(wu).T  # |a|, |b| with no cancellation: their float32 error
    # h's terms: what the float32 errors of a and b, a few U of aa and ba, may add is of their size, not of a's and b's
    tail = 64 * U / max(half_step(y.dtype), U)
    ha = np.abs(val * b) + tail * (aa * np.abs(b) * 1.1 + np.abs(val) * ba)
    check(y, ref[0], ha @ np.abs(wd).T, max(F, D), 1 if y.dtype != torch.float32 else 0, "y")
    if grads is None:
        return
    dha = np.abs(gn) @ np.abs(wd)
    daa = dha * (np.abs(b * der) + tail * (ba * 1.2 + 1.2 * aa * np.abs(b)))
    dba = dha * (np.abs(val) + tail * 1.2 * aa)
    if y.dtype != torch.float32:  # the rounding of a moves act' and act by half |a| times their slopes
        daa = daa + dha * np.abs(b) * 1.1 * np.abs(a) / 3
        dba = dba + dha * np.abs(a) * 1.2 / 3
    K = max(T, F, D, O)
    for name, got, want, terms, r in (
            ("grad_x", grads[0], ref[1], daa @ np.abs(wg) + dba @ np.abs(wu), 3),
            ("grad_w_gate", grads[1], ref[2], daa.T @ np.abs(x), 3), ("grad_w_up", grads[2], ref[3], dba.T @ np.abs(x), 3),
            ("grad_w_down", grads[3], ref[4], np.abs(gn).T @ ha, 1)):
        if got is not None:
            check(got, want, terms, K, r, name)


SHAPES = [
    # T, D, F, O, type, act
    (1, 64, 128, 64, "bf16", "silu"),
    (8, 256, 512, 256, "bf16", "silu"),
    (3, 64, 64, 128, "fp16", "gelu_tanh"),
    (16, 136, 264, 72, "fp16", "silu"),
    (17, 136, 264, 72, "bf16", "gelu_tanh"),
    (33, 512, 1000, 512, "bf16", "silu"),
    (128, 128, 256, 128, "bf16", "silu"),
    (129, 384, 640, 384, "fp16", "gelu_tanh"),
    (300, 384, 1536, 384, "bf16", "silu"),
    (1000, 192, 448, 320, "fp16", "silu"),
    (5000, 64, 72, 64, "bf16", "silu"),
    (9000, 72, 1112, 64, "bf16", "silu"),  # several tiles a pair of CTAs in every product
    (20000, 64, 264, 136, "fp16", "gelu_tanh"),
    (50, 333, 887, 101, "bf16", "silu"),
    (50, 333, 880, 104, "fp16", "silu"),
    (129, 63, 65, 67, "fp16", "gelu_tanh"),
    (1, 1, 1, 1, "fp32", "silu"),
    (1, 7, 9, 5, "bf16", "silu"),
    (65, 333, 200, 77, "fp32", "silu"),
    (130, 128, 192, 64, "fp32", "gelu_tanh"),
    (700, 40, 24, 56, "fp32", "silu"),
    (3, 64, 100, 37, "fp32", "gelu_tanh"),
    (4, 1028, 2052, 1030, "fp32", "silu"),
    (24, 72, 136, 260, "fp32", "silu"),
    (25, 72, 136, 260, "fp32", "silu"),
]


@pytest.mark.parametrize("T,D,F,O,dt,act", SHAPES)
def test_forward_and_gradients(T, D, F, O, dt, act):
    t, g = inputs(T, D, F, O, dt)
    leaves = [k.clone().requires_grad_(True) for k in t]
    y = ffn(*leaves, activation=act)
    assert y.dtype == DT[dt] and y.shape == (T, O)
    y.backward(g)
    check_all(t, g, act, y, [k.grad for k in leaves])
    with torch.no_grad():
        check_all(t, g, act, ffn(*t, activation=act))


@pytest.mark.parametrize("only", range(4))
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_single_gradients(only, dt):
    t, g = inputs(200, 128, 256, 192, dt)
    one = [k.clone().requires_grad_(i == only) for i, k in enumerate(t)]
    ffn(*one).backward(g)
    full = [k.clone().requires_grad_(True) for k in t]
    ffn(*full).backward(g)
    assert torch.equal(one[only].grad, full[only].grad)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_empty_batch_and_leading_dimensions(dt):
    t, g = inputs(0, 64, 128, 64, dt)
    leaves = [k.clone().requires_grad_(True) for k in t]
    ffn(*leaves).backward(g)
    assert all((k.grad == 0).all() for k in leaves)
    t, g = inputs(6, 64, 128, 72, dt)
    y = ffn(t[0].view(2, 3, 64), *t[1:])
    assert y.shape == (2, 3, 72) and torch.equal(y.view(6, 72), ffn(*t))


def test_strided_unaligned_and_mixed_dtypes():
    t, g = inputs(40, 128, 256, 64, "bf16")
    want = ffn(*t)
    flat = torch.zeros(t[0].numel() + 1, dtype=torch.bfloat16, device="cuda")
    flat[1:] = t[0].flatten()
    assert torch.equal(ffn(flat[1:].view_as(t[0]), *t[1:]), want)
    w = torch.zeros(t[1].numel() + 3, dtype=torch.bfloat16, device="cuda")
    w[3:] = t[1].flatten()
    assert torch.equal(ffn(t[0], w[3:].view_as(t[1]), *t[2:]), want)
    assert torch.equal(ffn(t[0].t().contiguous().t(), t[1], t[2].t().contiguous().t(), t[3]), want)
    # float32 master weights: cast to x's dtype, gradients in float32
    leaves = [k.float().requires_grad_(True) for k in t[1:]]
    y = ffn(t[0], *leaves)
    assert torch.equal(y, want)
    y.backward(g)
    assert all(k.grad.dtype == torch.float32 for k in leaves)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(ffn(t[0].float(), *[k.float() for k in t[1:]]), want)


def test_special_values_stay_in_their_rows():
    t, _ = inputs(40, 128, 256, 64, "bf16")
    want = ffn(*t)
    bad = t[0].clone()
    bad[7, 3] = float("nan")
    bad[20, 0] = float("inf")
    got = ffn(bad, *t[1:])
    keep = [i for i in range(40) if i not in (7, 20)]
    assert torch.equal(got[keep], want[keep]) and got[7].isnan().all() and not got[20].isfinite().all()


def test_large_pre_activations():
    """exp's range: strongly negative and positive pre-activations end in 0 and in b, not in NaN."""
    for act in ("silu", "gelu_tanh"):
        x = torch.tensor([[-300.0], [300.0], [0.0]], device="cuda").expand(3, 8).contiguous()
        w = torch.eye(8, device="cuda")
        for dt in (torch.float32, torch.bfloat16):
            leaves = [k.clone().to(dt).requires_grad_(True) for k in (x, w, w, w)]
            y = ffn(*leaves, activation=act)
            assert (y[0] == 0).all() and torch.allclose(y[1].float(), torch.full((8,), 9e4, device="cuda"), rtol=2 ** -7)
            y.backward(torch.ones_like(y))
            assert all(k.grad.isfinite().all() for k in leaves)


def test_gradients_against_differences():
    t, g = inputs(9, 16, 24, 12, "fp32")
    for act in ("silu", "gelu_tanh"):
        leaves = [k.clone().requires_grad_(True) for k in t]
        ffn(*leaves, activation=act).backward(g)
        rng = np.random.default_rng(0)
        a64 = [np64(k) for k in t]
        value = lambda s: (ob.gated_ffn(*s, act) * np64(g)).sum()  # noqa: E731
        for i, a in enumerate(a64):
            d, h = rng.standard_normal(a.shape), 1e-5
            up, dn = ([b + sgn * h * d if j == i else b for j, b in enumerate(a64)] for sgn in (1, -1))
            grad = np64(leaves[i].grad)
            assert abs((grad * d).sum() - (value(up) - value(dn)) / (2 * h)) <= 1e-5 * np.abs(grad * d).sum()
