"""GPU tests of gated_ffn's activation and its derivative, value by value.

With w_gate and w_down the identity and b = 1 for every element, y = h =
act(x) and the gradient of x for an upstream of ones is act'(x), each float32
arithmetic rounded once (the products add zeros only, and rounding a second
time changes nothing). With s = 1 / (1 + e^-2u) (SiLU: e^-a), val = a s and
der = s + a s (1 - s) w with w = d(2u)/da, so that

    |y - val|   <= half |val| + tiny + C 2^-24 |val|
    |dx - der|  <= half |der| + tiny + C 2^-24 (s + |a s (1 - s) w|)

C: the exponent's argument, at most 36 (in powers of two) for |a| <= 6, has five
roundings, which are 36 x 5 x ln 2 = 125 of the result; the exponential, the sum,
the inverse and the products are below 15 more (ex2.approx and rcp.approx: a few
2^-22). In der, 1 - s has up to 2 2^-24 of its own, which w |a| <= 56 takes to
112 where s is near 1 (the exponential's part is small there). So C = 160 for val
and 220 for der, below the half steps of the 16-bit types (2^13 2^-24 in fp16)."""

import numpy as np
import pytest
import torch

from tests.bounds import U, half_step, np64, tiny
from tests.test_ffn_gpu import DT, ffn

pytestmark = pytest.mark.gpu

COLS = 64


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")


def reference(a, act):
    """val, der and the absolute values of der's terms, in float64 and without a cancelling sum."""
    if act == "silu":
        arg, w = a, 1.0
    else:
        c = np.sqrt(2 / np.pi)
        arg, w = 2 * c * (a + 0.044715 * a**3), 2 * c * (1 + 3 * 0.044715 * a**2)
    s, rest = 1 / (1 + np.exp(-arg)), 1 / (1 + np.exp(arg))
    return a * s, s + a * s * rest * w, s + np.abs(a * s * rest * w)


@pytest.mark.parametrize("lo,hi", [(-6.0, -3.0), (-3.0, 6.0)])
@pytest.mark.parametrize("T", [3, 20, 40, 300])  # streamed weights, a few tokens, tiles
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_values(dt, act, T, lo, hi):
    x = torch.zeros(T, COLS + 8)
    x[:, :COLS] = torch.linspace(lo, hi, T * COLS).view(T, COLS)
    x[:, COLS] = 1.0
    eye = torch.zeros(COLS, COLS + 8)
    eye[:, :COLS] = torch.eye(COLS)
    one = torch.zeros(COLS, COLS + 8)
    one[:, COLS] = 1.0
    x, gate, up, down = (t.to(DT[dt]).cuda() for t in (x, eye, one, torch.eye(COLS)))
    leaf = x.requires_grad_(True)
    y = ffn(leaf, gate, up, down, activation=act)
    y.backward(torch.ones_like(y))
    val, der, amp = reference(np64(x)[:, :COLS], act)
    half, least = half_step(DT[dt]), tiny(DT[dt])
    for got, ref, a, chain in ((np64(y), val, np.abs(val), 160), (np64(leaf.grad)[:, :COLS], der, amp, 220)):
        err, bound = np.abs(got - ref), half * np.abs(ref) + least + chain * U * a
        assert (err <= bound).all(), f"{(err / bound).max():.2f} of the bound, at x = {np64(x)[:, :COLS][np.unravel_index((err / bound).argmax(), err.shape)]:.3f}"
