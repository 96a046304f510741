"""GPU test of gated_ffn with a width of 0: every sum of the formula is empty,
so that y and all gradients are 0, in their shapes."""

import pytest
import torch

from tests.test_ffn_gpu import DT, ffn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,D,F,O", [(5, 0, 16, 8), (5, 8, 0, 16), (5, 8, 16, 0), (0, 8, 0, 16), (0, 0, 0, 0), (3, 0, 0, 4)])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_empty_widths(T, D, F, O, dt):
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")
    t = [torch.ones(*s, dtype=DT[dt], device="cuda") for s in ((T, D), (F, D), (F, D), (O, F))]
    with torch.no_grad():
        y = ffn(*t)
    assert y.shape == (T, O) and y.dtype == DT[dt] and (y == 0).all()
    leaves = [a.requires_grad_(True) for a in t]
    y = ffn(*leaves)
    assert y.shape == (T, O) and (y == 0).all()
    y.backward(torch.ones_like(y))
    for a in leaves:
        assert a.grad.shape == a.shape and (a.grad == 0).all()
