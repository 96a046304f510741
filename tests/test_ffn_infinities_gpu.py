"""GPU test of gated_ffn where x holds infinities and the hidden width is no
multiple of 8: with positive weights every product of the formula is +inf, and
so is y, whatever the columns that only fill a row up hold."""

import pytest
import torch

from tests.test_ffn_gpu import DT, ffn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("F", [1, 20, 33, 64])
@pytest.mark.parametrize("T", [1, 4, 20, 40])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_infinite_rows(dt, act, T, F):
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")
    g = torch.Generator().manual_seed(F)
    pos = lambda *s: (0.5 + torch.rand(*s, generator=g)).to(DT[dt]).cuda()  # noqa: E731
    x, weights = pos(T, 24), [pos(F, 24), pos(F, 24), pos(16, F)]
    want = ffn(x, *weights, activation=act)
    x[0, 3] = float("inf")
    y = ffn(x, *weights, activation=act)
    assert (y[0] == float("inf")).all()
    assert torch.equal(y[1:], want[1:]) and want.isfinite().all()
